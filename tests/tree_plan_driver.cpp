// The work list of tree attention behind a plain C function, for tests without a GPU.
#include "attn_tree.hpp"

#include <cstring>

// out: per piece {cta, kv_head, row_begin, n_rows, tile_begin, n_tiles, slot, prefix, draft, token0, pt_off}; splits: per split
// {kv_head, row_begin, n_rows, token0, first_slot, n_parts, first_row, slot_step}; counts: {pieces, ctas, splits, merged rows, slots, slot rows}.
extern "C" int tree_work(size_t batch, size_t H, size_t KVH, const uint32_t* prefix, const uint32_t* draft, const uint32_t* pt_off,
                         uint32_t max_ctas, uint32_t* out, size_t out_words, uint32_t* splits, size_t split_words, uint32_t* row_split,
                         size_t row_words, uint32_t* counts) {
    mlcb::TreeShape s;
    s.batch = batch;
    s.H = H;
    s.KVH = KVH;
    mlcb::TreeTables t;
    t.prefix = prefix;
    t.draft = draft;
    t.pt_off = pt_off;
    mlcb::TreeWork w;
    mlcb::tree_work_list(s, t, max_ctas, &w);
    if (w.pieces.size() * 11 > out_words || w.splits.size() * 8 > split_words || w.row_split.size() > row_words) return 0;
    size_t n_out = 0;
    for (uint32_t c = 0; c < w.n_cta; ++c)
        for (uint32_t i = 0; i <= w.pieces[c].more; ++i, ++n_out) {
            const size_t at = i ? w.pieces[c].next + i - 1 : c;
            if (at >= w.pieces.size()) return 0;
            const mlcb::TreePiece& p = w.pieces[at];
            const uint32_t v[11] = {c, p.kv_head, p.row_begin, p.n_rows, p.tile_begin, p.n_tiles, p.slot,
                                    p.prefix, p.draft, p.token0, p.pt_off};
            std::memcpy(out + 11 * n_out, v, sizeof(v));
        }
    if (n_out != w.pieces.size()) return 0;
    for (size_t i = 0; i < w.splits.size(); ++i) {
        const mlcb::TreeSplit& p = w.splits[i];
        const uint32_t v[8] = {p.kv_head, p.row_begin, p.n_rows, p.token0, p.first_slot, p.n_parts, p.first_row, p.slot_step};
        std::memcpy(splits + 8 * i, v, sizeof(v));
    }
    if (!w.row_split.empty()) std::memcpy(row_split, w.row_split.data(), w.row_split.size() * 4);
    const uint32_t n[6] = {static_cast<uint32_t>(w.pieces.size()), w.n_cta,
                           static_cast<uint32_t>(w.splits.size()), static_cast<uint32_t>(w.row_split.size()), w.n_slots, w.slot_rows};
    std::memcpy(counts, n, sizeof(n));
    return 1;
}
