// Work list of the tensor-core kernel of tree attention (host arithmetic only).
//
// A unit is what shares K and V in one CTA: (request, KV head, row tile), a row tile being up to 128 query rows (drafted
// token, head of the group). Its work is the number of 64-token cache tiles. The units are laid end to end and cut into
// equal runs, one per CTA, so that every CTA gets the same number of tiles whatever the spread of context lengths; a unit
// cut between CTAs leaves partials that a second kernel joins. A CTA holds at most two partials this way.
#include <algorithm>

#include "attn_tree.hpp"

namespace mlcb {

namespace {

// Tiles a piece's fixed work (queries in, output or partial out) counts for.
constexpr uint32_t kPieceCost = 2;
// No cut leaves less than this: a short piece's partial costs more than the tiles it takes off another CTA.
constexpr uint32_t kMinPiece = 4;

}  // namespace

void tree_work_list(const TreeShape& s, const TreeTables& t, uint32_t max_ctas, TreeWork* out) {
    out->pieces.clear();
    out->splits.clear();
    out->row_split.clear();
    out->cta_off.assign(1, 0);
    out->n_slots = out->slot_rows = 0;
    const uint32_t G = static_cast<uint32_t>(s.H / s.KVH);
    struct Unit {
        TreePiece piece;
        uint32_t tiles;
    };
    std::vector<Unit> units;
    uint64_t total = 0;
    uint32_t token0 = 0;
    for (size_t r = 0; r < s.batch; ++r) {
        const uint32_t draft = t.draft[r];
        const uint64_t rows = static_cast<uint64_t>(draft) * G;
        const uint32_t tiles = (t.prefix[r] + draft + kTreeTile - 1) / kTreeTile;
        // rows spread evenly over the row tiles, whole warps each
        const uint64_t n_rt = (rows + kTreeRows - 1) / kTreeRows;
        const uint32_t per = n_rt ? static_cast<uint32_t>(((rows + n_rt - 1) / n_rt + 31) / 32 * 32) : 0;
        for (uint32_t h = 0; draft && h < s.KVH; ++h)
            for (uint64_t first = 0; first < rows; first += per) {
                TreePiece p{};
                p.kv_head = h;
                p.row_begin = static_cast<uint32_t>(first);
                p.n_rows = static_cast<uint32_t>(std::min<uint64_t>(per, rows - first));
                p.prefix = t.prefix[r];
                p.draft = draft;
                p.token0 = token0;
                p.pt_off = t.pt_off[r];
                p.slot = kTreeNoSlot;
                units.push_back({p, tiles});
                total += tiles + kPieceCost;
                out->slot_rows = std::max(out->slot_rows, p.n_rows);
            }
        token0 += draft;
    }
    if (units.empty() || max_ctas == 0) return;
    uint64_t quota = std::max<uint64_t>((total + max_ctas - 1) / max_ctas, kMinPiece + kPieceCost);
    for (;; quota += quota / 32 + 1) {   // rounding at the cuts may need a CTA more than there are: try again with longer runs
        out->pieces.clear();
        out->splits.clear();
        out->row_split.clear();
        out->cta_off.assign(1, 0);
        out->n_slots = 0;
        uint64_t used = 0;
        auto next_cta = [&] {
            out->cta_off.push_back(static_cast<uint32_t>(out->pieces.size()));
            used = 0;
        };
        for (const Unit& u : units) {
            uint32_t at = 0;
            const size_t first_piece = out->pieces.size();
            while (at < u.tiles) {
                if (used && used + kPieceCost + std::min(kMinPiece, u.tiles - at) > quota) next_cta();
                const uint64_t room = quota - used - kPieceCost;   // >= the smallest piece, see the quota's lower bound
                uint32_t take = static_cast<uint32_t>(std::min<uint64_t>(u.tiles - at, std::max<uint64_t>(room, 1)));
                if (u.tiles - at - take < kMinPiece) take = u.tiles - at;
                TreePiece p = u.piece;
                p.tile_begin = at;
                p.n_tiles = take;
                out->pieces.push_back(p);
                used += take + kPieceCost;
                at += take;
            }
            const size_t n = out->pieces.size() - first_piece;
            if (n > 1) {
                TreeSplit sp{};
                sp.kv_head = u.piece.kv_head;
                sp.row_begin = u.piece.row_begin;
                sp.n_rows = u.piece.n_rows;
                sp.token0 = u.piece.token0;
                sp.first_slot = out->n_slots;
                sp.n_parts = static_cast<uint32_t>(n);
                sp.first_row = static_cast<uint32_t>(out->row_split.size());
                for (size_t i = 0; i < n; ++i) out->pieces[first_piece + i].slot = out->n_slots++;
                out->row_split.insert(out->row_split.end(), u.piece.n_rows, static_cast<uint32_t>(out->splits.size()));
                out->splits.push_back(sp);
            }
        }
        next_cta();
        if (out->cta_off.size() - 1 <= max_ctas) return;
    }
}

}  // namespace mlcb
