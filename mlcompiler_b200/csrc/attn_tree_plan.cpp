// Work list of the tensor-core kernel of tree attention (host arithmetic only).
//
// A unit is what shares K and V: (request, KV head). Its query rows (drafted token, head of the group) make one or more row
// tiles of up to 128 rows, each the business of a CTA of its own; the CTAs of a unit's row tiles get the same run of cache
// tiles, so that they read it side by side and all but one of them from L2. Units with the same number of row tiles are laid
// end to end and cut into equal runs, one per group of CTAs: every CTA gets the same number of cache tiles whatever the
// spread of context lengths. A unit cut between groups leaves partials that a second kernel joins.
// (Row tiles dealt as units of their own: 16 requests x 64 drafted tokens over 12-30 thousand tokens, two row tiles each,
// read 1.9 times the cache from memory and took 474 us.)
#include <algorithm>

#include "attn_tree.hpp"

namespace mlcb {

namespace {

// Tiles a piece's fixed work (queries in, output or partial out) counts for: 32 requests of 1 to 4095 tokens take 32.7 us
// with 3, 32.0 with 4, 31.7 with 5.
constexpr uint32_t kPieceCost = 5;
// No cut leaves less than this. One request of 1000 tokens, 8 drafted: 7.7 us with 2, 8.6 with 4.
constexpr uint32_t kMinPiece = 2;
// Where every run has a CTA of its own and none is longer than this, nothing is cut: the second kernel costs more than
// the tiles it saves. 16 requests of 300 tokens (5 tiles): 8.0 us whole, 9.4 cut; of 500 (8 tiles): 10.5 whole, 9.1 cut.
constexpr uint32_t kWholeTiles = 6;
constexpr uint32_t kLanes = 8;

}  // namespace

void tree_work_list(const TreeShape& s, const TreeTables& t, uint32_t max_ctas, TreeWork* out) {
    out->pieces.clear();
    out->splits.clear();
    out->row_split.clear();
    out->n_cta = out->n_slots = out->slot_rows = out->max_parts = 0;
    const uint32_t G = static_cast<uint32_t>(s.H / s.KVH);
    // Row tiles side by side, at most: beyond, they share a run through L2 in turns. One where there are too few CTAs for
    // a group of every width.
    const uint32_t max_lanes = max_ctas >= kLanes * (kLanes + 1) / 2 ? kLanes : 1;
    struct Unit {
        TreePiece piece;          // rows of the first row tile
        uint32_t tiles, lanes;    // cache tiles, row tiles side by side
        uint32_t rows, per;       // rows of all of them, rows of a full one
    };
    std::vector<Unit> units[kLanes + 1];
    uint64_t total = 0, n_lanes = 0;
    uint32_t token0 = 0, longest = 0;
    for (size_t r = 0; r < s.batch; ++r) {
        const uint32_t draft = t.draft[r];
        const uint64_t rows = static_cast<uint64_t>(draft) * G;
        const uint32_t tiles = (t.prefix[r] + draft + kTreeTile - 1) / kTreeTile;
        // rows spread evenly over the row tiles, whole warps each
        const uint64_t n_rt = (rows + kTreeRows - 1) / kTreeRows;
        const uint32_t per = n_rt ? static_cast<uint32_t>(((rows + n_rt - 1) / n_rt + 31) / 32 * 32) : 0;
        for (uint32_t h = 0; draft && h < s.KVH; ++h)
            for (uint64_t first = 0; first < rows; first += static_cast<uint64_t>(per) * max_lanes) {
                Unit u{};
                u.rows = static_cast<uint32_t>(std::min<uint64_t>(static_cast<uint64_t>(per) * max_lanes, rows - first));
                u.per = per;
                u.lanes = (u.rows + per - 1) / per;
                u.tiles = tiles;
                u.piece.kv_head = h;
                u.piece.row_begin = static_cast<uint32_t>(first);
                u.piece.prefix = t.prefix[r];
                u.piece.draft = draft;
                u.piece.token0 = token0;
                u.piece.pt_off = t.pt_off[r];
                u.piece.slot = kTreeNoSlot;
                units[u.lanes].push_back(u);
                total += static_cast<uint64_t>(tiles + kPieceCost) * u.lanes;
                n_lanes += u.lanes;
                longest = std::max(longest, tiles);
                out->slot_rows = std::max(out->slot_rows, std::min(per, u.rows));
            }
        token0 += draft;
    }
    if (total == 0 || max_ctas == 0) return;
    std::vector<std::vector<TreePiece>> ctas;
    uint64_t quota = std::max<uint64_t>((total + max_ctas - 1) / max_ctas, kPieceCost + 1);
    if (n_lanes <= max_ctas && longest <= kWholeTiles) quota = std::max<uint64_t>(quota, longest + kPieceCost);
    for (;; quota += quota / 32 + 1) {   // rounding at the cuts may need a CTA more than there are: try again with longer runs
        ctas.clear();
        out->splits.clear();
        out->row_split.clear();
        out->n_slots = out->max_parts = 0;
        std::vector<std::vector<TreePiece>> group;   // pieces of the CTAs of the current group
        uint64_t used = 0;
        auto close_group = [&] {
            for (auto& lane : group) {
                ctas.push_back(std::move(lane));
                lane.clear();
            }
            used = 0;
        };
        for (uint32_t lanes = kLanes; lanes >= 1; --lanes) {
            if (units[lanes].empty()) continue;
            group.assign(lanes, {});
            for (const Unit& u : units[lanes]) {
                uint32_t at = 0, n_parts = 0;
                const uint32_t first_slot = out->n_slots;
                while (at < u.tiles) {
                    if (used && used + kPieceCost + std::min(kMinPiece, u.tiles - at) > quota) close_group();
                    const uint64_t room = std::max<uint64_t>(quota - used - kPieceCost, kMinPiece);
                    uint32_t take = static_cast<uint32_t>(std::min<uint64_t>(u.tiles - at, room));
                    if (u.tiles - at - take < kMinPiece) take = u.tiles - at;
                    const bool cut = at || take < u.tiles;
                    for (uint32_t i = 0; i < lanes; ++i) {
                        TreePiece p = u.piece;
                        p.row_begin += i * u.per;
                        p.n_rows = std::min(u.per, u.rows - i * u.per);
                        p.tile_begin = at;
                        p.n_tiles = take;
                        if (cut) p.slot = first_slot + n_parts * lanes + i; 
                        group[i].push_back(p);
                    }
                    n_parts += cut;
                    used += take + kPieceCost;
                    at += take;
                }
                if (n_parts == 0) continue;
                for (uint32_t i = 0; i < lanes; ++i) {
                    TreeSplit sp{};
                    sp.kv_head = u.piece.kv_head;
                    sp.row_begin = u.piece.row_begin + i * u.per;
                    sp.n_rows = std::min(u.per, u.rows - i * u.per);
                    sp.token0 = u.piece.token0;
                    sp.first_slot = first_slot + i;
                    sp.n_parts = n_parts;
                    sp.slot_step = lanes;
                    sp.first_row = static_cast<uint32_t>(out->row_split.size());
                    out->row_split.insert(out->row_split.end(), sp.n_rows, static_cast<uint32_t>(out->splits.size()));
                    out->splits.push_back(sp);
                }
                out->n_slots += n_parts * lanes;
                out->max_parts = std::max(out->max_parts, n_parts);
            }
            if (used) close_group();
        }
        if (ctas.size() <= max_ctas) break;
    }
    out->n_cta = static_cast<uint32_t>(ctas.size());
    uint32_t next = out->n_cta;
    for (const auto& c : ctas) {
        out->pieces.push_back(c.front());
        out->pieces.back().more = static_cast<uint32_t>(c.size() - 1);
        out->pieces.back().next = next;
        next += static_cast<uint32_t>(c.size() - 1);
    }
    for (const auto& c : ctas) out->pieces.insert(out->pieces.end(), c.begin() + 1, c.end());
}

}  // namespace mlcb
