// Attention of drafted tokens arranged as a tree over the paged cache: tables on the device, work list, launches.
#pragma once

#include <cstddef>
#include <cstdint>
#include <string>
#include <vector>

#include "ctx.hpp"

namespace mlcb {

// What one call is about, after its tables have been checked.
struct TreeShape {
    size_t batch = 0, H = 0, KVH = 0, D = 0, P = 0, capacity = 0, mask_words = 0;
    size_t n_flat = 0, tokens = 0;   // page-table words, drafted tokens of all requests
};

struct TreeTables {
    const uint32_t* pt_flat = nullptr;
    const uint32_t* pt_off = nullptr;
    const uint32_t* prefix = nullptr;   // committed tokens of a request
    const uint32_t* draft = nullptr;    // its drafted tokens, at positions prefix ...
    const uint32_t* mask = nullptr;     // [tokens][mask_words]
};

static constexpr uint32_t kTreeTile = 64;           // tokens of the cache per step of the tensor-core kernel
static constexpr uint32_t kTreeRows = 128;          // query rows (drafted token, head of the group) of a row tile
static constexpr uint32_t kTreeNoSlot = 0xFFFFFFFFu;

// A run of cache tiles of one (request, KV head, row tile), worked off by one CTA.
struct TreePiece {
    uint32_t kv_head, row_begin, n_rows;   // rows of the unit, row = drafted token * group + head of the group
    uint32_t tile_begin, n_tiles;
    uint32_t slot;                         // where the partial goes; kTreeNoSlot: the piece is the whole run
    uint32_t prefix, draft, token0, pt_off;
    uint32_t more, next;                   // first piece of a CTA: it has `more` others, from pieces[next] on
};
static_assert(sizeof(TreePiece) == 48, "read as three 16-byte vectors");

// A row tile whose run was cut: part k lies in slot first_slot + k * slot_step.
struct TreeSplit {
    uint32_t kv_head, row_begin, n_rows, token0, first_slot, n_parts, first_row, slot_step;
};
static_assert(sizeof(TreeSplit) == 32, "read as two 16-byte vectors");

struct TreeWork {
    std::vector<TreePiece> pieces;    // the first piece of every CTA, then the others, CTA by CTA
    uint32_t n_cta = 0;
    std::vector<TreeSplit> splits;
    std::vector<uint32_t> row_split;  // split of every merged row
    uint32_t n_slots = 0, slot_rows = 0, max_parts = 0;
};

struct TreeWorkView {   // a work list on the device
    const TreePiece* pieces = nullptr;
    const TreeSplit* splits = nullptr;
    const uint32_t* row_split = nullptr;
    uint32_t n_cta = 0, n_slots = 0, slot_rows = 0, merge_rows = 0, max_parts = 0;
};

// The tensor-core kernel runs two CTAs per SM, with fp32 queries or outputs and head_dim 128 one: a call with its tables in a
// plan may be either, so head_dim 128 has two lists.
static constexpr uint32_t kTreeLists = 2;   // [0]: two CTAs per SM, [1]: one
struct TreeWorks {
    TreeWork list[kTreeLists];
};

struct TreeView {   // device addresses inside one image
    const uint32_t *pt_flat = nullptr, *pt_off = nullptr, *prefix = nullptr, *draft = nullptr, *mask = nullptr;
    const uint32_t *token0 = nullptr;     // first drafted token of a request in q / o, [batch + 1]
    const uint32_t* token_req = nullptr;  // request of a drafted token
    TreeWorkView work[kTreeLists];
};

struct TreeArgs {
    const void* q = nullptr;
    const void* k_pages = nullptr;
    const void* v_pages = nullptr;
    void* o = nullptr;
    float scale = 0.f;
    int q_dtype = MLC_F16, o_dtype = MLC_F16;
};

// Whether the tensor-core kernel takes this shape: head_dim 64 or 128, pages of 16, 32 or a multiple of 64 tokens, a pool of
// known size; and these buffers.
bool tree_tcgen05_shape(const TreeShape& s);
bool tree_tcgen05_buffers(const TreeArgs& a);
// Cuts the units of a call into pieces for `max_ctas` CTAs (host arithmetic only).
void tree_work_list(const TreeShape& s, const TreeTables& t, uint32_t max_ctas, TreeWork* out);
// Device scratch for the partials of cut units.
size_t tree_scratch_bytes(const TreeShape& s, uint32_t n_slots, uint32_t slot_rows);

int launch_tree_tcgen05(mlc_ctx* ctx, const TreeShape& s, const TreeView& v, const TreeArgs& a);
int launch_tree_general(mlc_ctx* ctx, const TreeShape& s, const TreeView& v, const TreeArgs& a);

}  // namespace mlcb
