// Copies inside the paged pools: whole pages (a forked request gets its own copy of a shared page) and rows of accepted
// drafted tokens (they move up behind the committed ones). Byte movement, bit-exact; the K and V pools of every layer go
// in one launch.
//
// The reference gives every request its own pages for good (compiler/runtime/paged_kv.cpp:44-81) and has no
// counterpart; page and row layout are its (paged_kv.hpp:101-105).
//
// What bounds them: a call reads and writes every byte once, so the copy bandwidth of the memory for large calls (121 pages
// from 80 different ones in 64 pools, 1690 MB in and out: 255 us on the device) and one launch for small ones (three pages in
// 44 pools: 1.9 us on the device, 5 with the host's part; rows of 32 requests in 64 pools, 20 MB: 4.3 and 10). That is why the
// pools' addresses and short id lists travel as kernel parameters: an upload in front of the kernel costs about as much as the
// kernel itself.
#include <algorithm>
#include <cstring>

#include "op_util.hpp"

namespace mlcb {

namespace {

constexpr uint32_t kMaxPools = 128;      // per launch; a call with more takes several
// (source, destination) pairs that travel as kernel parameters: a kernel with few, since parameters cost the host's launch time, and
// one with many (121 page pairs: 255.6 us, uploaded 259.7; 32 requests' rows: 9.9 us and 4.3 on the device, uploaded 11.9 and 9.5)
constexpr uint32_t kFewPairs = 16, kManyPairs = 240;

template <uint32_t INLINE>
struct CopyParams {
    char* pools[kMaxPools];
    const uint2* pairs;                  // device list, or null: `inline_pairs`
    uint2 inline_pairs[INLINE];
    uint64_t unit_bytes;                 // a page, or a row
    uint32_t n_pairs;
};

constexpr uint32_t kBatch = 8;   // vectors a thread has in flight

// Launched as a programmatic dependent of the kernel in front; it does not let its own dependents go before it is done, so
// that nothing behind it reads a page early.
template <typename Vec, uint32_t INLINE>
__global__ void __launch_bounds__(256) copy_pages_kernel(const __grid_constant__ CopyParams<INLINE> p, uint32_t chunks) {
    const uint32_t pair_i = blockIdx.x / chunks, chunk = blockIdx.x - pair_i * chunks;
    const uint2 pair = p.pairs ? p.pairs[pair_i] : p.inline_pairs[pair_i];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (pair.x == pair.y) return;
    char* pool = p.pools[blockIdx.y];
    const Vec* src = reinterpret_cast<const Vec*>(pool + static_cast<uint64_t>(pair.x) * p.unit_bytes);
    Vec* dst = reinterpret_cast<Vec*>(pool + static_cast<uint64_t>(pair.y) * p.unit_bytes);
    const uint64_t n = p.unit_bytes / sizeof(Vec), first = static_cast<uint64_t>(chunk) * (256 * kBatch) + threadIdx.x;
    Vec v[kBatch];
#pragma unroll
    for (uint32_t i = 0; i < kBatch; ++i)
        if (first + 256 * i < n) v[i] = src[first + 256 * i];
#pragma unroll
    for (uint32_t i = 0; i < kBatch; ++i)
        if (first + 256 * i < n) dst[first + 256 * i] = v[i];
}

// Rows of one request move from rising source rows to rising destination rows, never upwards (destination <= source in
// token order). A thread owns one column of the row in one pool and works through the request's moves in order, so a row
// is always read before a later move can write it, whatever the other threads do. It has kBatch rows in flight: the rows it has not
// read yet lie behind every destination of the batch.
template <uint32_t INLINE>
struct MoveParams {
    char* pools[kMaxPools];
    const uint2* moves;                  // device list, or null: `inline_moves`
    const uint32_t* first;               // [n_requests + 1] first move of a request, or null: `inline_first`
    uint2 inline_moves[INLINE];
    uint32_t inline_first[INLINE + 1];
    uint64_t row_bytes;
    uint32_t n_requests;
};

template <typename Vec, uint32_t INLINE>
__global__ void __launch_bounds__(128) move_rows_kernel(const __grid_constant__ MoveParams<INLINE> p, uint32_t vecs, uint64_t threads) {
    const uint64_t id = static_cast<uint64_t>(blockIdx.x) * 128 + threadIdx.x;
    if (id >= threads) return;
    const uint32_t req = static_cast<uint32_t>(id / vecs), column = static_cast<uint32_t>(id - static_cast<uint64_t>(req) * vecs);
    char* pool = p.pools[blockIdx.y] + static_cast<uint64_t>(column) * sizeof(Vec);
    const uint32_t* first = p.first ? p.first : p.inline_first;
    const uint2* moves = p.moves ? p.moves : p.inline_moves;
    const uint32_t end = first[req + 1];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (uint32_t i = first[req]; i < end; i += kBatch) {
        Vec v[kBatch];
        uint32_t to[kBatch];
#pragma unroll
        for (uint32_t k = 0; k < kBatch; ++k)
            if (i + k < end) {
                const uint2 m = moves[i + k];
                to[k] = m.y;
                v[k] = *reinterpret_cast<const Vec*>(pool + m.x * p.row_bytes);
            }
#pragma unroll
        for (uint32_t k = 0; k < kBatch; ++k)
            if (i + k < end) *reinterpret_cast<Vec*>(pool + to[k] * p.row_bytes) = v[k];
    }
}

// The widest vector (16, 8, 4 or 2 bytes) that divides the unit and the pools' addresses.
uint32_t vector_bytes(void* const* pools, size_t n_pools, uint64_t unit_bytes) {
    uint64_t bits = unit_bytes;
    for (size_t i = 0; i < n_pools; ++i) bits |= reinterpret_cast<uintptr_t>(pools[i]);
    uint32_t v = 16;
    while (v > 2 && bits % v != 0) v /= 2;
    return v;
}

int check_pools(mlc_ctx* ctx, void* const* pools, size_t n_pools, size_t P, size_t KVH, size_t D, size_t dtype_bytes) {
    if (!pools) return ctx->fail(MLC_ERR_INVALID_ARG, "null argument");
    if (n_pools == 0 || P == 0 || KVH == 0 || D == 0) return ctx->fail(MLC_ERR_INVALID_ARG, "zero dimension");
    if (dtype_bytes != 2 && dtype_bytes != 4) return ctx->fail(MLC_ERR_INVALID_ARG, "dtype_bytes must be 2 or 4");
    if (KVH >= (size_t(1) << 20) || D >= (size_t(1) << 20) || P >= (size_t(1) << 40) / (KVH * D))
        return ctx->fail(MLC_ERR_UNSUPPORTED, "dimension too large");
    const void* few[256];
    std::vector<const void*> many;
    const void** sorted = few;
    if (n_pools > 256) {
        many.resize(n_pools);
        sorted = many.data();
    }
    std::copy(pools, pools + n_pools, sorted);
    std::sort(sorted, sorted + n_pools);
    if (!sorted[0]) return ctx->fail(MLC_ERR_INVALID_ARG, "null pool");
    for (size_t i = 0; i < n_pools; ++i) {
        if (i && sorted[i] == sorted[i - 1]) return ctx->fail(MLC_ERR_INVALID_ARG, "a pool is named twice");
        if (!aligned_to(sorted[i], dtype_bytes)) return ctx->fail(MLC_ERR_INVALID_ARG, "a pool is not aligned to its elements");
    }
    return MLC_OK;
}

// Pages a call may name: the caller's claim, or what the smallest of the pools allocated by this context holds.
size_t pools_capacity(mlc_ctx* ctx, void* const* pools, size_t n_pools, size_t claimed, size_t page_bytes) {
    if (claimed) return claimed;
    size_t cap = 0;
    for (size_t i = 0; i < n_pools; ++i) {
        const size_t c = resolve_capacity(ctx, pools[i], 0, page_bytes);
        if (c && (!cap || c < cap)) cap = c;
    }
    return cap;
}

// Owner of every page that the current call names. Ids below 2^20 have an entry in a table of the context that a newer
// call's number makes stale; larger ones (a pool that large is rare) go to a map.
class PageOwners {
public:
    explicit PageOwners(mlc_ctx* ctx) : table_(ctx->page_marks) {
        if (++ctx->page_mark >> 32) {   // the numbers are used up: forget all entries
            std::fill(table_.begin(), table_.end(), 0);
            ctx->page_mark = 1;
        }
        call_ = ctx->page_mark;
    }
    // The owner noted for `id`, noting `owner` if there is none yet.
    uint32_t claim(uint32_t id, uint32_t owner) {
        if (id >= kTable) return map_.emplace(id, owner).first->second;
        if (id >= table_.size()) table_.resize(static_cast<size_t>(id) + id / 2 + 64, 0);
        uint64_t& e = table_[id];
        if ((e >> 32) != call_) e = (call_ << 32) | owner;
        return static_cast<uint32_t>(e);
    }
    bool known(uint32_t id) const {
        if (id >= kTable) return map_.count(id) != 0;
        return id < table_.size() && (table_[id] >> 32) == call_;
    }

private:
    static constexpr uint32_t kTable = 1u << 20;
    std::vector<uint64_t>& table_;
    uint64_t call_;
    std::unordered_map<uint32_t, uint32_t> map_;
};

int wait_for_copy(mlc_ctx* ctx, const char* what) {
    const cudaError_t e = cudaStreamSynchronize(ctx->stream);
    if (!ctx->pass_open) stage_reset(ctx);
    if (e != cudaSuccess) return ctx->fail(MLC_ERR_CUDA, "%s failed: %s", what, cudaGetErrorString(e));
    return MLC_OK;
}

template <uint32_t INLINE>
int launch_copies(mlc_ctx* ctx, void* const* pools, size_t n_pools, const uint32_t* src, const uint32_t* dst, size_t n_pairs,
                  uint64_t page_bytes) {
    std::vector<uint2> list;
    CopyParams<INLINE> p{};
    uint2* to = p.inline_pairs;
    if (n_pairs > INLINE) {
        list.resize(n_pairs);
        to = list.data();
    }
    for (size_t i = 0; i < n_pairs; ++i) to[i] = make_uint2(src[i], dst[i]);
    p.unit_bytes = page_bytes;
    p.n_pairs = static_cast<uint32_t>(n_pairs);
    const uint32_t vec = vector_bytes(pools, n_pools, page_bytes);
    const uint64_t chunks = (page_bytes / vec + 256 * kBatch - 1) / (256 * kBatch);
    if (chunks * n_pairs >= (uint64_t(1) << 31)) return ctx->fail(MLC_ERR_UNSUPPORTED, "too many pages in one call");
    if (n_pairs > INLINE && !(p.pairs = static_cast<const uint2*>(stage_to_device(ctx, list.data(), n_pairs * sizeof(uint2)))))
        return MLC_ERR_OOM;
    for (size_t p0 = 0; p0 < n_pools; p0 += kMaxPools) {
        const size_t n = n_pools - p0 < kMaxPools ? n_pools - p0 : kMaxPools;
        for (size_t i = 0; i < n; ++i) p.pools[i] = static_cast<char*>(pools[p0 + i]);
        const dim3 grid(static_cast<unsigned>(chunks * n_pairs), static_cast<unsigned>(n));
        const uint32_t c = static_cast<uint32_t>(chunks);
        cudaError_t e;
        switch (vec) {
            case 16: e = launch_dependent(ctx, copy_pages_kernel<uint4, INLINE>, grid, 256, 0, p, c); break;
            case 8: e = launch_dependent(ctx, copy_pages_kernel<uint2, INLINE>, grid, 256, 0, p, c); break;
            case 4: e = launch_dependent(ctx, copy_pages_kernel<uint32_t, INLINE>, grid, 256, 0, p, c); break;
            default: e = launch_dependent(ctx, copy_pages_kernel<uint16_t, INLINE>, grid, 256, 0, p, c); break;
        }
        MLCB_CUDA(ctx, e);
        ++ctx->launches;
    }
    return MLC_OK;
}

template <uint32_t INLINE>
int launch_moves(mlc_ctx* ctx, void* const* pools, size_t n_pools, const std::vector<uint2>& moves, const std::vector<uint32_t>& first,
                 uint64_t row_bytes) {
    const size_t n_requests = first.size() - 1;
    const uint32_t vec = vector_bytes(pools, n_pools, row_bytes);
    const uint64_t vecs = row_bytes / vec, threads = vecs * n_requests;
    if (vecs >> 32 || (threads + 127) / 128 >= (uint64_t(1) << 31)) return ctx->fail(MLC_ERR_UNSUPPORTED, "rows too long");
    MoveParams<INLINE> p{};
    if (moves.size() <= INLINE) {
        std::memcpy(p.inline_moves, moves.data(), moves.size() * sizeof(uint2));
        std::memcpy(p.inline_first, first.data(), first.size() * 4);
    } else {
        std::vector<uint32_t> image(moves.size() * 2 + first.size());
        std::memcpy(image.data(), moves.data(), moves.size() * sizeof(uint2));
        std::memcpy(image.data() + moves.size() * 2, first.data(), first.size() * 4);
        const void* d = stage_to_device(ctx, image.data(), image.size() * 4);
        if (!d) return MLC_ERR_OOM;
        p.moves = static_cast<const uint2*>(d);
        p.first = static_cast<const uint32_t*>(d) + moves.size() * 2;
    }
    p.row_bytes = row_bytes;
    p.n_requests = static_cast<uint32_t>(n_requests);
    for (size_t p0 = 0; p0 < n_pools; p0 += kMaxPools) {
        const size_t n = n_pools - p0 < kMaxPools ? n_pools - p0 : kMaxPools;
        for (size_t i = 0; i < n; ++i) p.pools[i] = static_cast<char*>(pools[p0 + i]);
        const dim3 grid(static_cast<unsigned>((threads + 127) / 128), static_cast<unsigned>(n));
        const uint32_t v = static_cast<uint32_t>(vecs);
        cudaError_t e;
        switch (vec) {
            case 16: e = launch_dependent(ctx, move_rows_kernel<uint4, INLINE>, grid, 128, 0, p, v, threads); break;
            case 8: e = launch_dependent(ctx, move_rows_kernel<uint2, INLINE>, grid, 128, 0, p, v, threads); break;
            case 4: e = launch_dependent(ctx, move_rows_kernel<uint32_t, INLINE>, grid, 128, 0, p, v, threads); break;
            default: e = launch_dependent(ctx, move_rows_kernel<uint16_t, INLINE>, grid, 128, 0, p, v, threads); break;
        }
        MLCB_CUDA(ctx, e);
        ++ctx->launches;
    }
    return MLC_OK;
}

int copy_pages(mlc_ctx* ctx, bool sync, void* const* pools, size_t n_pools, const uint32_t* src, const uint32_t* dst,
               size_t n_pairs, size_t P, size_t KVH, size_t D, size_t dtype_bytes, size_t capacity_pages) {
    if (!ctx) return MLC_ERR_INVALID_ARG;
    int st = check_pools(ctx, pools, n_pools, P, KVH, D, dtype_bytes);
    if (st != MLC_OK) return st;
    if (!sync && !ctx->pass_open) return ctx->fail(MLC_ERR_NO_OPEN_PASS, "encode without an open pass");
    if (ctx->capturing) return ctx->fail(MLC_ERR_UNSUPPORTED, "host page ids inside a graph capture");
    if (n_pairs == 0) return MLC_OK;
    if (!src || !dst) return ctx->fail(MLC_ERR_INVALID_ARG, "null argument");
    const uint64_t page_bytes = static_cast<uint64_t>(P) * KVH * D * dtype_bytes;
    const size_t cap = pools_capacity(ctx, pools, n_pools, capacity_pages, page_bytes);
    if (n_pairs >= (size_t(1) << 32)) return ctx->fail(MLC_ERR_UNSUPPORTED, "too many pages in one call");
    PageOwners destinations(ctx);
    for (size_t i = 0; i < n_pairs; ++i) {
        for (const uint32_t id : {src[i], dst[i]})
            if (cap && id >= cap) return ctx->fail(MLC_ERR_BOUNDS, "page id %u of pair %zu >= capacity %zu", id, i, cap);
        if (src[i] != dst[i] && destinations.claim(dst[i], static_cast<uint32_t>(i)) != i)
            return ctx->fail(MLC_ERR_INVALID_ARG, "page %u is the destination of two pairs", dst[i]);
    }
    for (size_t i = 0; i < n_pairs; ++i)
        if (src[i] != dst[i] && destinations.known(src[i]))
            return ctx->fail(MLC_ERR_INVALID_ARG, "page %u is a source and a destination", src[i]);
    DeviceGuard guard(ctx->device);
    st = n_pairs <= kFewPairs ? launch_copies<kFewPairs>(ctx, pools, n_pools, src, dst, n_pairs, page_bytes)
                              : launch_copies<kManyPairs>(ctx, pools, n_pools, src, dst, n_pairs, page_bytes);
    if (st != MLC_OK) return st;
    note_pool_writes(ctx, pools, n_pools);
    return sync ? wait_for_copy(ctx, "page copy") : MLC_OK;
}

int compact_rows(mlc_ctx* ctx, bool sync, void* const* pools, size_t n_pools, const uint32_t* pt_flat, size_t n_flat,
                 const uint32_t* pt_off, const uint32_t* start, const uint32_t* kept, const uint32_t* kept_off, size_t batch,
                 size_t P, size_t KVH, size_t D, size_t dtype_bytes, size_t capacity_pages) {
    if (!ctx) return MLC_ERR_INVALID_ARG;
    int st = check_pools(ctx, pools, n_pools, P, KVH, D, dtype_bytes);
    if (st != MLC_OK) return st;
    if (batch == 0) return ctx->fail(MLC_ERR_INVALID_ARG, "zero dimension");
    if (!pt_off || !start || !kept_off || (!pt_flat && n_flat)) return ctx->fail(MLC_ERR_INVALID_ARG, "null table");
    if (!sync && !ctx->pass_open) return ctx->fail(MLC_ERR_NO_OPEN_PASS, "encode without an open pass");
    if (ctx->capturing) return ctx->fail(MLC_ERR_UNSUPPORTED, "host tables inside a graph capture");
    for (size_t r = 0; r < batch; ++r) {
        if (pt_off[r + 1] < pt_off[r]) return ctx->fail(MLC_ERR_BOUNDS, "page_table_offsets not monotone at %zu", r);
        if (kept_off[r + 1] < kept_off[r]) return ctx->fail(MLC_ERR_BOUNDS, "kept_offsets not monotone at %zu", r);
    }
    if (n_flat < pt_off[batch]) return ctx->fail(MLC_ERR_INVALID_ARG, "page_tables_flat shorter than the last offset");
    if (kept_off[batch] > kept_off[0] && !kept) return ctx->fail(MLC_ERR_INVALID_ARG, "null table");
    const uint64_t row_bytes = static_cast<uint64_t>(KVH) * D * dtype_bytes;
    const size_t cap = pools_capacity(ctx, pools, n_pools, capacity_pages, P * row_bytes);
    std::vector<uint2> moves;
    std::vector<uint32_t> first(1, 0);
    PageOwners owners(ctx);
    for (size_t r = 0; r < batch; ++r) {
        const uint32_t* table = pt_flat + pt_off[r];
        const uint64_t room = static_cast<uint64_t>(pt_off[r + 1] - pt_off[r]) * P;
        const uint32_t n = kept_off[r + 1] - kept_off[r];
        const uint32_t* list = kept + kept_off[r];
        for (uint32_t i = 0; i < n; ++i) {
            if (i && list[i] <= list[i - 1]) return ctx->fail(MLC_ERR_INVALID_ARG, "kept rows of request %zu do not rise", r);
            const uint64_t from = static_cast<uint64_t>(start[r]) + list[i], to = static_cast<uint64_t>(start[r]) + i;
            if (from >= room)
                return ctx->fail(MLC_ERR_BOUNDS, "kept row %u of request %zu lies behind its %u pages", list[i], r, pt_off[r + 1] - pt_off[r]);
            if (from == to) continue;
            const uint32_t src_page = table[from / P], dst_page = table[to / P];
            for (const uint64_t pos : {from, to}) {
                const uint32_t at = static_cast<uint32_t>(pos / P), id = table[at];
                if (cap && id >= cap)
                    return ctx->fail(MLC_ERR_BOUNDS, "page id %u of request %zu >= capacity %zu", id, r, cap);
                // The requests run side by side: none may touch a page whose rows another one moves. Nor may a page stand twice in
                // a table: a row could be read after it has been written under its other position.
                if (owners.claim(id, pt_off[r] + at) != pt_off[r] + at)
                    return ctx->fail(MLC_ERR_INVALID_ARG, "rows of page %u move in two places of the page tables, one of them request %zu's", id, r);
            }
            const uint64_t src_row = src_page * static_cast<uint64_t>(P) + from % P, dst_row = dst_page * static_cast<uint64_t>(P) + to % P;
            if ((src_row | dst_row) >> 32) return ctx->fail(MLC_ERR_UNSUPPORTED, "pool of 2^32 rows or more");
            moves.push_back(make_uint2(static_cast<uint32_t>(src_row), static_cast<uint32_t>(dst_row)));
        }
        // a request that moves nothing takes no thread
        if (moves.size() > first.back()) first.push_back(static_cast<uint32_t>(moves.size()));
    }
    if (moves.empty()) return MLC_OK;
    DeviceGuard guard(ctx->device);
    st = moves.size() <= kFewPairs ? launch_moves<kFewPairs>(ctx, pools, n_pools, moves, first, row_bytes)
                                   : launch_moves<kManyPairs>(ctx, pools, n_pools, moves, first, row_bytes);
    if (st != MLC_OK) return st;
    note_pool_writes(ctx, pools, n_pools);
    return sync ? wait_for_copy(ctx, "row compaction") : MLC_OK;
}

}  // namespace

}  // namespace mlcb

using namespace mlcb;

extern "C" {

int mlc_run_copy_kv_pages(mlc_ctx* ctx, void* const* pools, size_t n_pools, const uint32_t* src_page_ids,
                          const uint32_t* dst_page_ids, size_t n_pairs, size_t page_size_tokens, size_t n_kv_heads,
                          size_t head_dim, size_t dtype_bytes, size_t capacity_pages) {
    return no_throw(ctx, [&] {
        return copy_pages(ctx, true, pools, n_pools, src_page_ids, dst_page_ids, n_pairs, page_size_tokens, n_kv_heads, head_dim,
                          dtype_bytes, capacity_pages);
    });
}

int mlc_encode_copy_kv_pages(mlc_ctx* ctx, void* const* pools, size_t n_pools, const uint32_t* src_page_ids,
                             const uint32_t* dst_page_ids, size_t n_pairs, size_t page_size_tokens, size_t n_kv_heads,
                             size_t head_dim, size_t dtype_bytes, size_t capacity_pages) {
    return no_throw(ctx, [&] {
        return copy_pages(ctx, false, pools, n_pools, src_page_ids, dst_page_ids, n_pairs, page_size_tokens, n_kv_heads, head_dim,
                          dtype_bytes, capacity_pages);
    });
}

int mlc_run_compact_kv_rows(mlc_ctx* ctx, void* const* pools, size_t n_pools, const uint32_t* page_tables_flat,
                            size_t n_page_tables_flat, const uint32_t* page_table_offsets, const uint32_t* start_positions,
                            const uint32_t* kept_rows, const uint32_t* kept_offsets, size_t batch, size_t page_size_tokens,
                            size_t n_kv_heads, size_t head_dim, size_t dtype_bytes, size_t capacity_pages) {
    return no_throw(ctx, [&] {
        return compact_rows(ctx, true, pools, n_pools, page_tables_flat, n_page_tables_flat, page_table_offsets, start_positions,
                            kept_rows, kept_offsets, batch, page_size_tokens, n_kv_heads, head_dim, dtype_bytes, capacity_pages);
    });
}

int mlc_encode_compact_kv_rows(mlc_ctx* ctx, void* const* pools, size_t n_pools, const uint32_t* page_tables_flat,
                               size_t n_page_tables_flat, const uint32_t* page_table_offsets, const uint32_t* start_positions,
                               const uint32_t* kept_rows, const uint32_t* kept_offsets, size_t batch, size_t page_size_tokens,
                               size_t n_kv_heads, size_t head_dim, size_t dtype_bytes, size_t capacity_pages) {
    return no_throw(ctx, [&] {
        return compact_rows(ctx, false, pools, n_pools, page_tables_flat, n_page_tables_flat, page_table_offsets, start_positions,
                            kept_rows, kept_offsets, batch, page_size_tokens, n_kv_heads, head_dim, dtype_bytes, capacity_pages);
    });
}

}  // extern "C"
