// Entry points of tree attention: the attention of a request's drafted tokens - a tree of continuations of its committed
// tokens, as a speculative decoder verifies them in one pass - over the paged cache.
//
// The reference decodes one continuation per request, one token per pass (compiler/runtime/batched_walker.cpp:299-331);
// these entry points stand beside its paged attention (metal_runtime.hpp:510-523) with its tables and page layout. The
// drafted tokens' K / V rows are scattered into the pages first, in the reference's order scatter -> attention.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <new>

#include "attn_tree.hpp"
#include "op_util.hpp"

using namespace mlcb;

// The tables of one pass on the device, used by the calls of all its layers.
struct mlc_tree_plan {
    mlc_ctx* ctx = nullptr;
    TreeShape shape;
    TreeView view;
    uint8_t* host = nullptr;   // pinned image
    uint8_t* dev = nullptr;
    size_t cap = 0;
    cudaEvent_t uploaded = nullptr;
    bool ready = false;   // the image of `view` is on its way to the device
    mutable bool captured = false;
};

namespace {

size_t align16(size_t v) { return (v + 15) / 16 * 16; }

// Offsets of an image's parts.
struct TreeLayout {
    size_t flat, off, prefix, draft, token0, token_req, mask, total;
    size_t pieces[kTreeLists], splits[kTreeLists], row_split[kTreeLists];
};

TreeLayout layout_of(const TreeShape& s, const TreeWorks& w) {
    TreeLayout l{};
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at = align16(at + bytes);
        return here;
    };
    for (uint32_t i = 0; i < kTreeLists; ++i) {
        l.pieces[i] = take(w.list[i].pieces.size() * sizeof(TreePiece));
        l.splits[i] = take(w.list[i].splits.size() * sizeof(TreeSplit));
        l.row_split[i] = take(w.list[i].row_split.size() * 4);
    }
    l.flat = take(s.n_flat * 4);
    l.off = take((s.batch + 1) * 4);
    l.prefix = take(s.batch * 4);
    l.draft = take(s.batch * 4);
    l.token0 = take((s.batch + 1) * 4);
    l.token_req = take(s.tokens * 4);
    l.mask = take(s.tokens * s.mask_words * 4);
    l.total = std::max<size_t>(at, 16);
    return l;
}

void put(uint8_t* at, const void* src, size_t bytes) {
    if (bytes) std::memcpy(at, src, bytes);
}

void fill_image(uint8_t* h, const TreeLayout& l, const TreeShape& s, const TreeTables& t, const TreeWorks& w) {
    for (uint32_t i = 0; i < kTreeLists; ++i) {
        put(h + l.pieces[i], w.list[i].pieces.data(), w.list[i].pieces.size() * sizeof(TreePiece));
        put(h + l.splits[i], w.list[i].splits.data(), w.list[i].splits.size() * sizeof(TreeSplit));
        put(h + l.row_split[i], w.list[i].row_split.data(), w.list[i].row_split.size() * 4);
    }
    put(h + l.flat, t.pt_flat, s.n_flat * 4);
    put(h + l.off, t.pt_off, (s.batch + 1) * 4);
    put(h + l.prefix, t.prefix, s.batch * 4);
    put(h + l.draft, t.draft, s.batch * 4);
    uint32_t* token0 = reinterpret_cast<uint32_t*>(h + l.token0);
    uint32_t* token_req = reinterpret_cast<uint32_t*>(h + l.token_req);
    uint32_t n = 0;
    for (size_t r = 0; r < s.batch; ++r) {
        token0[r] = n;
        for (uint32_t i = 0; i < t.draft[r]; ++i) token_req[n++] = static_cast<uint32_t>(r);
    }
    token0[s.batch] = n;
    put(h + l.mask, t.mask, s.tokens * s.mask_words * 4);
}

TreeView view_of(const uint8_t* dev, const TreeLayout& l, const TreeWorks& w) {
    TreeView v;
    auto words = [&](size_t at) { return reinterpret_cast<const uint32_t*>(dev + at); };
    v.pt_flat = words(l.flat);
    v.pt_off = words(l.off);
    v.prefix = words(l.prefix);
    v.draft = words(l.draft);
    v.token0 = words(l.token0);
    v.token_req = words(l.token_req);
    v.mask = words(l.mask);
    for (uint32_t i = 0; i < kTreeLists; ++i) {
        const TreeWork& list = w.list[i];
        TreeWorkView& out = v.work[i];
        out.pieces = reinterpret_cast<const TreePiece*>(dev + l.pieces[i]);
        out.splits = reinterpret_cast<const TreeSplit*>(dev + l.splits[i]);
        out.row_split = words(l.row_split[i]);
        out.n_cta = list.n_cta;
        out.n_slots = list.n_slots;
        out.slot_rows = list.slot_rows;
        out.max_parts = list.max_parts;
        out.merge_rows = static_cast<uint32_t>(list.row_split.size());
    }
    return v;
}

// The rules every entry point applies to its tables. Host arithmetic only; `why` receives the message.
int check_tables(TreeShape& s, const TreeTables& t, size_t n_flat, std::string* why) {
    auto no = [&](int status, const char* fmt, ...) {
        char buf[200];
        va_list args;
        va_start(args, fmt);
        std::vsnprintf(buf, sizeof(buf), fmt, args);
        va_end(args);
        *why = buf;
        return status;
    };
    if (s.batch == 0 || s.H == 0 || s.D == 0 || s.P == 0) return no(MLC_ERR_INVALID_ARG, "zero dimension");
    if (s.KVH == 0 || s.H % s.KVH != 0) return no(MLC_ERR_INVALID_ARG, "num_heads must be a multiple of kv_heads");
    if (s.D > 256) return no(MLC_ERR_UNSUPPORTED, "head_dim > 256");
    if (s.P >= (size_t(1) << 31) || s.mask_words > (size_t(1) << 27)) return no(MLC_ERR_UNSUPPORTED, "page_size_tokens or mask_words too large");
    if (!t.pt_off || !t.prefix || !t.draft || (!t.pt_flat && n_flat)) return no(MLC_ERR_INVALID_ARG, "null table");
    for (size_t r = 0; r < s.batch; ++r)
        if (t.pt_off[r + 1] < t.pt_off[r]) return no(MLC_ERR_BOUNDS, "page_table_offsets not monotone at %zu", r);
    if (n_flat < t.pt_off[s.batch]) return no(MLC_ERR_INVALID_ARG, "page_tables_flat shorter than the last offset");
    s.n_flat = t.pt_off[s.batch];
    s.tokens = 0;
    for (size_t r = 0; r < s.batch; ++r) {
        const uint64_t room = static_cast<uint64_t>(t.pt_off[r + 1] - t.pt_off[r]) * s.P;
        const uint64_t len = static_cast<uint64_t>(t.prefix[r]) + t.draft[r];
        if (len > room)
            return no(MLC_ERR_BOUNDS, "prefix_lens[%zu] + draft_lens[%zu] = %llu exceeds its %u pages", r, r,
                      static_cast<unsigned long long>(len), t.pt_off[r + 1] - t.pt_off[r]);
        if (len > 0xFFFFFF00ull) return no(MLC_ERR_UNSUPPORTED, "request %zu too long", r);
        if (t.draft[r] > s.mask_words * 32)
            return no(MLC_ERR_INVALID_ARG, "draft_lens[%zu]=%u needs more than %zu mask words", r, t.draft[r], s.mask_words);
        s.tokens += t.draft[r];
    }
    if (s.tokens && !t.mask) return no(MLC_ERR_INVALID_ARG, "null mask");
    if (s.tokens * s.H >= (size_t(1) << 31)) return no(MLC_ERR_UNSUPPORTED, "drafted tokens * heads too large");
    if (s.capacity)
        for (size_t i = 0; i < s.n_flat; ++i)
            if (t.pt_flat[i] >= s.capacity)
                return no(MLC_ERR_BOUNDS, "page_tables_flat[%zu]=%u >= capacity %zu", i, t.pt_flat[i], s.capacity);
    return MLC_OK;
}

// Without drafted tokens there is nothing to read or write: q and o may be null then.
int check_call(mlc_ctx* ctx, const TreeArgs& a, bool rows) {
    if ((rows && (!a.q || !a.o)) || !a.k_pages || !a.v_pages) return ctx->fail(MLC_ERR_INVALID_ARG, "null buffer");
    if ((a.q_dtype != MLC_F32 && a.q_dtype != MLC_F16) || (a.o_dtype != MLC_F32 && a.o_dtype != MLC_F16))
        return ctx->fail(MLC_ERR_INVALID_ARG, "q / o dtype must be MLC_F16 or MLC_F32");
    if (!aligned_to(a.q, a.q_dtype == MLC_F32 ? 4 : 2) || !aligned_to(a.o, a.o_dtype == MLC_F32 ? 4 : 2) || !aligned_to(a.k_pages, 2) ||
        !aligned_to(a.v_pages, 2))
        return ctx->fail(MLC_ERR_INVALID_ARG, "buffers must be aligned to their elements");
    return MLC_OK;
}

int launch(mlc_ctx* ctx, const TreeShape& s, const TreeView& v, TreeArgs a) {
    if (s.tokens == 0) return MLC_OK;
    const size_t elems = s.tokens * s.H * s.D;
    if (overlap(a.q, elems * (a.q_dtype == MLC_F32 ? 4 : 2), a.o, elems * (a.o_dtype == MLC_F32 ? 4 : 2)))
        return ctx->fail(MLC_ERR_INVALID_ARG, "o overlaps q");
    if (!(a.scale > 0.f)) a.scale = 1.0f / std::sqrt(static_cast<float>(s.D));
    if (v.work[0].n_cta && !ctx->force_general && tree_tcgen05_buffers(a)) {
        ctx->last_attention_kernel = 4;
        return launch_tree_tcgen05(ctx, s, v, a);
    }
    ctx->last_attention_kernel = 1;
    return launch_tree_general(ctx, s, v, a);
}

// The work lists of the tensor-core kernel, and room for their partials.
int prepare_work(mlc_ctx* ctx, const TreeShape& s, const TreeTables& t, TreeWorks* w) {
    if (!tree_tcgen05_shape(s)) return MLC_OK;
    size_t bytes = 0;
    for (uint32_t i = 0; i < (s.D == 128 ? kTreeLists : 1u); ++i) {
        tree_work_list(s, t, static_cast<uint32_t>(ctx->sm_count) * (i ? 1u : 2u), &w->list[i]);
        bytes = std::max(bytes, tree_scratch_bytes(s, w->list[i].n_slots, w->list[i].slot_rows));
    }
    return ensure_op_scratch(ctx, ctx->tree_scratch, bytes, "tree attention scratch");
}

// One call with host tables: the image goes through the context's staging area.
int tree_impl(mlc_ctx* ctx, bool sync, const TreeArgs& a, TreeShape s, const TreeTables& t, size_t n_flat) {
    if (!ctx) return MLC_ERR_INVALID_ARG;
    s.capacity = resolve_capacity(ctx, a.k_pages, s.capacity, s.P * s.KVH * s.D * 2);
    std::string why;
    int st = check_tables(s, t, n_flat, &why);
    if (st != MLC_OK) return ctx->fail(st, "%s", why.c_str());
    if ((st = check_call(ctx, a, s.tokens > 0)) != MLC_OK) return st;
    if (!sync && !ctx->pass_open) return ctx->fail(MLC_ERR_NO_OPEN_PASS, "encode without an open pass");
    if (ctx->capturing) return ctx->fail(MLC_ERR_UNSUPPORTED, "host tables inside a graph capture: use a plan");
    if (s.tokens == 0) return MLC_OK;
    DeviceGuard guard(ctx->device);
    TreeWorks w;
    if ((st = prepare_work(ctx, s, t, &w)) != MLC_OK) return st;
    const TreeLayout l = layout_of(s, w);
    void *h = nullptr, *d = nullptr;
    if (!stage_reserve(ctx, l.total, &h, &d)) return MLC_ERR_OOM;
    fill_image(static_cast<uint8_t*>(h), l, s, t, w);
    if (!stage_commit(ctx, h, d, l.total)) return MLC_ERR_CUDA;
    if ((st = launch(ctx, s, view_of(static_cast<uint8_t*>(d), l, w), a)) != MLC_OK) return st;
    if (!sync) return MLC_OK;
    const cudaError_t e = cudaStreamSynchronize(ctx->stream);
    if (!ctx->pass_open) stage_reset(ctx);
    if (e != cudaSuccess) return ctx->fail(MLC_ERR_CUDA, "tree attention failed: %s", cudaGetErrorString(e));
    uint32_t word = 0;
    MLCB_CUDA(ctx, cudaMemcpy(&word, ctx->d_err, 4, cudaMemcpyDeviceToHost));
    if (word) {
        reset_after_device_error(ctx);
        return ctx->fail(MLC_ERR_DEVICE_FLAG, "tree attention recorded error word 0x%x", word);
    }
    return MLC_OK;
}

void release_buffers(mlc_tree_plan& p) {
    if (p.uploaded) cudaEventSynchronize(p.uploaded);
    if (p.host) cudaFreeHost(p.host);
    if (p.dev) cudaFree(p.dev);
    p.host = p.dev = nullptr;
    p.cap = 0;
}

// Puts new tables into the plan. On failure the plan keeps its old ones.
int fill_plan(mlc_ctx* ctx, mlc_tree_plan& p, TreeShape s, const TreeTables& t, size_t n_flat) {
    std::string why;
    int st = check_tables(s, t, n_flat, &why);
    if (st != MLC_OK) return ctx->fail(st, "%s", why.c_str());
    if (ctx->capturing) return ctx->fail(MLC_ERR_UNSUPPORTED, "new tables inside a graph capture: create the plan before capturing");
    DeviceGuard guard(ctx->device);
    TreeWorks w;
    if ((st = prepare_work(ctx, s, t, &w)) != MLC_OK) return st;
    const TreeLayout l = layout_of(s, w);
    if (!p.uploaded) MLCB_CUDA(ctx, cudaEventCreateWithFlags(&p.uploaded, cudaEventDisableTiming));
    if (l.total > p.cap) {
        const size_t want = l.total + l.total / 2;
        uint8_t *h = nullptr, *d = nullptr;
        if (cudaHostAlloc(reinterpret_cast<void**>(&h), want, cudaHostAllocDefault) != cudaSuccess) {
            cudaGetLastError();
            return ctx->fail(MLC_ERR_OOM, "pinned memory for the plan unavailable");
        }
        if (cudaMalloc(reinterpret_cast<void**>(&d), want) != cudaSuccess) {
            cudaGetLastError();
            cudaFreeHost(h);
            return ctx->fail(MLC_ERR_OOM, "device memory for the plan unavailable");
        }
        MLCB_CUDA(ctx, cudaStreamSynchronize(ctx->stream));   // kernels that read the old image
        release_buffers(p);
        p.ready = false;      // until the new image is on its way
        p.host = h;
        p.dev = d;
        p.cap = want;
        ctx->allocations += 2;
    } else {
        MLCB_CUDA(ctx, cudaEventSynchronize(p.uploaded));     // the last upload has left the pinned image
    }
    fill_image(p.host, l, s, t, w);
    // in stream order, behind the kernels already enqueued with the old tables
    MLCB_CUDA(ctx, cudaMemcpyAsync(p.dev, p.host, l.total, cudaMemcpyHostToDevice, ctx->stream));
    MLCB_CUDA(ctx, cudaEventRecord(p.uploaded, ctx->stream));
    p.shape = s;
    p.view = view_of(p.dev, l, w);
    p.ready = true;
    return MLC_OK;
}

}  // namespace

extern "C" {

int mlc_run_paged_tree_attention(mlc_ctx* ctx, const void* q, const void* k_pages, const void* v_pages, void* o,
                                 const uint32_t* page_tables_flat, size_t n_page_tables_flat,
                                 const uint32_t* page_table_offsets, const uint32_t* prefix_lens,
                                 const uint32_t* draft_lens, const uint32_t* tree_mask, size_t mask_words, size_t batch,
                                 size_t num_heads, size_t kv_heads, size_t head_dim, size_t page_size_tokens, float scale,
                                 int q_dtype, int o_dtype, size_t capacity_pages) {
    return no_throw(ctx, [&] { return tree_impl(ctx, true, {q, k_pages, v_pages, o, scale, q_dtype, o_dtype},
                     {batch, num_heads, kv_heads, head_dim, page_size_tokens, capacity_pages, mask_words},
                     {page_tables_flat, page_table_offsets, prefix_lens, draft_lens, tree_mask}, n_page_tables_flat); });
}

int mlc_encode_paged_tree_attention(mlc_ctx* ctx, const void* q, const void* k_pages, const void* v_pages, void* o,
                                    const uint32_t* page_tables_flat, size_t n_page_tables_flat,
                                    const uint32_t* page_table_offsets, const uint32_t* prefix_lens,
                                    const uint32_t* draft_lens, const uint32_t* tree_mask, size_t mask_words, size_t batch,
                                    size_t num_heads, size_t kv_heads, size_t head_dim, size_t page_size_tokens, float scale,
                                    int q_dtype, int o_dtype, size_t capacity_pages) {
    return no_throw(ctx, [&] { return tree_impl(ctx, false, {q, k_pages, v_pages, o, scale, q_dtype, o_dtype},
                     {batch, num_heads, kv_heads, head_dim, page_size_tokens, capacity_pages, mask_words},
                     {page_tables_flat, page_table_offsets, prefix_lens, draft_lens, tree_mask}, n_page_tables_flat); });
}

int mlc_tree_plan_create(mlc_ctx* ctx, const uint32_t* page_tables_flat, size_t n_page_tables_flat,
                         const uint32_t* page_table_offsets, const uint32_t* prefix_lens, const uint32_t* draft_lens,
                         const uint32_t* tree_mask, size_t mask_words, size_t batch, size_t num_heads, size_t kv_heads,
                         size_t head_dim, size_t page_size_tokens, size_t capacity_pages, mlc_tree_plan** out) {
    if (!ctx || !out) return MLC_ERR_INVALID_ARG;
    *out = nullptr;
    auto* p = new (std::nothrow) mlc_tree_plan();
    if (!p) return ctx->fail(MLC_ERR_OOM, "host memory for the plan unavailable");
    p->ctx = ctx;
    const int st = no_throw(ctx, [&] {
        return fill_plan(ctx, *p, {batch, num_heads, kv_heads, head_dim, page_size_tokens, capacity_pages, mask_words},
                         {page_tables_flat, page_table_offsets, prefix_lens, draft_lens, tree_mask}, n_page_tables_flat);
    });
    if (st != MLC_OK) {
        mlc_tree_plan_destroy(ctx, p);
        return st;
    }
    *out = p;
    return MLC_OK;
}

int mlc_tree_plan_update(mlc_ctx* ctx, mlc_tree_plan* plan, const uint32_t* page_tables_flat, size_t n_page_tables_flat,
                         const uint32_t* page_table_offsets, const uint32_t* prefix_lens, const uint32_t* draft_lens,
                         const uint32_t* tree_mask, size_t mask_words, size_t batch) {
    if (!ctx || !plan) return MLC_ERR_INVALID_ARG;
    if (plan->ctx != ctx) return ctx->fail(MLC_ERR_INVALID_ARG, "the plan belongs to another context");
    // a replay launches the grid of the tables that were captured
    if (plan->captured) return ctx->fail(MLC_ERR_UNSUPPORTED, "the plan is part of a captured graph: create another one");
    TreeShape s = plan->shape;
    s.batch = batch;
    s.mask_words = mask_words;
    return no_throw(ctx, [&] {
        return fill_plan(ctx, *plan, s, {page_tables_flat, page_table_offsets, prefix_lens, draft_lens, tree_mask},
                         n_page_tables_flat);
    });
}

void mlc_tree_plan_destroy(mlc_ctx* ctx, mlc_tree_plan* plan) {
    if (!ctx || !plan) return;
    DeviceGuard guard(ctx->device);
    if (ctx->capturing) {
        // waiting or freeing here would spoil the capture: the buffers go with the context
        no_throw(ctx, [&] {
            if (plan->dev) ctx->tree_scratch.retired.push_back(plan->dev);
            if (plan->host) ctx->tree_scratch.retired_host.push_back(plan->host);
            return MLC_OK;
        });
    } else {
        cudaStreamSynchronize(ctx->stream);
        release_buffers(*plan);
    }
    if (plan->uploaded) cudaEventDestroy(plan->uploaded);
    delete plan;
}

int mlc_encode_paged_tree_attention_planned(mlc_ctx* ctx, const mlc_tree_plan* plan, const void* q, const void* k_pages,
                                            const void* v_pages, void* o, float scale, int q_dtype, int o_dtype) {
    if (!ctx || !plan) return MLC_ERR_INVALID_ARG;
    if (plan->ctx != ctx) return ctx->fail(MLC_ERR_INVALID_ARG, "the plan belongs to another context");
    if (!ctx->pass_open) return ctx->fail(MLC_ERR_NO_OPEN_PASS, "encode without an open pass");
    if (!plan->ready) return ctx->fail(MLC_ERR_INVALID_ARG, "the plan lost its tables in a failed update");
    const TreeArgs a{q, k_pages, v_pages, o, scale, q_dtype, o_dtype};
    const int st = check_call(ctx, a, plan->shape.tokens > 0);
    if (st != MLC_OK) return st;
    DeviceGuard guard(ctx->device);
    if (ctx->capturing) plan->captured = true;
    return launch(ctx, plan->shape, plan->view, a);
}

}  // extern "C"
