// One selection step of beam search on the device. Per group of `beams` beams over a vocabulary:
//   score(p, t) = cum[p] + x[p, t] - log sum_u exp x[p, u]
// and the n_select best (p, t) of the group, best first, ties to the lowest p, then the lowest t. A finished beam has one
// candidate, (p, pad token) with its score as it is. Candidates whose score is -inf or no number are never selected; places
// that stay empty get score -inf and 0xFFFFFFFF. The reference samples greedily on the host
// (compiler/runtime/scheduler.cpp:101-118); this stands beside the device argmax.
//
// What bounds it: every logit is read once, so the memory's read bandwidth for large calls; a launch and the two chained
// steps for small ones. One pass over the logits does both jobs: a CTA holds a chunk of a row in registers, takes its
// maximum, its sum of exponentials and its n_select largest values, and the last CTA of a group to finish joins the chunks.
// Inside a row the order by score is the order by logit, so a chunk needs no logarithm. The values of a chunk are
// found with a threshold: the n_select-th largest of 64 maxima over disjoint parts of the chunk has at least n_select
// values at or above it, and on real logits few more. The cross-beam comparison needs the differences of nearly
// equal sums: sums over 32 values are taken in fp32, what joins them and the scores in fp64.
#include <cuda_fp16.h>

#include <cstring>

#include "op_util.hpp"

namespace mlcb {

namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kParts = 64;        // maxima the threshold is taken from: one per four threads
constexpr uint32_t kMaxSelect = 64;    // = kParts: the threshold needs that many
constexpr uint32_t kMaxBeams = 64;
constexpr uint32_t kListCap = 512;
constexpr float kLog2e = 1.4426950408889634f;

struct BeamParams {
    const float* logits;
    const float* cum;
    const uint8_t* finished;   // may be null
    uint64_t* keys;            // [rows * chunks][n_select]
    float2* sums;              // [rows * chunks] (maximum, sum of exponentials relative to it)
    uint32_t* counters;        // [groups], zero between launches
    float* out_scores;
    uint32_t* out_parents;
    uint32_t* out_tokens;
    uint32_t rows, beams, vocab, group_rows, chunks_per_part, chunks, chunk_len, n_select, pad;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// exp(a - b) for a <= b; b > -inf
__device__ __forceinline__ float exp_diff(float a, float b) { return ex2((a - b) * kLog2e); }

// Larger key = larger value, then lower token; 0 is below every key.
__device__ __forceinline__ uint64_t make_key(float x, uint32_t token) {
    const uint32_t b = __float_as_uint(x);
    const uint32_t ordered = (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return (static_cast<uint64_t>(ordered) << 32) | (0xFFFFFFFFu - token);
}
__device__ __forceinline__ float key_value(uint64_t key) {
    const uint32_t o = static_cast<uint32_t>(key >> 32);
    return __uint_as_float((o & 0x80000000u) ? o & 0x7FFFFFFFu : ~o);
}
__device__ __forceinline__ uint32_t key_token(uint64_t key) { return 0xFFFFFFFFu - static_cast<uint32_t>(key); }

// The k-th largest of 64 values in shared memory, computed by one warp (every lane gets it).
template <typename T>
__device__ __forceinline__ T kth_of_64(const T* v, uint32_t k, uint32_t lane, T lowest) {
    const T a = v[lane], b = v[lane + 32];
    uint32_t above_a = 0, above_b = 0, with_a = 0, with_b = 0;
#pragma unroll 8
    for (uint32_t j = 0; j < 64; ++j) {
        const T x = v[j];
        above_a += x > a;
        above_b += x > b;
        with_a += x >= a;
        with_b += x >= b;
    }
    const bool is_a = above_a < k && k <= with_a, is_b = above_b < k && k <= with_b;
    const uint32_t va = __ballot_sync(0xffffffffu, is_a), vb = __ballot_sync(0xffffffffu, is_b);
    if (va) return __shfl_sync(0xffffffffu, a, __ffs(va) - 1);
    if (vb) return __shfl_sync(0xffffffffu, b, __ffs(vb) - 1);
    return lowest;
}

struct Candidate {
    double score;
    uint32_t parent, token;
};
__device__ __forceinline__ bool better(const Candidate& a, const Candidate& b) {
    if (a.score != b.score) return a.score > b.score;
    return a.parent != b.parent ? a.parent < b.parent : a.token < b.token;
}

struct Shared {
    uint64_t list[kListCap];
    Candidate found[kListCap];
    double part_d[kParts];
    double lse[kMaxBeams];
    float part[kParts];
    float warp_m[8], warp_s[8];
    uint64_t warp_key[8];
    Candidate warp_best[8];
    float threshold;
    double threshold_d;
    uint32_t count, last;
};

// Joins the chunks of one group: run by the CTA that finished last.
__device__ __noinline__ void join_group(const BeamParams& p, Shared& sh, uint32_t group) {
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t row0 = group * p.beams;
    for (uint32_t b = warp; b < p.beams; b += kThreads / 32) {
        float m = -INFINITY;
        for (uint32_t c = lane; c < p.chunks; c += 32) m = fmaxf(m, __ldcg(&p.sums[static_cast<size_t>(row0 + b) * p.chunks + c].x));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        double s = 0.0;
        for (uint32_t c = lane; c < p.chunks; c += 32) {
            const float2 ms = __ldcg(&p.sums[static_cast<size_t>(row0 + b) * p.chunks + c]);
            if (ms.x > -INFINITY || ms.y != 0.0f) s += static_cast<double>(ms.y) * exp(static_cast<double>(ms.x) - static_cast<double>(m));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        // (a row of -inf alone has no candidates that would use it; one with +inf gives NaN, and so no candidates)
        if (lane == 0) sh.lse[b] = static_cast<double>(m) + log(s);
    }
    if (tid == 0) sh.count = 0;
    __syncthreads();

    const uint32_t per_row = p.chunks * p.n_select, total = p.beams * per_row;
    // candidate i of the group: a chunk's list entry; behind them one per beam for finished beams
    auto candidate = [&](uint32_t i, Candidate& c) {
        if (i >= total) {
            const uint32_t b = i - total;
            if (!p.finished || !p.finished[row0 + b]) return false;
            c = {static_cast<double>(p.cum[row0 + b]), b, p.pad};
        } else {
            const uint32_t b = i / per_row;
            if (p.finished && p.finished[row0 + b]) return false;
            const uint64_t key = __ldcg(&p.keys[static_cast<size_t>(row0) * per_row + i]);
            if (key == 0) return false;
            c = {static_cast<double>(p.cum[row0 + b]) + (static_cast<double>(key_value(key)) - sh.lse[b]), b, key_token(key)};
        }
        return c.score > -INFINITY;   // not for NaN either
    };
    double top = -INFINITY;
    for (uint32_t i = tid; i < total + p.beams; i += kThreads) {
        Candidate c;
        if (candidate(i, c)) top = fmax(top, c.score);
    }
    top = fmax(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmax(top, __shfl_xor_sync(0xffffffffu, top, 2));
    if ((tid & 3) == 0) sh.part_d[tid >> 2] = top;
    __syncthreads();
    if (warp == 0) {
        const double t = kth_of_64(sh.part_d, p.n_select, lane, static_cast<double>(-INFINITY));
        if (lane == 0) sh.threshold_d = t;
    }
    __syncthreads();
    const double threshold = sh.threshold_d;
    for (uint32_t i = tid; i < total + p.beams; i += kThreads) {
        Candidate c;
        if (candidate(i, c) && c.score >= threshold) {
            const uint32_t at = atomicAdd(&sh.count, 1u);
            if (at < kListCap) sh.found[at] = c;
        }
    }
    __syncthreads();
    const uint32_t n = sh.count;
    const size_t out = static_cast<size_t>(group) * p.n_select;
    auto write = [&](uint32_t at, const Candidate& c) {
        p.out_scores[out + at] = static_cast<float>(c.score);
        p.out_parents[out + at] = c.parent;
        p.out_tokens[out + at] = c.token;
    };
    uint32_t have = n;
    if (n <= kListCap) {
        for (uint32_t i = tid; i < n; i += kThreads) {
            const Candidate mine = sh.found[i];
            uint32_t rank = 0;
            for (uint32_t j = 0; j < n; ++j) rank += better(sh.found[j], mine);
            if (rank < p.n_select) write(rank, mine);
        }
    } else {
        // many equal scores: take the best, then the best below it, and so on
        Candidate last{INFINITY, 0, 0};
        bool first = true;
        for (have = 0; have < p.n_select; ++have) {
            Candidate best{-INFINITY, 0xFFFFFFFFu, 0xFFFFFFFFu};
            for (uint32_t i = tid; i < total + p.beams; i += kThreads) {
                Candidate c;
                if (candidate(i, c) && (first || better(last, c)) && better(c, best)) best = c;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const Candidate c{__shfl_xor_sync(0xffffffffu, best.score, o), __shfl_xor_sync(0xffffffffu, best.parent, o),
                                  __shfl_xor_sync(0xffffffffu, best.token, o)};
                if (better(c, best)) best = c;
            }
            if (lane == 0) sh.warp_best[warp] = best;
            __syncthreads();
            best = sh.warp_best[0];
            for (uint32_t w = 1; w < kThreads / 32; ++w)
                if (better(sh.warp_best[w], best)) best = sh.warp_best[w];
            __syncthreads();
            if (!(best.score > -INFINITY)) break;
            if (tid == 0) write(have, best);
            last = best;
            first = false;
        }
    }
    for (uint32_t i = have + tid; i < p.n_select; i += kThreads) write(i, {-INFINITY, 0xFFFFFFFFu, 0xFFFFFFFFu});
}

// NV: float4 vectors of a chunk that a thread holds.
template <int NV>
__global__ void __launch_bounds__(kThreads) beam_select_kernel(const __grid_constant__ BeamParams p) {
    __shared__ Shared sh;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t row = blockIdx.x / p.chunks, chunk = blockIdx.x - row * p.chunks;
    const uint32_t group = row / p.beams;
    if (!p.finished || !p.finished[row]) {
        const uint32_t part = chunk / p.chunks_per_part, begin = (chunk - part * p.chunks_per_part) * p.chunk_len;
        const uint32_t part_rows = min(p.group_rows, p.vocab - part * p.group_rows);
        const uint32_t len = begin < part_rows ? min(p.chunk_len, part_rows - begin) : 0u;   // the last part may be short
        const uint32_t token0 = part * p.group_rows + begin;
        const float* x0 = p.logits + static_cast<size_t>(p.rows) * part * p.group_rows + static_cast<size_t>(row) * part_rows + begin;
        const uint32_t lead = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(x0) >> 2) & 3u;   // floats behind a 16-byte boundary
        float x[NV][4];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int at = static_cast<int>(4 * (tid + kThreads * j)) - static_cast<int>(lead);
            if (at >= 0 && at + 4 <= static_cast<int>(len)) {
                const float4 v = __ldcs(reinterpret_cast<const float4*>(x0 + at));
                x[j][0] = v.x; x[j][1] = v.y; x[j][2] = v.z; x[j][3] = v.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[j][e] = at + e >= 0 && at + e < static_cast<int>(len) ? x0[at + e] : -INFINITY;
            }
        }
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[j][e] += 0.0f;                                     // -0 and 0 are one value
                if (!(x[j][e] == x[j][e])) x[j][e] = -INFINITY;      // NaN
                top = fmaxf(top, x[j][e]);
            }
        float s = 0.0f;
        if (top > -INFINITY) {
#pragma unroll
            for (int j = 0; j < NV; ++j)
                s += (exp_diff(x[j][0], top) + exp_diff(x[j][1], top)) + (exp_diff(x[j][2], top) + exp_diff(x[j][3], top));
        }
        float quad = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        quad = fmaxf(quad, __shfl_xor_sync(0xffffffffu, quad, 2));
        if ((tid & 3) == 0) sh.part[tid >> 2] = quad;
        float m = quad;
#pragma unroll
        for (int o = 16; o > 2; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        s = top > -INFINITY ? s * exp_diff(top, m) : 0.0f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) { sh.warp_m[warp] = m; sh.warp_s[warp] = s; }
        if (tid == 0) sh.count = 0;
        __syncthreads();
        if (warp == 0) {
            const float t = kth_of_64(sh.part, p.n_select, lane, -INFINITY);
            if (lane == 0) sh.threshold = t;
        } else if (tid == 32) {
            float all = -INFINITY;
            for (int w = 0; w < 8; ++w) all = fmaxf(all, sh.warp_m[w]);
            double sum = 0.0;
            for (int w = 0; w < 8; ++w)
                if (sh.warp_m[w] > -INFINITY) sum += static_cast<double>(sh.warp_s[w]) * static_cast<double>(exp_diff(sh.warp_m[w], all));
            p.sums[blockIdx.x] = make_float2(all, static_cast<float>(sum));
        }
        __syncthreads();
        const float threshold = sh.threshold;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (x[j][e] >= threshold && x[j][e] > -INFINITY) {
                    const uint32_t at = atomicAdd(&sh.count, 1u);
                    if (at < kListCap) sh.list[at] = make_key(x[j][e], token0 + 4 * (tid + kThreads * j) + e - lead);
                }
        __syncthreads();
        uint64_t* keys = p.keys + static_cast<size_t>(blockIdx.x) * p.n_select;
        const uint32_t n = sh.count;
        uint32_t have = n;
        if (n <= kListCap) {
            for (uint32_t i = tid; i < n; i += kThreads) {
                const uint64_t mine = sh.list[i];
                uint32_t rank = 0;
                for (uint32_t j = 0; j < n; ++j) rank += sh.list[j] > mine;
                if (rank < p.n_select) keys[rank] = mine;
            }
        } else {
            // many equal values at the threshold: take the best key, then the best below it, and so on
            uint64_t last = ~0ull;
            for (have = 0; have < p.n_select; ++have) {
                uint64_t best = 0;
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (x[j][e] > -INFINITY) {
                            const uint64_t k = make_key(x[j][e], token0 + 4 * (tid + kThreads * j) + e - lead);
                            if (k < last && k > best) best = k;
                        }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    const uint64_t k = __shfl_xor_sync(0xffffffffu, best, o);
                    if (k > best) best = k;
                }
                if (lane == 0) sh.warp_key[warp] = best;
                __syncthreads();
                for (int w = 0; w < 8; ++w)
                    if (sh.warp_key[w] > best) best = sh.warp_key[w];
                __syncthreads();
                if (best == 0) break;
                if (tid == 0) keys[have] = best;
                last = best;
            }
        }
        for (uint32_t i = have + tid; i < p.n_select; i += kThreads) keys[i] = 0;
    }
    // the last CTA of the group joins
    __threadfence();
    __syncthreads();
    if (tid == 0) sh.last = atomicAdd(&p.counters[group], 1u) == p.beams * p.chunks - 1 ? 1u : 0u;
    __syncthreads();
    if (!sh.last) return;
    __threadfence();
    if (tid == 0) p.counters[group] = 0;
    join_group(p, sh, group);
}

int beam_select(mlc_ctx* ctx, const void* logits, const void* cum, const void* finished, size_t groups, size_t beams, size_t vocab,
                size_t group_rows, size_t n_select, uint32_t pad_token, void* out_scores, void* out_parents, void* out_tokens) {
    if (!ctx) return MLC_ERR_INVALID_ARG;
    if (!ctx->pass_open) return ctx->fail(MLC_ERR_NO_OPEN_PASS, "encode without an open pass");
    if (!logits || !cum || !out_scores || !out_parents || !out_tokens) return ctx->fail(MLC_ERR_INVALID_ARG, "null buffer");
    if (groups == 0 || beams == 0 || vocab == 0 || n_select == 0) return ctx->fail(MLC_ERR_INVALID_ARG, "zero dimension");
    if (beams > kMaxBeams || n_select > kMaxSelect)
        return ctx->fail(MLC_ERR_UNSUPPORTED, "more than %u beams or %u selected candidates", kMaxBeams, kMaxSelect);
    if (vocab >= (size_t(1) << 31) || groups >= (size_t(1) << 24)) return ctx->fail(MLC_ERR_UNSUPPORTED, "dimension too large");
    if (finished && pad_token >= vocab) return ctx->fail(MLC_ERR_INVALID_ARG, "pad token %u outside the vocabulary", pad_token);
    if (!aligned_to(logits, 4) || !aligned_to(cum, 4) || !aligned_to(out_scores, 4) || !aligned_to(out_parents, 4) ||
        !aligned_to(out_tokens, 4))
        return ctx->fail(MLC_ERR_INVALID_ARG, "buffers must be aligned to their elements");
    if (group_rows == 0 || group_rows > vocab) group_rows = vocab;
    const size_t rows = groups * beams, parts = (vocab + group_rows - 1) / group_rows;
    int nv = 8;
    size_t per_part = 0;
    for (;; nv /= 2) {   // shorter chunks while they are needed to give every SM one
        const size_t most = static_cast<size_t>(nv) * kThreads * 4 - 4;   // an unaligned row takes a vector more
        per_part = (group_rows + most - 1) / most;
        if (nv == 2 || rows * parts * per_part >= static_cast<size_t>(ctx->sm_count)) break;
    }
    const size_t chunks = parts * per_part;
    const size_t chunk_len = ((group_rows + per_part - 1) / per_part + 3) / 4 * 4;
    if (rows * chunks >= (size_t(1) << 31) || beams * chunks * n_select >= (size_t(1) << 31))
        return ctx->fail(MLC_ERR_UNSUPPORTED, "too many rows");
    DeviceGuard guard(ctx->device);
    const size_t key_bytes = rows * chunks * n_select * 8, sum_bytes = rows * chunks * sizeof(float2);
    int st = ensure_op_scratch(ctx, ctx->beam_scratch, key_bytes + sum_bytes, "beam selection scratch");
    if (st == MLC_OK) st = ensure_op_scratch(ctx, ctx->beam_counters, groups * 4, "beam selection counters");
    if (st != MLC_OK) return st;
    BeamParams p{};
    p.logits = static_cast<const float*>(logits);
    p.cum = static_cast<const float*>(cum);
    p.finished = static_cast<const uint8_t*>(finished);
    p.keys = static_cast<uint64_t*>(ctx->beam_scratch.dev);
    p.sums = reinterpret_cast<float2*>(static_cast<char*>(ctx->beam_scratch.dev) + key_bytes);
    p.counters = static_cast<uint32_t*>(ctx->beam_counters.dev);
    p.out_scores = static_cast<float*>(out_scores);
    p.out_parents = static_cast<uint32_t*>(out_parents);
    p.out_tokens = static_cast<uint32_t*>(out_tokens);
    p.rows = static_cast<uint32_t>(rows);
    p.beams = static_cast<uint32_t>(beams);
    p.vocab = static_cast<uint32_t>(vocab);
    p.group_rows = static_cast<uint32_t>(group_rows);
    p.chunks_per_part = static_cast<uint32_t>(per_part);
    p.chunks = static_cast<uint32_t>(chunks);
    p.chunk_len = static_cast<uint32_t>(chunk_len);
    p.n_select = static_cast<uint32_t>(n_select);
    p.pad = pad_token;
    const dim3 grid(static_cast<unsigned>(rows * chunks));
    auto kernel = nv == 8 ? beam_select_kernel<8> : nv == 4 ? beam_select_kernel<4> : beam_select_kernel<2>;
    MLCB_CUDA(ctx, launch_dependent(ctx, kernel, grid, kThreads, 0, p));
    ++ctx->launches;
    return MLC_OK;
}

}  // namespace

}  // namespace mlcb

extern "C" int mlc_encode_beam_select(mlc_ctx* ctx, const void* logits, const void* cum_scores, const void* finished,
                                      size_t groups, size_t beams, size_t vocab, size_t group_rows, size_t n_select,
                                      uint32_t pad_token, void* out_scores, void* out_parents, void* out_tokens) {
    return mlcb::no_throw(ctx, [&] {
        return mlcb::beam_select(ctx, logits, cum_scores, finished, groups, beams, vocab, group_rows, n_select, pad_token,
                                 out_scores, out_parents, out_tokens);
    });
}
