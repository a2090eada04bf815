// One selection step of beam search on the device. Per group of `beams` beams over a vocabulary:
//   score(p, t) = cum[p] + x[p, t] - log sum_u exp x[p, u]
// and the n_select best (p, t) of the group, best first, ties to the lowest p, then the lowest t. A finished beam has one
// candidate, (p, pad token) with its score as it is. Candidates whose score is -inf or no number are never selected; places
// that stay empty get score -inf and 0xFFFFFFFF. The reference samples greedily on the host
// (compiler/runtime/scheduler.cpp:101-118); this stands beside the device argmax.
//
// What bounds it: every logit is read once, so the memory's read bandwidth for large calls; a launch and the two chained
// steps for small ones. One pass over the logits does both jobs: a warp walks a segment of a row, 512 logits a step with
// the next two steps' in flight, and keeps a running maximum, a running sum of exponentials and the n_select largest logits
// so far; the last CTA of a group to finish joins the segments. Inside a row the order by score is the order by logit, so a
// segment needs no logarithm. The largest logits are kept as a list in shared memory with a threshold, the n_select-th
// largest at the last clean-up: on real logits few pass it after the first step, and a step in which none does costs one
// vote. Warps work on their own: 512 rows of 128000, a quarter of them finished, take 59 us (the read
// of the others 30); with a CTA per 8192 logits and its five barriers it was 180, with the next step in registers 64.
// The comparison between beams needs the differences of nearly equal sums: a lane's sum over a step, and the warp's over its
// lanes, are taken in fp32, a lane's steps are added with what their rounding leaves carried along, and what joins the segments
// and the scores is fp64.
#include <cuda_fp16.h>

#include <algorithm>
#include <cstring>

#include "op_util.hpp"

namespace mlcb {

namespace {

constexpr uint32_t kThreads = 256, kWarps = kThreads / 32;
constexpr uint32_t kCtasPerSm = 3;     // four, with room for two steps a warp: 62 us instead of 61 for 512 rows of 128000
constexpr uint32_t kStep = 512;        // logits a warp takes at a time: four float4 a lane
constexpr uint32_t kRing = 3;          // steps a warp has room for: two are under way while it works on one
constexpr uint32_t kParts = 64;        // maxima a threshold is taken from
constexpr uint32_t kMaxSelect = 64;    // = kParts: a threshold needs that many
constexpr uint32_t kMaxBeams = 64;
constexpr uint32_t kListCap = 128;     // of a warp's list
constexpr uint32_t kFoundCap = 1024;   // of the joining CTA's
constexpr uint32_t kMaxLists = 512;    // segments of a group's rows that one CTA should join
constexpr float kLog2e = 1.4426950408889634f, kLowest = -3.402823466e38f;

struct BeamParams {
    const float* logits;
    const float* cum;
    const uint8_t* finished;   // may be null
    uint64_t* keys;            // [rows * segments][n_select]
    float2* sums;              // [rows * segments] (maximum, sum of exponentials relative to it)
    uint32_t* counters;        // [groups], zero between launches
    float* out_scores;
    uint32_t* out_parents;
    uint32_t* out_tokens;
    uint32_t rows, beams, vocab, group_rows, per_block, segments, segment_len, ctas_per_group, n_select, pad;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// exp(a - b) for a <= b; b > -inf
__device__ __forceinline__ float exp_diff(float a, float b) { return ex2((a - b) * kLog2e); }

// Two fp32 operations in one instruction, on register pairs.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
    return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
    return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float max3(float a, float b, float c) {   // passes over NaN
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

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

// The k-th largest of 64 values in shared memory, by one warp (every lane gets it): the smallest value that fewer than k of
// them exceed.
template <typename T>
__device__ __forceinline__ T kth_of_64(const T* v, uint32_t k, uint32_t lane) {
    const T a = v[lane], b = v[lane + 32];
    uint32_t above_a = 0, above_b = 0;
#pragma unroll 16
    for (uint32_t j = 0; j < 64; ++j) {
        const T x = v[j];
        above_a += x > a;
        above_b += x > b;
    }
    T kth = static_cast<T>(INFINITY);
    if (above_a < k) kth = a;
    if (above_b < k && b < kth) kth = b;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const T x = __shfl_xor_sync(0xffffffffu, kth, o);
        if (x < kth) kth = x;
    }
    return kth;
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
    union {
        float4 ring[kWarps][kRing][kStep / 4];   // logits on their way in
        Candidate found[kFoundCap];
    };
    uint64_t list[kWarps][kListCap];
    uint32_t listed[kWarps];
    float tops[kThreads];
    double lse[kMaxBeams];
    float part[kWarps][kParts];
    Candidate warp_best[kWarps];
    uint32_t count, last;
};

// Joins the segments of one group: run by the CTA that finished last.
__device__ __noinline__ void join_group(const BeamParams& p, Shared& sh, uint32_t group) {
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t row0 = group * p.beams, lists = p.beams * p.segments;
    // the head of this thread's first list is on its way while the sums are joined
    const uint64_t head_key = tid < lists ? __ldcg(&p.keys[(static_cast<size_t>(row0) * p.segments + tid) * p.n_select]) : 0;
    for (uint32_t b = warp; b < p.beams; b += kWarps) {
        const float2* sums = p.sums + static_cast<size_t>(row0 + b) * p.segments;
        float m = -INFINITY;
        double s = 0.0;
        for (uint32_t i = lane; i < p.segments; i += 32) {   // a segment of -inf alone has the sum 0
            const float2 v = __ldcg(sums + i);
            const float both = fmaxf(m, v.x);
            if (both > -INFINITY)
                s = s * static_cast<double>(exp_diff(m, both)) + static_cast<double>(v.y) * static_cast<double>(exp_diff(v.x, both));
            m = both;
        }
        float all = m;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, o));
        if (m > -INFINITY) s *= static_cast<double>(exp_diff(m, all));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        // (a row of -inf alone has no candidates that would use it; one with +inf gives NaN, and so no candidates)
        if (lane == 0) sh.lse[b] = static_cast<double>(all) + log(s);
    }
    if (tid == 0) sh.count = 0;
    __syncthreads();

    // Candidate c of list i: of a segment, largest first, or - behind the segments' lists - the only one of a finished beam.
    auto candidate = [&](uint32_t i, uint32_t c, Candidate& got) {
        if (i >= lists) {
            const uint32_t b = i - lists;
            if (c || !p.finished || !p.finished[row0 + b]) return false;
            got = {static_cast<double>(p.cum[row0 + b]), b, p.pad};
        } else {
            const uint32_t b = i / p.segments;
            if (c >= p.n_select || (p.finished && p.finished[row0 + b])) return false;
            const uint64_t key = i == tid && c == 0
                                     ? head_key : __ldcg(&p.keys[(static_cast<size_t>(row0) * p.segments + i) * p.n_select + c]);
            if (key == 0) return false;
            got = {static_cast<double>(p.cum[row0 + b]) + (static_cast<double>(key_value(key)) - sh.lse[b]), b, key_token(key)};
        }
        return got.score > -INFINITY;   // not for NaN either
    };
    // The n_select-th largest of 64 maxima over parts of the lists' first entries: at least that many candidates reach it. With
    // 64 lists or more a head each is enough, with fewer each gives several.
    const uint32_t deep = min(p.n_select, (2 * kParts - 1) / lists + 1);
    float top = -INFINITY;   // rounded down: no more than a few candidates too many pass
    for (uint32_t i = tid; i < lists * deep + p.beams; i += kThreads) {
        const uint32_t d = i / lists;
        Candidate c;
        if (d < deep ? candidate(i - d * lists, d, c) : candidate(i - lists * deep + lists, 0, c))
            top = fmaxf(top, __double2float_rd(c.score));
    }
    sh.tops[tid] = top;
    __syncthreads();
    if (warp == 0) {
        for (uint32_t i = lane; i < kParts; i += 32)
            sh.tops[i] = fmaxf(fmaxf(sh.tops[i], sh.tops[i + 64]), fmaxf(sh.tops[i + 128], sh.tops[i + 192]));
        __syncwarp();
        const float t = kth_of_64(sh.tops, p.n_select, lane);
        __syncwarp();
        if (lane == 0) sh.tops[0] = t;
    }
    __syncthreads();
    const float threshold = sh.tops[0];
    for (uint32_t i = tid; i < lists + p.beams; i += kThreads) {
        Candidate c;
        for (uint32_t j = 0; candidate(i, j, c) && c.score >= threshold; ++j) {
            const uint32_t at = atomicAdd(&sh.count, 1u);
            if (at < kFoundCap) sh.found[at] = c;
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
    if (n <= kFoundCap) {
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
            for (uint32_t i = tid; i < lists + p.beams; i += kThreads) {
                Candidate c;
                for (uint32_t j = 0; candidate(i, j, c); ++j) {   // the first of a list that is not taken yet is its best
                    if (!first && !better(last, c)) continue;
                    if (better(c, best)) best = c;
                    break;
                }
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
            for (uint32_t w = 1; w < kWarps; ++w)
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

// Keeps the `keep` largest of a warp's n <= 32 * PER listed keys, largest first; returns how many there are.
template <uint32_t PER>
__device__ __forceinline__ uint32_t shorten_to(uint64_t* list, uint32_t n, uint32_t keep, uint32_t lane) {
    uint64_t mine[PER];
    uint32_t rank[PER];
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) {
        mine[i] = lane + 32 * i < n ? list[lane + 32 * i] : 0;
        rank[i] = 0;
    }
#pragma unroll 4
    for (uint32_t j = 0; j < n; ++j) {
        const uint64_t k = list[j];
#pragma unroll
        for (uint32_t i = 0; i < PER; ++i) rank[i] += k > mine[i];
    }
    __syncwarp();
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i)
        if (mine[i] && rank[i] < keep) list[rank[i]] = mine[i];
    __syncwarp();
    return min(n, keep);
}
__device__ __noinline__ uint32_t shorten(uint64_t* list, uint32_t n, uint32_t keep, uint32_t lane) {
    if (n <= 32) return shorten_to<1>(list, n, keep, lane);
    if (n <= 64) return shorten_to<2>(list, n, keep, lane);
    return shorten_to<kListCap / 32>(list, n, keep, lane);
}

// The largest of every four of 16 logits, and of all of them; NaN is passed over.
__device__ __forceinline__ float four_maxima(const float (&x)[16], float (&quarter)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) quarter[j] = fmaxf(max3(x[4 * j], x[4 * j + 1], x[4 * j + 2]), x[4 * j + 3]);
    return fmaxf(max3(quarter[0], quarter[1], quarter[2]), quarter[3]);
}
// Sum of the exponentials of 16 logits, the largest of which is `top`, on top of s, relative to the running maximum m. `left` is what
// the additions before have rounded off (Kahan's summation): a step may be smaller than the sum's last bit for hundreds of steps. 512
// rows of 128000 take 59.3 us so, 60.5 with the sum in fp64, 59.0 without either.
__device__ __forceinline__ void add_step(const float (&x)[16], float top, float& m, float& s, float& left) {
    const float both = fmaxf(m, top), ref = both == -INFINITY ? 0.f : both;
    const float2 minus = make_float2(-ref, -ref), log2e = make_float2(kLog2e, kLog2e);
    float2 t[2] = {};
#pragma unroll
    for (int i = 0; i < 8; ++i) {   // the difference first: its rounding is relative to it, not to the maximum
        const float2 d = mul2(add2(make_float2(x[2 * i], x[2 * i + 1]), minus), log2e);
        t[i & 1] = add2(t[i & 1], make_float2(ex2(d.x), ex2(d.y)));
    }
    t[0] = add2(t[0], t[1]);
    const float scale = exp_diff(m, ref), before = s * scale;
    const float add = left * scale + (t[0].x + t[0].y);
    s = before + add;
    left = add - (s - before);
    m = both;
}

// One segment of a row, by one warp.
__device__ __forceinline__ void segment(const BeamParams& p, float4 (*ring)[kStep / 4], uint64_t* list, uint32_t* listed, float* part,
                                        uint32_t row, uint32_t seg, uint32_t lane) {
    const uint32_t block = seg / p.per_block, begin = (seg - block * p.per_block) * p.segment_len;
    const uint32_t block_rows = min(p.group_rows, p.vocab - block * p.group_rows);
    const int len = begin < block_rows ? static_cast<int>(min(p.segment_len, block_rows - begin)) : 0;   // the last block may be short
    const float* x0 = p.logits + static_cast<size_t>(p.rows) * block * p.group_rows + static_cast<size_t>(row) * block_rows + begin;
    // The body is whole float4s; up to three logits in front of it and behind it are taken first, a lane each.
    const int head = min(static_cast<int>((16u - (static_cast<uint32_t>(reinterpret_cast<uintptr_t>(x0)) & 15u)) & 15u) / 4, len);
    const int vecs = (len - head) / 4, edges = head + ((len - head) & 3);
    const int steps = (vecs + static_cast<int>(kStep / 4) - 1) / static_cast<int>(kStep / 4);
    const uint32_t token0 = block * p.group_rows + begin;
    const float4* body = reinterpret_cast<const float4*>(x0 + head);
    // Loads are the same in every step: a lane whose vector lies behind the body reads the last one again, and drops it.
    auto load = [&](int step, float (&x)[16]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float4 v = __ldcs(body + min(step * static_cast<int>(kStep / 4) + static_cast<int>(lane) + 32 * j, vecs - 1));
            x[4 * j] = v.x; x[4 * j + 1] = v.y; x[4 * j + 2] = v.z; x[4 * j + 3] = v.w;
        }
    };
    // A lane copies to shared memory what it will read itself: no registers wait for the logits, and nothing has to be synchronised
    // but its own copies.
    auto fetch = [&](int step) {
        if (step < steps) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float4* src = body + min(step * static_cast<int>(kStep / 4) + static_cast<int>(lane) + 32 * j, vecs - 1);
                const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(&ring[step % kRing][lane + 32 * j]));
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto drop_behind = [&](int step, float (&x)[16]) {
        if ((step + 1) * static_cast<int>(kStep / 4) <= vecs) return;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (step * static_cast<int>(kStep / 4) + static_cast<int>(lane) + 32 * j >= vecs)
                x[4 * j] = x[4 * j + 1] = x[4 * j + 2] = x[4 * j + 3] = -INFINITY;
    };
    float m = -INFINITY, s = 0.f, left = 0.f, threshold = kLowest;   // (at least the lowest number, so that -inf never passes)
    uint64_t lowest = 0;    // once n_select keys are listed: the n_select-th
    uint32_t n = 0;
    auto clean_up = [&] {
        n = shorten(list, n, p.n_select, lane);
        lowest = list[p.n_select - 1];
        threshold = fmaxf(threshold, key_value(lowest));
        __syncwarp();
    };
#pragma unroll
    for (int i = 0; i < static_cast<int>(kRing) - 1; ++i) fetch(i);
    const int edge_at = static_cast<int>(lane) < head ? static_cast<int>(lane) : 4 * vecs + static_cast<int>(lane);
    const float edge = static_cast<int>(lane) < edges ? x0[edge_at] : -INFINITY;
    if (edges) {
        if (edge > -INFINITY) {
            m = edge;
            s = exp_diff(edge, edge);   // 1, or NaN of +inf
        }
        const uint32_t in = __ballot_sync(0xffffffffu, edge > -INFINITY);
        if ((in >> lane) & 1u) list[__popc(in & ((1u << lane) - 1u))] = make_key(edge + 0.0f, token0 + edge_at);
        n = __popc(in);
        __syncwarp();
    }
#pragma unroll 1
    for (int step = 0; step < steps; ++step) {
        float x[16];
        asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 2) : "memory");
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float4 v = ring[step % kRing][lane + 32 * j];
            x[4 * j] = v.x; x[4 * j + 1] = v.y; x[4 * j + 2] = v.z; x[4 * j + 3] = v.w;
        }
        fetch(step + static_cast<int>(kRing) - 1);   // where the step before this one lay
        drop_behind(step, x);
        float quarter[4];
        const float top = four_maxima(x, quarter);
        add_step(x, top, m, s, left);
        if (step == 0) {   // 64 disjoint parts: at least n_select logits reach the n_select-th largest of their maxima
            // (a part of NaN alone counts as -inf: NaN is never above anything, and the lanes would not agree on a threshold)
            part[lane] = max3(quarter[0], quarter[1], -INFINITY);
            part[lane + 32] = max3(quarter[2], quarter[3], -INFINITY);
            __syncwarp();
            threshold = fmaxf(kLowest, kth_of_64(part, p.n_select, lane));
        }
        if (!__any_sync(0xffffffffu, top >= threshold)) continue;
        const uint32_t token = token0 + head + step * kStep + 4 * lane;
        auto key_of = [&](int i) { return make_key(x[i] + 0.0f, token + 128 * (i >> 2) + (i & 3)); };   // -0 and 0 are one value
        if (lane == 0) *listed = n;
        __syncwarp();
        // Every lane reserves places for all it has and then fetches them from the ring one by one: most have none or one.
        uint32_t mine = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) mine |= x[i] >= threshold ? 1u << i : 0u;
        if (mine) {
            uint32_t at = atomicAdd(listed, static_cast<uint32_t>(__popc(mine)));
            const float* from = reinterpret_cast<const float*>(&ring[step % kRing][lane]);
            for (; mine; mine &= mine - 1, ++at) {
                const uint32_t i = __ffs(mine) - 1, place = 128 * (i >> 2) + (i & 3);
                if (at < kListCap) list[at] = make_key(from[place] + 0.0f, token + place);
            }
        }
        __syncwarp();
        const uint32_t now = *listed;
        __syncwarp();
        if (now <= kListCap) {
            n = now;
        } else {
            // more than there is room for: once more, 32 at a time, with clean-ups in between
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                if (!__any_sync(0xffffffffu, x[i] >= threshold)) continue;
                if (n + 32 > kListCap) clean_up();
                const uint64_t key = key_of(i);
                const uint32_t in = __ballot_sync(0xffffffffu, x[i] >= threshold && key > lowest);
                if ((in >> lane) & 1u) list[n + __popc(in & ((1u << lane) - 1u))] = key;
                n += __popc(in);
                __syncwarp();
            }
        }
        // 12 or more new ones are worth a higher threshold (16 selected of 128000: 60.6 us when the list has doubled, 59.1 so, 61.0 with 4)
        if (n >= p.n_select + max(12u, p.n_select / 2)) clean_up();
    }
    if (__any_sync(0xffffffffu, !(s == s))) {   // NaN among the logits counts as -inf (a sum that +inf spoils stays NaN)
        m = edge > -INFINITY ? edge : -INFINITY;
        s = edge > -INFINITY ? exp_diff(edge, edge) : 0.f;
        left = 0.f;
#pragma unroll 1
        for (int step = 0; step < steps; ++step) {
            float x[16];
            load(step, x);
            drop_behind(step, x);
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (!(x[i] == x[i])) x[i] = -INFINITY;
            float quarter[4];
            add_step(x, four_maxima(x, quarter), m, s, left);
        }
    }
    float top = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    s = m > -INFINITY ? (s + left) * exp_diff(m, top) : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    n = shorten(list, n, p.n_select, lane);
    const size_t unit = static_cast<size_t>(row) * p.segments + seg;
    if (lane == 0) p.sums[unit] = make_float2(top, s);
    for (uint32_t i = lane; i < p.n_select; i += 32) p.keys[unit * p.n_select + i] = i < n ? list[i] : 0;
}

__global__ void __launch_bounds__(kThreads, kCtasPerSm) beam_select_kernel(const __grid_constant__ BeamParams p) {
    extern __shared__ __align__(16) uint8_t smem[];
    Shared& sh = *reinterpret_cast<Shared*>(smem);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t group = blockIdx.x / p.ctas_per_group;
    // (beam, segment) of the group; a CTA's warps are far apart, so that every CTA has its share of a finished beam's idle ones
    const uint32_t unit = warp * p.ctas_per_group + (blockIdx.x - group * p.ctas_per_group);
    if (unit < p.beams * p.segments) {
        const uint32_t row = group * p.beams + unit / p.segments;
        if (!p.finished || !p.finished[row])
            segment(p, sh.ring[warp], sh.list[warp], &sh.listed[warp], sh.part[warp], row, unit % p.segments, lane);
    }
    // the last CTA of the group joins: thread 0 publishes what the CTA wrote, and sees what the others published
    __syncthreads();
    if (tid == 0) {
        __threadfence();
        sh.last = atomicAdd(&p.counters[group], 1u) == p.ctas_per_group - 1 ? 1u : 0u;
        __threadfence();
    }
    __syncthreads();
    if (!sh.last) return;
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
    if (vocab >= (size_t(1) << 30) || groups >= (size_t(1) << 24)) return ctx->fail(MLC_ERR_UNSUPPORTED, "dimension too large");
    if (finished && pad_token >= vocab) return ctx->fail(MLC_ERR_INVALID_ARG, "pad token %u outside the vocabulary", pad_token);
    if (!aligned_to(logits, 4) || !aligned_to(cum, 4) || !aligned_to(out_scores, 4) || !aligned_to(out_parents, 4) ||
        !aligned_to(out_tokens, 4))
        return ctx->fail(MLC_ERR_INVALID_ARG, "buffers must be aligned to their elements");
    if (group_rows == 0 || group_rows > vocab) group_rows = vocab;
    const size_t rows = groups * beams, blocks = (vocab + group_rows - 1) / group_rows;
    // Segments: enough to give every SM its warps once (twice as many take 68 us instead of 61), but no more lists per
    // group than one CTA joins in a few microseconds, and at least a step each.
    const size_t wanted = std::min<size_t>(static_cast<size_t>(ctx->sm_count) * kCtasPerSm * kWarps / rows, kMaxLists / beams);
    size_t per_block = std::min<size_t>(std::max<size_t>(wanted / blocks, 1), (group_rows + kStep - 1) / kStep);
    const size_t segment_len = ((group_rows + per_block - 1) / per_block + 3) / 4 * 4;
    per_block = (group_rows + segment_len - 1) / segment_len;
    const size_t segments = blocks * per_block;
    const size_t ctas_per_group = (beams * segments + kWarps - 1) / kWarps;
    if (rows * segments >= (size_t(1) << 31) || groups * ctas_per_group >= (size_t(1) << 31) ||
        beams * segments * n_select >= (size_t(1) << 31))
        return ctx->fail(MLC_ERR_UNSUPPORTED, "too many rows");
    // a group may still read its scores when another one has written its results
    struct { const void* at; size_t bytes; } in[] = {{logits, rows * vocab * 4}, {cum, rows * 4}, {finished, finished ? rows : 0}};
    const void* out[] = {out_scores, out_parents, out_tokens};
    const size_t out_bytes = groups * n_select * 4;
    for (size_t i = 0; i < 3; ++i) {
        for (const auto& x : in)
            if (overlap(out[i], out_bytes, x.at, x.bytes)) return ctx->fail(MLC_ERR_INVALID_ARG, "an output overlaps an input");
        for (size_t j = 0; j < i; ++j)
            if (overlap(out[i], out_bytes, out[j], out_bytes)) return ctx->fail(MLC_ERR_INVALID_ARG, "two outputs overlap");
    }
    DeviceGuard guard(ctx->device);
    const size_t key_bytes = rows * segments * n_select * 8, sum_bytes = rows * segments * sizeof(float2);
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
    p.per_block = static_cast<uint32_t>(per_block);
    p.segments = static_cast<uint32_t>(segments);
    p.segment_len = static_cast<uint32_t>(segment_len);
    p.ctas_per_group = static_cast<uint32_t>(ctas_per_group);
    p.n_select = static_cast<uint32_t>(n_select);
    p.pad = pad_token;
    if (!ctx->beam_smem_set) {
        MLCB_CUDA(ctx, cudaFuncSetAttribute(beam_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(sizeof(Shared))));
        ctx->beam_smem_set = true;
    }
    static_assert((sizeof(Shared) + 1024) * kCtasPerSm <= 228 * 1024, "CTAs per SM");
    MLCB_CUDA(ctx, launch_dependent(ctx, beam_select_kernel, dim3(static_cast<unsigned>(groups * ctas_per_group)), kThreads, sizeof(Shared), p));
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
