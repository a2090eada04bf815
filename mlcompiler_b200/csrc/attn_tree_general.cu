// Attention of drafted tokens over the paged cache, any shape: any head_dim <= 256, any page size, any head grouping,
// fp32 or fp16 Q / O, fp32 arithmetic throughout.
//
//   O[i,h] = sum_s w_s V[s] / sum_s w_s,  w_s = exp(scale q[i,h].K[s]),  s over the committed tokens and the drafted
//   tokens whose bit is set in token i's mask row; a row that sees nothing is zeros.
//
// One CTA per (drafted token, query head): its 4 warps take the tokens round-robin, the 32 lanes of a warp split
// head_dim, every warp keeps its own running maximum, sum and output, and the four states are merged through shared
// memory. A token that is not seen is never read, so whatever lies there has no effect. Every CTA reads its request's
// whole cache, which makes this the kernel for shapes the tensor-core kernel does not take, not for speed.
#include <cuda_fp16.h>

#include "attn_tree.hpp"

namespace mlcb {

namespace {

constexpr int kWarps = 4;
constexpr int kMaxPerLane = 8;   // head_dim <= 256

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__half x) { return __half2float(x); }

template <typename QT, typename OT>
__global__ void __launch_bounds__(kWarps * 32)
paged_tree_general_kernel(const QT* __restrict__ q, const __half* __restrict__ k_pages, const __half* __restrict__ v_pages,
                          OT* __restrict__ o, TreeView t, uint32_t H, uint32_t KVH, uint32_t D, uint32_t P,
                          uint32_t mask_words, float scale, uint32_t capacity, uint32_t* __restrict__ err) {
    const uint32_t token = blockIdx.x / H, head = blockIdx.x % H;
    const uint32_t kv_h = head / (H / KVH);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t req = t.token_req[token];
    const uint32_t prefix = t.prefix[req], S = prefix + t.draft[req];
    const uint32_t* table = t.pt_flat + t.pt_off[req];
    const uint32_t* mask = t.mask + static_cast<size_t>(token) * mask_words;
    const size_t row = (static_cast<size_t>(token) * H + head) * D;
    const size_t page_elems = static_cast<size_t>(P) * KVH * D;

    float qv[kMaxPerLane], acc[kMaxPerLane];
#pragma unroll
    for (int i = 0; i < kMaxPerLane; ++i) {
        const uint32_t d = lane + 32 * i;
        qv[i] = d < D ? as_float(q[row + d]) : 0.0f;
        acc[i] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    for (uint32_t pos = warp; pos < S; pos += kWarps) {
        if (pos >= prefix) {
            const uint32_t j = pos - prefix;
            if (!((mask[j >> 5] >> (j & 31)) & 1u)) continue;
        }
        const uint32_t page = table[pos / P];
        if (page >= capacity) {
            if (lane == 0) atomicOr(err, MLC_DEVERR_BAD_PAGE);
            continue;
        }
        const size_t base = static_cast<size_t>(page) * page_elems + static_cast<size_t>(pos % P) * (static_cast<size_t>(KVH) * D) +
                            static_cast<size_t>(kv_h) * D;
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < kMaxPerLane; ++i) {
            const uint32_t d = lane + 32 * i;
            if (d < D) dot += qv[i] * __half2float(k_pages[base + d]);
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
        const float s = dot * scale;
        if (s == -INFINITY) continue;   // weight 0
        const float m_new = fmaxf(m, s);
        const float alpha = m == -INFINITY ? 0.0f : expf(m - m_new);
        const float p = expf(s - m_new);
        l = l * alpha + p;
#pragma unroll
        for (int i = 0; i < kMaxPerLane; ++i) {
            const uint32_t d = lane + 32 * i;
            if (d < D) acc[i] = acc[i] * alpha + p * __half2float(v_pages[base + d]);
        }
        m = m_new;
    }

    __shared__ float s_m[kWarps], s_l[kWarps];
    __shared__ float s_o[kWarps][kMaxPerLane * 32];
    if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
#pragma unroll
    for (int i = 0; i < kMaxPerLane; ++i) s_o[warp][lane + 32 * i] = acc[i];
    __syncthreads();
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w]);
    float weight[kWarps], sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        // a warp that saw nothing has m = -inf and l = 0; one whose scores were NaN has m = -inf and l = NaN
        weight[w] = s_m[w] == -INFINITY ? (s_l[w] == 0.0f ? 0.0f : 1.0f) : expf(s_m[w] - top);
        sum += s_l[w] * weight[w];
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    for (uint32_t d = threadIdx.x; d < D; d += blockDim.x) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w)
            if (weight[w] != 0.0f) v += s_o[w][d] * weight[w];
        v *= inv;
        if constexpr (sizeof(OT) == 4) o[row + d] = v;
        else o[row + d] = __float2half_rn(v);
    }
}

}  // namespace

int launch_tree_general(mlc_ctx* ctx, const TreeShape& s, const TreeView& v, const TreeArgs& a) {
    const dim3 grid(static_cast<unsigned>(s.tokens * s.H)), block(kWarps * 32);
    const uint32_t cap32 = s.capacity && s.capacity < 0xFFFFFFFFu ? static_cast<uint32_t>(s.capacity) : 0xFFFFFFFFu;
    auto kp = static_cast<const __half*>(a.k_pages);
    auto vp = static_cast<const __half*>(a.v_pages);
#define MLCB_TREE_LAUNCH(QT, OT)                                                                                       \
    paged_tree_general_kernel<QT, OT><<<grid, block, 0, ctx->stream>>>(                                                \
        static_cast<const QT*>(a.q), kp, vp, static_cast<OT*>(a.o), v, static_cast<uint32_t>(s.H),                     \
        static_cast<uint32_t>(s.KVH), static_cast<uint32_t>(s.D), static_cast<uint32_t>(s.P),                          \
        static_cast<uint32_t>(s.mask_words), a.scale, cap32, ctx->d_err)
    if (a.q_dtype == MLC_F32 && a.o_dtype == MLC_F32) MLCB_TREE_LAUNCH(float, float);
    else if (a.q_dtype == MLC_F32) MLCB_TREE_LAUNCH(float, __half);
    else if (a.o_dtype == MLC_F32) MLCB_TREE_LAUNCH(__half, float);
    else MLCB_TREE_LAUNCH(__half, __half);
#undef MLCB_TREE_LAUNCH
    ++ctx->launches;
    MLCB_CUDA(ctx, cudaGetLastError());
    return MLC_OK;
}

}  // namespace mlcb
