// Attention of drafted tokens over the paged cache on the 5th-generation tensor cores: tcgen05.mma with accumulators
// in tensor memory, K and V staged by TMA.
//
// The rows that share a KV head - G heads of every drafted token of a request - are one operand: with 16 drafted
// tokens and a group of 8 they fill the 128 rows of the tensor core's tile, and every K / V tile is read once for all of
// them. Per 64 tokens of the cache:
//   S[128x64]  = Q[128xD] . K^T       A and B from shared memory, fp32 accumulator in tensor memory
//   softmax    : thread t owns row t; reference maximum and sum in fp32, base-2 exponentials, P rounded to fp16 back into
//                tensor memory as the next A operand: 2^-11 of each weight at most, as much as the result's own rounding. The
//                reference is the maximum of the run's first tile and moves up only when the weights outgrow fp16 (exact: the
//                final 1 / l uses the same reference). Its weight is 2^8: fp16 has 15 powers of two above 1 and loses bits
//                below 2^-14, which beside one dominant token is where all others lie; 64 equal weights sum to half the limit
//   O[128xD] += P[128x64] . V
// The tree mask only matters in the tiles that hold drafted tokens, the last ones of a request: there a row's 64 mask
// bits are cut out of its mask words. In those tiles V is also searched for infinities and NaN - a masked token has
// weight 0, and 0 * inf would reach rows that do not see it; they are replaced by 0, and added at the end to the rows
// that do see them.
//
// fp32 queries or outputs (EXACT): an fp16 operand carries 11 bits, so Q (scaled by a power of two per row) and P enter as
// two fp16 halves, two products each; K and V are fp16 as they are. The products of a tile are added to those before it
// outside the tensor core, so every tile has a reference of its own, its maximum, with a weight of 2^15: 22 bits of a weight
// down to 2^-18 of the tile's largest, 2^-40 of the largest below. With one token 9 or 15 nats above 600 equal ones, and of
// value 0, the result is off by 7e-7 and 2e-7 of its size; with the first tile's maximum at 1 it was 2e-4 and 2e-2. (8 requests
// in fp32: 19.1 us, 18.8 with the shared reference.)
//
// What bounds it: the cache is read once, 4 * rows flop per byte - memory up to about 128 rows, the exponentials and the
// tensor core's issue above. The cache tiles of all (request, KV head, row tile) units are dealt evenly to a resident
// grid (attn_tree_plan.cpp); units cut between CTAs leave un-normalised partials that tree_merge_kernel joins, launched as
// a programmatic dependent.
//
// Warps 0-3: softmax and output (warp w reads tensor-memory lanes 32w..32w+31), warp 4: MMA issue, warps 5 / 6: TMA
// producers of K / V, warp 7: none. S is double-buffered so that Q.K^T of tile j+1 runs under the softmax of tile j. No cluster.
#include <cuda.h>
#include <cuda_fp16.h>

#include "attn_tree.hpp"
#include "op_util.hpp"
#include "tcgen05_util.hpp"

namespace mlcb {

namespace {

constexpr uint32_t kSlabQ = kTreeRows * 128;   // 64 halfs of every query row
constexpr uint32_t kSlabKV = kTreeTile * 128;  // 64 halfs of every token of a tile
constexpr uint32_t kThreads = 256;   // two whole warpgroups, for the register split; warp 7 has no work
constexpr uint32_t kRegsSoftmax = 168, kRegsOther = 88;   // registers a thread of the two warpgroups, where they are split
constexpr uint32_t kStageBytes = 32 * 128;     // per softmax warp: 128 bytes of each of its rows, on the way in or out
// Exponent of the reference's weight, and where the sum of a tile's weights has outgrown it (each is below the sum)
constexpr float kRefLog2 = 8.f, kRefLog2Exact = 15.f, kSumLimit = 32768.f;

template <int D, bool EXACT>
struct Config {
    static constexpr uint32_t slabs = D / 64;
    // Q as an operand in tensor memory where there is room beside O and S: read from shared memory, its 128 rows cost
    // every product twice what the 64 rows of K do
    static constexpr bool q_tmem = D == 64 && !EXACT;
    // Columns of tensor memory: O, then Q or (EXACT) the sum over the tiles before, then two S buffers
    static constexpr uint32_t tmem_q = D, tmem_sum = D, tmem_s = D == 128 && EXACT ? 256 : 128;
    static constexpr uint32_t tmem_cols = D == 128 && EXACT ? 512 : 256;
    static constexpr uint32_t q_bytes = q_tmem ? 0 : slabs * kSlabQ * (EXACT ? 2 : 1);
    static constexpr uint32_t kv_bytes = slabs * kSlabKV;   // one tile of K, or of V
    // two CTAs per SM share 226 KB; with D = 128 the two halves of Q leave room for one CTA only
    static constexpr uint32_t ctas = EXACT && D == 128 ? 1 : 2;
    static constexpr uint32_t stages = EXACT ? 4 : D == 64 ? 6 : 2;
    static constexpr uint32_t tile_bytes = q_bytes + stages * 2 * kv_bytes;
    static constexpr uint32_t smem_bytes = tile_bytes + 4 * kStageBytes;   // and the barriers behind that
};

template <uint32_t STAGES>
struct Bars {
    uint64_t q_full, k_full[STAGES], k_empty[STAGES], v_full[STAGES], v_empty[STAGES], s_full[2], p_full[2], pv_done;
    uint32_t tmem_slot;
    uint32_t not_finite[2];   // pieces in turn: a warp may be in the next one before another has read the last one's
};

struct TreeParams {
    const void* q;
    const __half* v_pages;
    void* o;
    float* part_o;    // [slot][slot_rows][D]
    float2* part_ml;  // [slot][slot_rows] (exponent that takes the part to a common scale, sum)
    const TreePiece* pieces;
    const uint32_t *pt_flat, *mask;
    uint32_t* err;
    uint32_t H, KVH, G, P, mask_words, slot_rows;
    uint32_t box_rows, boxes;   // TMA boxes of a tile: boxes * box_rows = 64
    float scale_log2;
    int q_f32, o_f32;
};

using tc::smem_u32;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two fp32 operations in one instruction, on register pairs.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)),
        "l"(*reinterpret_cast<uint64_t*>(&c)));
    return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
    return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ void expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3) : "memory");
}
// A poll that finds the phase open suspends for a while: 2^18 polls are about a second.
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity) {
    for (uint32_t i = 0; i < (1u << 18); ++i)
        if (tc::mbar_try_wait(bar, parity)) return true;
    return false;
}
// The same for a whole warp, which stays together whatever its lanes saw.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)); }
// The A operand from tensor memory: lane = row, one 32-bit column = two consecutive fp16 elements along K.
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
          "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
          "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void st_shared16(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
// fp32 accumulator, fp16 A and B, A K-major, B K-major or MN-major
__host__ __device__ constexpr uint32_t idesc(uint32_t M, uint32_t N, uint32_t b_mn_major) {
    return tc::idesc_f16_kmajor(M, N) | (b_mn_major << 16);
}
__device__ __forceinline__ TreePiece load_piece(const TreePiece* p) {
    TreePiece out;
    const uint4* src = reinterpret_cast<const uint4*>(p);
    uint4* dst = reinterpret_cast<uint4*>(&out);
#pragma unroll
    for (int i = 0; i < 3; ++i) dst[i] = __ldg(src + i);
    return out;
}
// Bit 15 / 31 of the result: the lower / upper fp16 of w is infinite or NaN.
__device__ __forceinline__ uint32_t not_finite(uint32_t w) { return ((w & 0x7C007C00u) + 0x04000400u) & 0x80008000u; }

// Rows of q and o lie a token apart or a head apart; a thread that moves its own row touches 32 lines per instruction and warp.
// The warp moves 128 bytes of four rows at a time instead, eight lanes a row, by way of shared memory, where a thread finds
// its own row. 16-byte chunk c of row r sits at r * 128 + ((c ^ r) & 7) * 16.
__device__ __forceinline__ uint32_t staged(uint32_t stage, uint32_t r, uint32_t c) { return stage + r * 128 + (((c ^ r) & 7u) << 4); }

// 128 bytes, from byte `offset` of this lane's row on (rows of invalid lanes: zeros), into registers: lane i holds chunk i % 8 of
// row i / 8 and of every fourth row behind it.
__device__ __forceinline__ void stage_load(uint4 (&v)[8], uint32_t lane, const char* row, bool valid, uint32_t offset) {
    const uint32_t rows = __ballot_sync(0xffffffffu, valid);
    const uint64_t mine = reinterpret_cast<uint64_t>(row + offset);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t r = 4 * i + (lane >> 3);
        const char* src = reinterpret_cast<const char*>(__shfl_sync(0xffffffffu, mine, r));
        v[i] = (rows >> r) & 1u ? __ldg(reinterpret_cast<const uint4*>(src) + (lane & 7u)) : make_uint4(0, 0, 0, 0);
    }
}
__device__ __forceinline__ void stage_put(uint32_t stage, uint32_t lane, const uint4 (&v)[8]) {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) st_shared16(staged(stage, 4 * i + (lane >> 3), lane & 7u), v[i]);
    __syncwarp();
}

// The reverse: w is 128 bytes of this lane's row.
__device__ __forceinline__ void stage_out(uint32_t stage, uint32_t lane, char* row, bool valid, uint32_t offset, const uint32_t (&w)[32]) {
    const uint32_t rows = __ballot_sync(0xffffffffu, valid);
    const uint64_t mine = reinterpret_cast<uint64_t>(row + offset);
    __syncwarp();
#pragma unroll
    for (int c = 0; c < 8; ++c) st_shared16(staged(stage, lane, c), make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]));
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t r = 4 * i + (lane >> 3);
        char* dst = reinterpret_cast<char*>(__shfl_sync(0xffffffffu, mine, r));
        if ((rows >> r) & 1u) reinterpret_cast<uint4*>(dst)[lane & 7u] = ld_shared16(staged(stage, r, lane & 7u));
    }
}

template <int N>
struct Blocks {
    static constexpr int value = N;
};

// Puts the warp's query rows (zeros for invalid lanes) into the operand tile(s), in shared memory (swizzled) or in tensor
// memory; returns what the lane's scores have to be multiplied with to undo its row's scaling.
template <int D, bool EXACT>
__device__ __forceinline__ float load_queries(uint32_t sQ, uint32_t tQ, uint32_t stage, uint32_t row, const void* q, int q_f32, bool valid,
                                              size_t elem) {
    constexpr bool TMEM = Config<D, EXACT>::q_tmem;
    const uint32_t lane = row & 31u;
    const uint32_t base = sQ + (row >> 3) * 1024u + (row & 7u) * 128u;
    auto to_shared = [&](uint32_t half, uint32_t c, const uint32_t* w) {   // 16 bytes
        st_shared16(base + (half * (D / 64) + (c >> 3)) * kSlabQ + (((c ^ row) & 7u) << 4), make_uint4(w[0], w[1], w[2], w[3]));
    };
    const char* src = static_cast<const char*>(q) + elem * (q_f32 ? 4 : 2);
    if constexpr (!EXACT) {
        uint4 v[D / 64][8];
#pragma unroll
        for (int block = 0; block < D / 64; ++block) stage_load(v[block], lane, src, valid, block * 128);   // 64 halfs
#pragma unroll
        for (int block = 0; block < D / 64; ++block) {
            stage_put(stage, lane, v[block]);
            uint32_t w[32];
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const uint4 x = ld_shared16(staged(stage, lane, c));
                w[4 * c] = x.x; w[4 * c + 1] = x.y; w[4 * c + 2] = x.z; w[4 * c + 3] = x.w;
            }
            if constexpr (TMEM) {
                tmem_st32(tQ, w);
            } else {
#pragma unroll
                for (int c = 0; c < 8; ++c) to_shared(0, block * 8 + c, w + 4 * c);
            }
        }
        if constexpr (TMEM) tmem_wait_st();
        return 1.0f;
    } else {
        // All of the row is under way at once, then each lane finds its own in shared memory and keeps it.
        float scale_down = 1.0f;
        auto run = [&](auto n_blocks, auto column) {
            constexpr int N = decltype(n_blocks)::value;
            uint32_t w[N][32];
            {
                uint4 v[N][8];
#pragma unroll
                for (int i = 0; i < N; ++i) stage_load(v[i], lane, src, valid, i * 128);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    stage_put(stage, lane, v[i]);
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        const uint4 x = ld_shared16(staged(stage, lane, c));
                        w[i][4 * c] = x.x; w[i][4 * c + 1] = x.y; w[i][4 * c + 2] = x.z; w[i][4 * c + 3] = x.w;
                    }
                }
            }
            float top = 0.f;
#pragma unroll
            for (int d = 0; d < D; ++d) top = fmaxf(top, fabsf(column(w, d)));
            // largest magnitude to [2^7, 2^8): well inside fp16, and the low halves stay clear of its subnormals
            int shift = 0;
            if (top > 0.f && top < INFINITY) shift = max(-120, min(120, 7 - ilogbf(top)));
            const float up = __int_as_float((127 + shift) << 23);
            scale_down = __int_as_float((127 - shift) << 23);
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float a = column(w, 8 * c + 2 * i) * up, b = column(w, 8 * c + 2 * i + 1) * up;
                    const __half2 h = __floats2half2_rn(a, b);
                    const float2 back = __half22float2(h);
                    hi[i] = *reinterpret_cast<const uint32_t*>(&h);
                    lo[i] = pack(a - back.x, b - back.y);
                }
                to_shared(0, c, hi);
                to_shared(1, c, lo);
            }
        };
        if (q_f32)
            run(Blocks<D / 32>(), [](const auto& w, int d) { return __uint_as_float(w[d / 32][d % 32]); });
        else
            run(Blocks<D / 64>(), [](const auto& w, int d) {
                const uint32_t x = w[d / 64][d % 64 / 2];
                return __half2float(__ushort_as_half(static_cast<unsigned short>(d % 2 ? x >> 16 : x & 0xFFFFu)));
            });
        return scale_down;
    }
}

template <int D, bool EXACT>
__global__ void __launch_bounds__(kThreads, (Config<D, EXACT>::ctas))
paged_tree_tcgen05_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                          const __grid_constant__ TreeParams prm) {
    using C = Config<D, EXACT>;
    constexpr uint32_t STAGES = C::stages;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    Bars<STAGES>& bars = *reinterpret_cast<Bars<STAGES>*>(smem_raw + C::smem_bytes);
    const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t base = smem_u32(smem_raw);
    if (base & 1023u) {   // the swizzle needs it; never expected
        if (threadIdx.x == 0) atomicOr(prm.err, MLC_DEVERR_WAIT_TIMEOUT | (0x50u << 8));
        return;
    }
    const uint32_t sQ = base, sKV = base + C::q_bytes;   // stage s: K at sKV + s * 2 * kv_bytes, V right behind it
    if (threadIdx.x == 0) {
        tc::mbar_init(smem_u32(&bars.q_full), 128);
        for (uint32_t s = 0; s < STAGES; ++s) {
            tc::mbar_init(smem_u32(&bars.k_full[s]), 1);
            tc::mbar_init(smem_u32(&bars.k_empty[s]), 1);
            tc::mbar_init(smem_u32(&bars.v_full[s]), 1);
            tc::mbar_init(smem_u32(&bars.v_empty[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            tc::mbar_init(smem_u32(&bars.s_full[b]), 1);
            tc::mbar_init(smem_u32(&bars.p_full[b]), 128);   // two, like the S buffers: softmax may be a tile ahead of the MMA warp
        }
        tc::mbar_init(smem_u32(&bars.pv_done), 1);
        bars.not_finite[0] = bars.not_finite[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 4) tc::tmem_alloc(smem_u32(&bars.tmem_slot), C::tmem_cols);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = bars.tmem_slot;
    // The work list and the page tables were uploaded before the kernel in front was launched, and no kernel writes them:
    // they are read before the wait for that kernel.
    TreePiece p = load_piece(prm.pieces + blockIdx.x);
    const uint32_t n_pieces = 1 + p.more, next_piece = p.next;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    // A wait that ran out: which wait (bits 8-15 of the error word) and at which tile (bits 16-31).
    auto give_up = [&](uint32_t where, uint32_t tile) {
        if (lane == 0 && atomicCAS(prm.err, 0u, MLC_DEVERR_WAIT_TIMEOUT | (where << 8) | (tile << 16)) != 0u)
            atomicOr(prm.err, MLC_DEVERR_WAIT_TIMEOUT);
    };

    // Two fp32 CTAs an SM leave a thread 128 registers at launch, and softmax with both halves of P spills: the other warpgroup
    // gives it some (the sum stays 2 * 128). 8 requests in fp32: 19.5 us without, 18.9 with; fp16 does not gain.
    if constexpr (EXACT && C::ctas == 2) {
        if (warp < 4) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
        else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    }
    if (warp == 7) {
        asm volatile("griddepcontrol.wait;" ::: "memory");
    } else if (warp >= 5) {
        // ---------------- TMA producers: warp 5 the K tiles, warp 6 the V tiles ----------------
        // Each has its own ring: a K tile is free when its Q.K^T is done, a V tile only after its P.V.
        const bool is_v = warp == 6;
        const CUtensorMap* map = is_v ? &tmV : &tmK;
        uint64_t* full = is_v ? bars.v_full : bars.k_full;
        uint64_t* empty = is_v ? bars.v_empty : bars.k_empty;
        const uint32_t ring = sKV + (is_v ? C::kv_bytes : 0u);
        if (lane == 0) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
        uint32_t g = 0;   // tiles of this CTA so far
        bool ok = true;
        for (uint32_t pi = 0; ok && pi < n_pieces; ++pi) {
            if (pi) p = load_piece(prm.pieces + next_piece + pi - 1);
            const uint32_t len = p.prefix + p.draft;
            const uint32_t token_begin = p.tile_begin * kTreeTile;
            // boxes of the piece that hold tokens; their page ids are fetched 32 at a time, a lane each
            const uint32_t n_boxes = (min(len, token_begin + p.n_tiles * kTreeTile) - token_begin + prm.box_rows - 1) / prm.box_rows;
            auto fetch_ids = [&](uint32_t box) {
                const uint32_t mine = box + lane;
                return mine < n_boxes ? __ldg(prm.pt_flat + p.pt_off + (token_begin + mine * prm.box_rows) / prm.P) : 0u;
            };
            uint32_t box = 0, ids = fetch_ids(0);
            if (pi == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
            for (uint32_t j = 0; j < p.n_tiles; ++j, ++g) {
                const uint32_t s = g % STAGES;
                if (g >= STAGES && !warp_wait(smem_u32(&empty[s]), (g / STAGES - 1) & 1u)) {
                    give_up(is_v ? 0x31 : 0x30, g);
                    ok = false;
                    break;
                }
                const uint32_t in_tile = min(prm.boxes, n_boxes - box);
                const uint32_t bar = smem_u32(&full[s]), dst = ring + s * 2 * C::kv_bytes;
                if (lane == 0) expect_tx(bar, in_tile * prm.box_rows * D * 2);
                for (uint32_t b = 0; b < in_tile; ++b, ++box) {
                    if (box && (box & 31u) == 0) ids = fetch_ids(box);
                    const int page = static_cast<int>(__shfl_sync(0xffffffffu, ids, box & 31u));
                    const int slot = static_cast<int>((token_begin + box * prm.box_rows) % prm.P);
                    if (lane == 0) {
#pragma unroll
                        for (uint32_t c = 0; c < C::slabs; ++c)
                            tma_load_4d(dst + c * kSlabKV + b * prm.box_rows * 128, map, bar, static_cast<int>(c * 64),
                                        static_cast<int>(p.kv_head), slot, page);
                    }
                }
                __syncwarp();
            }
        }
        if (!ok && lane == 0) {   // copies in flight must land before the CTA ends
            for (uint32_t t = g > STAGES ? g - STAGES : 0; t < g; ++t) wait(smem_u32(&full[t % STAGES]), (t / STAGES) & 1u);
        }
    } else if (warp == 4) {
        // ---------------- MMA issue: the warp walks the loop together, one elected lane issues ----------------
        constexpr uint32_t idesc_qk = idesc(kTreeRows, kTreeTile, 0);   // B = K tile, K-major
        constexpr uint32_t idesc_pv = idesc(kTreeRows, D, 1);           // B = V tile, MN-major
        const uint64_t desc_k = tc::smem_desc_sw128(0, 16, 1024);
        const uint64_t desc_v = tc::smem_desc_sw128(0, kSlabKV, 1024);
        const uint32_t tmem_u = __shfl_sync(0xffffffffu, tmem, 0), sQ_u = __shfl_sync(0xffffffffu, sQ, 0);
        const uint32_t sKV_u = sQ_u + C::q_bytes;
        auto issue_qk = [&](uint32_t g) {
            const uint32_t s = g % STAGES, sK = sKV_u + s * 2 * C::kv_bytes, d = tmem_u + C::tmem_s + (g & 1u) * kTreeTile;
            if (tc::elect_one()) {
#pragma unroll
                for (uint32_t h = 0; h < (EXACT ? 2u : 1u); ++h) {   // the low halves first: fewer roundings at full magnitude
                    const uint32_t half = EXACT ? 1 - h : 0;
#pragma unroll
                    for (uint32_t k = 0; k < D / 16; ++k) {
                        const uint32_t b = sK + (k >> 2) * kSlabKV + (k & 3) * 32;
                        if constexpr (C::q_tmem) {
                            mma_f16_ts(d, tmem_u + C::tmem_q + k * 8, desc_k | (b >> 4), idesc_qk, k > 0);
                        } else {
                            const uint32_t a = sQ_u + (half * C::slabs + (k >> 2)) * kSlabQ + (k & 3) * 32;
                            tc::mma_f16(d, desc_k | (a >> 4), desc_k | (b >> 4), idesc_qk, h + k > 0);
                        }
                    }
                }
                tc::commit(smem_u32(&bars.k_empty[s]));
                tc::commit(smem_u32(&bars.s_full[g & 1u]));
            }
            __syncwarp();
        };
        uint32_t g = 0, where = 0x10, issued_qk = 0, issued_pv = 0;
        bool ok = true;
        auto all_wait = [&](uint64_t* bar, uint32_t parity, uint32_t code) {
            where = code;
            return warp_wait(smem_u32(bar), parity);
        };
        // Q.K^T of tile t: its K has landed, and P of tile t - 2, which lies in the same buffer, has been used. The wait is
        // for the newest P.V issued (t - 2 inside a piece, t - 1 at its start): a parity wait for an older phase would be ambiguous.
        auto start_tile = [&](uint32_t t) {
            if (!all_wait(&bars.k_full[t % STAGES], (t / STAGES) & 1u, 0x11)) return false;
            if (issued_pv && !all_wait(&bars.pv_done, (issued_pv - 1) & 1u, 0x12)) return false;
            tc::fence_after();
            issue_qk(t);
            issued_qk = t + 1;
            return true;
        };
        asm volatile("griddepcontrol.wait;" ::: "memory");
        for (uint32_t pi = 0; ok && pi < n_pieces; ++pi) {
            const uint32_t n_tiles = pi ? __ldg(&prm.pieces[next_piece + pi - 1].n_tiles) : p.n_tiles;
            if (!all_wait(&bars.q_full, pi & 1u, 0x10) || !start_tile(g)) {
                ok = false;
                break;
            }
            for (uint32_t j = 0; j < n_tiles; ++j, ++g) {
                if (j + 1 < n_tiles && !start_tile(g + 1)) { ok = false; break; }   // runs under this tile's softmax
                const uint32_t s = g % STAGES;
                if (!all_wait(&bars.v_full[s], (g / STAGES) & 1u, 0x13) || !all_wait(&bars.p_full[g & 1u], (g >> 1) & 1u, 0x14)) {
                    ok = false;
                    break;
                }
                tc::fence_after();
                const uint32_t sV = sKV_u + s * 2 * C::kv_bytes + C::kv_bytes;
                const uint32_t P = tmem_u + C::tmem_s + (g & 1u) * kTreeTile;
                if (tc::elect_one()) {
#pragma unroll
                    for (uint32_t h = 0; h < (EXACT ? 2u : 1u); ++h)
#pragma unroll
                        for (uint32_t k = 0; k < kTreeTile / 16; ++k)   // 16 tokens per step: 8 columns of P, 16 rows of V
                            mma_f16_ts(tmem_u, P + (EXACT ? 1 - h : 0) * 32 + k * 8, desc_v | ((sV + k * 16 * 128) >> 4), idesc_pv,
                                       (j > 0 && !EXACT) || h + k > 0);
                    tc::commit(smem_u32(&bars.v_empty[s]));
                    tc::commit(smem_u32(&bars.pv_done));
                }
                __syncwarp();
                issued_pv = g + 1;
            }
        }
        if (!ok) {   // nothing may still read shared or tensor memory when the CTA ends
            give_up(where, g);
            if (issued_qk) wait(smem_u32(&bars.s_full[(issued_qk - 1) & 1u]), ((issued_qk - 1) >> 1) & 1u);
            if (issued_pv) wait(smem_u32(&bars.pv_done), (issued_pv - 1) & 1u);
        }
    } else {
        // ---------------- softmax and output: thread = query row ----------------
        const uint32_t row = threadIdx.x, lane_base = (warp * 32u) << 16;
        uint32_t g = 0, where = 0x20;
        bool ok = true;
        float row_down = 1.0f;
        const uint32_t stage = base + C::tile_bytes + warp * kStageBytes;
        auto put_query = [&](const TreePiece& pc) {
            const uint32_t r = pc.row_begin + row;
            const size_t elem = (static_cast<size_t>(pc.token0 + r / prm.G) * prm.H + pc.kv_head * prm.G + r % prm.G) * D;
            row_down = load_queries<D, EXACT>(sQ, tmem + lane_base + C::tmem_q, stage, row, prm.q, prm.q_f32, row < pc.n_rows, elem);
            if constexpr (C::q_tmem) tc::fence_before();
            else tc::fence_proxy_async_smem();
            tc::mbar_arrive(smem_u32(&bars.q_full));
        };
        asm volatile("griddepcontrol.wait;" ::: "memory");
        put_query(p);
        for (uint32_t pi = 0; ok && pi < n_pieces; ++pi) {
            const uint32_t len = p.prefix + p.draft;
            const bool busy = warp * 32u < p.n_rows;   // the warp has rows
            const uint32_t r = p.row_begin + min(row, p.n_rows - 1);
            const uint32_t* mask = prm.mask + static_cast<size_t>(p.token0 + r / prm.G) * prm.mask_words;
            const float scale = prm.scale_log2 * row_down;      // of a raw score, base-2 units
            // A weight is 2^(score * scale + offset), the offset that of the accumulator's reference; infinite: nothing seen yet.
            // It is this rounded number that all factors are taken from, so that its rounding cancels.
            float m_ref = -INFINITY, offset = INFINITY, l_sum = 0.f;   // reference maximum (raw scores), row sum
            float o_factor = 1.0f;                              // EXACT: of the last tile's products, to the reference
            for (uint32_t j = 0; j < p.n_tiles; ++j, ++g) {
                const uint32_t kv0 = (p.tile_begin + j) * kTreeTile;
                where = 0x20;
                ok = warp_wait(smem_u32(&bars.s_full[g & 1u]), (g >> 1) & 1u);
                if (!ok) break;
                tc::fence_after();
                if (busy) {
                    const uint32_t tS = tmem + lane_base + C::tmem_s + (g & 1u) * kTreeTile;
                    uint32_t hi[32], lo[EXACT ? 32 : 1];
                    float alpha = 1.0f;
                    uint32_t s[64];
                    auto load_scores = [&] {
                        {
                            uint32_t a[32], b[32];
                            tc::tmem_ld32(tS, a);
                            tc::tmem_ld32(tS + 32, b);
                            tc::tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; ++i) { s[i] = a[i]; s[32 + i] = b[i]; }
                        }
                        if (kv0 + kTreeTile > p.prefix) {
                            // 64 bits of what the row sees: committed tokens, then its mask from drafted token j0 on
                            const uint32_t committed = p.prefix > kv0 ? p.prefix - kv0 : 0u;
                            const uint32_t j0 = kv0 > p.prefix ? kv0 - p.prefix : 0u;
                            const uint32_t w = j0 >> 5, sh = j0 & 31u;
                            auto word = [&](uint32_t i) { return i < prm.mask_words ? __ldg(mask + i) : 0u; };
                            const uint32_t w0 = word(w), w1 = word(w + 1), w2 = word(w + 2);
                            uint64_t see = static_cast<uint64_t>(__funnelshift_r(w0, w1, sh)) |
                                           (static_cast<uint64_t>(__funnelshift_r(w1, w2, sh)) << 32);
                            if (committed) see = (see << committed) | ((uint64_t(1) << committed) - 1);
                            if (len - kv0 < kTreeTile) see &= (uint64_t(1) << (len - kv0)) - 1;
                            const uint32_t see_lo = static_cast<uint32_t>(see), see_hi = static_cast<uint32_t>(see >> 32);
#pragma unroll
                            for (int c = 0; c < 32; ++c) {
                                if (!((see_lo >> c) & 1u)) s[c] = 0xff800000u;        // -inf
                                if (!((see_hi >> c) & 1u)) s[32 + c] = 0xff800000u;
                            }
                        }
                    };
                    auto largest = [&](float top) {   // fmaxf passes over NaN
#pragma unroll
                        for (int c = 0; c < 64; ++c) top = fmaxf(top, __uint_as_float(s[c]));
                        return top;
                    };
                    auto weights = [&](float from) {   // into hi (and lo); returns their sum
                        const float add = from == INFINITY ? 0.f : from;
                        const float2 scale2 = make_float2(scale, scale), add2s = make_float2(add, add);
                        float2 ps[2] = {};
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const float2 raw = make_float2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1]));
                            float2 x = fma2(raw, scale2, add2s);
                            x = make_float2(ex2(x.x), ex2(x.y));
                            ps[i & 1] = add2(ps[i & 1], x);
                            const __half2 h = __float22half2_rn(x);
                            hi[i] = *reinterpret_cast<const uint32_t*>(&h);
                            if constexpr (EXACT) {
                                const float2 back = __half22float2(h);
                                lo[i] = pack(x.x - back.x, x.y - back.y);
                            }
                        }
                        ps[0] = add2(ps[0], ps[1]);
                        return ps[0].x + ps[0].y;
                    };
                    float before_factor = 1.0f;   // EXACT: o_factor of the tile before
                    if constexpr (EXACT) {
                        load_scores();
                        const float top = largest(-INFINITY);
                        const float own = top == -INFINITY ? INFINITY : fmaf(-top, scale, kRefLog2Exact);
                        const float both = fminf(offset, own);
                        alpha = offset == INFINITY ? 0.f : ex2(both - offset);
                        before_factor = o_factor;
                        o_factor = own == INFINITY ? 0.f : ex2(both - own);
                        offset = both;
                        l_sum = l_sum * alpha + weights(own) * o_factor;
                    } else {
                        // First with the reference as it is, without looking for the tile's maximum: every weight is below the row's
                        // sum over the tile, and while that is below the limit the weights fit fp16. Where some row's sum is not
                        // (or is NaN), and on a run's first tile, the tile is done (again) with a new reference.
                        for (bool moved = j == 0;; moved = true) {
                            load_scores();
                            if (moved) {
                                const float top = largest(m_ref);
                                if (top > m_ref) {
                                    const float from = fmaf(-top, scale, kRefLog2);
                                    alpha = m_ref == -INFINITY ? 0.f : ex2(from - offset);
                                    m_ref = top;
                                    offset = from;
                                }
                                l_sum *= alpha;
                            }
                            const float sum = weights(offset);
                            if (!moved) {
                                if (__any_sync(0xffffffffu, !(sum < kSumLimit) || offset == INFINITY)) continue;
                            } else if (j > 0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
                                where = 0x21;
                                ok = warp_wait(smem_u32(&bars.pv_done), (g - 1) & 1u);   // O may only be touched once P.V is done
                                if (!ok) break;
                                tc::fence_after();
#pragma unroll 1
                                for (int c0 = 0; c0 < D; c0 += 32) {
                                    uint32_t o[32];
                                    tc::tmem_ld32(tmem + lane_base + c0, o);
                                    tc::tmem_wait_ld();
#pragma unroll
                                    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                                    tmem_st32(tmem + lane_base + c0, o);
                                }
                            }
                            l_sum += sum;
                            break;
                        }
                    }
                    if (!ok) break;
                    // P over this tile's scores (own lane, already read): the halves in 32 columns each
                    tmem_st32(tS, hi);
                    if constexpr (EXACT) {
                        tmem_st32(tS + 32, lo);
                        // The tensor core drops what falls below an accumulator's last bit, always towards zero: over a few
                        // hundred tokens that is 1e-6 of the result. So P.V of a tile starts from zero, and the tiles are added
                        // here, rounding to nearest.
                        if (j > 0) {
                            where = 0x26;
                            ok = warp_wait(smem_u32(&bars.pv_done), (g - 1) & 1u);
                            if (!ok) break;
                            tc::fence_after();
#pragma unroll 1
                            for (int c0 = 0; c0 < D; c0 += 32) {
                                uint32_t o[32], sum[32];
                                tc::tmem_ld32(tmem + lane_base + c0, o);
                                if (j > 1) tc::tmem_ld32(tmem + lane_base + C::tmem_sum + c0, sum);
                                tc::tmem_wait_ld();
#pragma unroll
                                for (int i = 0; i < 32; ++i) {
                                    const float before = j > 1 ? __uint_as_float(sum[i]) : 0.f;
                                    sum[i] = __float_as_uint(fmaf(__uint_as_float(o[i]), before_factor, before) * alpha);
                                }
                                tmem_st32(tmem + lane_base + C::tmem_sum + c0, sum);
                            }
                        }
                    }
                    tmem_wait_st();
                }
                if (kv0 + kTreeTile > p.prefix) {
                    // V rows of drafted tokens lose what is not finite, rows behind the last token become zeros
                    const uint32_t s = g % STAGES;
                    where = 0x22;
                    ok = warp_wait(smem_u32(&bars.v_full[s]), (g / STAGES) & 1u);
                    if (!ok) break;
                    const uint32_t from = p.prefix > kv0 ? p.prefix - kv0 : 0u, end = min(len - kv0, kTreeTile);
                    const uint32_t sV = sKV + s * 2 * C::kv_bytes + C::kv_bytes;
                    for (uint32_t i = row; i < (kTreeTile - from) * (D / 8); i += 128) {
                        const uint32_t vr = from + i / (D / 8), c = i % (D / 8);
                        const uint32_t addr = sV + (c >> 3) * kSlabKV + vr * 128 + ((c & 7) << 4);
                        if (vr >= end) {
                            st_shared16(addr, make_uint4(0, 0, 0, 0));
                            continue;
                        }
                        uint4 x = ld_shared16(addr);
                        uint32_t* w = &x.x;
                        uint32_t any = 0;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t bad = not_finite(w[k]);
                            w[k] &= ~((bad >> 15) * 0xFFFFu);
                            any |= bad;
                        }
                        if (any) {
                            st_shared16(addr, x);
                            *reinterpret_cast<volatile uint32_t*>(&bars.not_finite[pi & 1u]) = pi + 1;
                        }
                    }
                    tc::fence_proxy_async_smem();
                }
                // A parity wait for P.V of a tile needs the one before it to be done. For every other wait the tile's scores
                // say so (they were issued behind it); the wait for the run's last P.V below has nothing in between.
                if (j + 1 == p.n_tiles && g > 0) {
                    where = 0x24;
                    ok = warp_wait(smem_u32(&bars.pv_done), (g - 1) & 1u);
                    if (!ok) break;
                }
                tc::fence_before();
                tc::mbar_arrive(smem_u32(&bars.p_full[g & 1u]));
            }
            if (!ok) break;
            // every Q.K^T of this piece is done: the next one's queries may move in while the last P.V runs
            const TreePiece done = p;
            if (pi + 1 < n_pieces) {
                p = load_piece(prm.pieces + next_piece + pi);
                put_query(p);
            }
            where = 0x23;
            ok = warp_wait(smem_u32(&bars.pv_done), (g - 1) & 1u);
            if (!ok) break;
            tc::fence_after();
            if (busy) {
                const bool mine = row < done.n_rows;
                const bool whole = done.slot == kTreeNoSlot;
                const float inv = whole ? (l_sum == 0.f ? 0.f : 1.0f / l_sum) : 1.0f;
                const size_t out = (static_cast<size_t>(done.token0 + r / prm.G) * prm.H + done.kv_head * prm.G + r % prm.G) * D;
                const size_t part = static_cast<size_t>(done.slot) * prm.slot_rows + row;
                const bool repair = *reinterpret_cast<volatile uint32_t*>(&bars.not_finite[pi & 1u]) == pi + 1;
                if (!whole && mine) prm.part_ml[part] = make_float2(-offset, l_sum);
                // drafted tokens of this piece that the row sees: what is not finite in V belongs in its output
                auto put_back = [&](int c0, uint32_t (&o)[32]) {
                    const uint32_t begin = done.tile_begin * kTreeTile, stop = min(len, begin + done.n_tiles * kTreeTile);
                    for (uint32_t pos = max(begin, done.prefix); pos < stop; ++pos) {
                        const uint32_t t = pos - done.prefix;
                        if (!((__ldg(mask + (t >> 5)) >> (t & 31u)) & 1u)) continue;
                        const size_t page = __ldg(prm.pt_flat + done.pt_off + pos / prm.P);
                        const __half* v = prm.v_pages + ((page * prm.P + pos % prm.P) * prm.KVH + done.kv_head) * D + c0;
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const float x = __half2float(v[i]);
                            if (!(fabsf(x) < INFINITY)) o[i] = __float_as_uint(__uint_as_float(o[i]) + x);
                        }
                    }
                };
                const bool wide = !whole || prm.o_f32;   // 4 bytes a column leave, or 2
                char* dst = whole ? static_cast<char*>(prm.o) + out * (prm.o_f32 ? 4 : 2) : reinterpret_cast<char*>(prm.part_o + part * D);
#pragma unroll 1
                for (int c0 = 0; c0 < D; c0 += 64) {
                    uint32_t w[32];
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        uint32_t o[32];
                        tc::tmem_ld32(tmem + lane_base + c0 + 32 * half, o);
                        tc::tmem_wait_ld();
                        if (EXACT && done.n_tiles > 1) {
                            uint32_t sum[32];
                            tc::tmem_ld32(tmem + lane_base + C::tmem_sum + c0 + 32 * half, sum);
                            tc::tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(fmaf(__uint_as_float(o[i]), o_factor, __uint_as_float(sum[i])));
                        }
                        if (repair && mine) put_back(c0 + 32 * half, o);
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * inv);
                        if (wide) {
                            stage_out(stage, lane, dst, mine, (c0 + 32 * half) * 4, o);
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; ++i) w[16 * half + i] = pack(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1]));
                        }
                    }
                    if (!wide) stage_out(stage, lane, dst, mine, c0 * 2, w);
                }
            }
        }
        if (!ok) give_up(where, g);
    }
    // every tcgen05 operation is finished: free the tensor memory
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    if (warp == 4) tc::tmem_dealloc(tmem, C::tmem_cols);
}

// O of the rows whose run was cut: sum_k o_k 2^(m_k - m) / sum_k l_k 2^(m_k - m), parts in fixed order. A row has SHARES groups of
// D / 4 threads, four columns a thread; a group takes every SHARES-th part, four in flight. The tables are read before the
// wait for the kernel in front.
constexpr uint32_t merge_rows_per_cta(int D, int shares) { return D / 4 * shares < 128 ? 512 / (D * shares) : 1; }

template <int D, int SHARES, typename OT>
__global__ void __launch_bounds__(D / 4 * SHARES * merge_rows_per_cta(D, SHARES))
tree_merge_kernel(const float* __restrict__ part_o, const float2* __restrict__ part_ml, const TreeSplit* __restrict__ splits,
                  const uint32_t* __restrict__ row_split, OT* __restrict__ o, uint32_t rows, uint32_t slot_rows, uint32_t H, uint32_t G) {
    constexpr uint32_t kLanes = D / 4, kFlight = 4, kRows = merge_rows_per_cta(D, SHARES);
    __shared__ float4 s_o[kRows][SHARES][kLanes];
    __shared__ float2 s_ml[kRows][SHARES];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t column = threadIdx.x % kLanes, share = threadIdx.x / kLanes % SHARES, in_cta = threadIdx.x / (kLanes * SHARES);
    const uint32_t row = min(blockIdx.x * kRows + in_cta, rows - 1);   // (the last CTA may work on the last row several times)
    const TreeSplit sp = splits[row_split[row]];
    const uint32_t r = row - sp.first_row;
    auto index = [&](uint32_t k) { return static_cast<size_t>(sp.first_slot + k * sp.slot_step) * slot_rows + r; };
    asm volatile("griddepcontrol.wait;" ::: "memory");
    float top = -INFINITY, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float2 ml, float4 v) {   // a part that saw nothing has m = -inf, l = 0 and o = 0
        const float w = ml.x == -INFINITY ? 1.0f : ex2(ml.x - top);
        l += ml.y * w;
        acc.x += v.x * w; acc.y += v.y * w; acc.z += v.z * w; acc.w += v.w * w;
    };
    for (uint32_t k0 = share; k0 < sp.n_parts; k0 += SHARES * kFlight) {
        float2 ml[kFlight];
        float4 v[kFlight];
#pragma unroll
        for (uint32_t i = 0; i < kFlight; ++i) {
            const uint32_t k = k0 + i * SHARES;
            ml[i] = make_float2(-INFINITY, 0.f);
            v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (k < sp.n_parts) {
                ml[i] = __ldcg(&part_ml[index(k)]);
                v[i] = __ldcg(reinterpret_cast<const float4*>(part_o + index(k) * D) + column);
            }
        }
        float both = top;
#pragma unroll
        for (uint32_t i = 0; i < kFlight; ++i) both = fmaxf(both, ml[i].x);
        const float w = top == -INFINITY ? 0.f : ex2(top - both);
        top = both;
        l *= w;
        acc.x *= w; acc.y *= w; acc.z *= w; acc.w *= w;
#pragma unroll
        for (uint32_t i = 0; i < kFlight; ++i) add(ml[i], v[i]);
    }
    if constexpr (SHARES > 1) {
        if (column == 0) s_ml[in_cta][share] = make_float2(top, l);
        s_o[in_cta][share][column] = acc;
        __syncthreads();
        if (share) return;
        for (int i = 1; i < SHARES; ++i) top = fmaxf(top, s_ml[in_cta][i].x);
        l = 0.f;
        acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < SHARES; ++i) add(s_ml[in_cta][i], s_o[in_cta][i][column]);
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    const uint32_t rr = sp.row_begin + r;
    OT* dst = o + (static_cast<size_t>(sp.token0 + rr / G) * H + sp.kv_head * G + rr % G) * D + column * 4;
    if constexpr (sizeof(OT) == 4) *reinterpret_cast<float4*>(dst) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    else *reinterpret_cast<uint2*>(dst) = make_uint2(pack(acc.x * inv, acc.y * inv), pack(acc.z * inv, acc.w * inv));
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int pool_map(mlc_ctx* ctx, CUtensorMap* out, const void* pool, const TreeShape& s, uint32_t box_rows) {
    if (!ctx->tmap_encode_fn) {
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ctx->tmap_encode_fn, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess || !ctx->tmap_encode_fn)
            return ctx->fail(MLC_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
    }
    const cuuint64_t dims[4] = {s.D, s.KVH, s.P, s.capacity};
    const cuuint64_t strides[3] = {s.D * 2, s.KVH * s.D * 2, s.P * s.KVH * s.D * 2};
    const cuuint32_t box[4] = {64, 1, box_rows, 1}, unit[4] = {1, 1, 1, 1};
    const CUresult r = reinterpret_cast<EncodeTiledFn>(ctx->tmap_encode_fn)(
        out, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(pool), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return ctx->fail(MLC_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
    return MLC_OK;
}

template <int D, typename OT>
cudaError_t merge_launch(mlc_ctx* ctx, const TreeShape& s, const TreeWorkView& v, const float* part_o, const float2* part_ml, void* o) {
    auto go = [&](auto n_shares) {
        constexpr int SHARES = decltype(n_shares)::value;
        constexpr uint32_t kRows = merge_rows_per_cta(D, SHARES);
        return launch_dependent(ctx, tree_merge_kernel<D, SHARES, OT>, dim3((v.merge_rows + kRows - 1) / kRows), D / 4 * SHARES * kRows, 0,
                                part_o, part_ml, v.splits, v.row_split, static_cast<OT*>(o), v.merge_rows, v.slot_rows,
                                static_cast<uint32_t>(s.H), static_cast<uint32_t>(s.H / s.KVH));
    };
    // More threads a row where there are parts for them and room: beyond the threads that are resident at once, the waiting
    // of a second wave costs more.
    const uint64_t room = static_cast<uint64_t>(ctx->sm_count) * 1280 / (static_cast<uint64_t>(v.merge_rows) * (D / 4));
    constexpr int kMost = D == 64 ? 16 : 8;
    if (v.max_parts > 16 && room >= kMost) return go(Blocks<kMost>());
    if (v.max_parts > 4 && room >= 4) return go(Blocks<4>());
    return go(Blocks<1>());
}

template <int D, bool EXACT>
int launch_t(mlc_ctx* ctx, const TreeShape& s, const TreeView& v, const TreeArgs& a) {
    using C = Config<D, EXACT>;
    constexpr size_t smem = C::smem_bytes + sizeof(Bars<C::stages>);
    static_assert((smem + 1024) * C::ctas <= 228 * 1024, "CTAs per SM");
    const TreeWorkView& w = v.work[C::ctas == 1 ? 1 : 0];
    const uint32_t box_rows = static_cast<uint32_t>(s.P < kTreeTile ? s.P : kTreeTile);
    CUtensorMap mk, mv;
    int st = pool_map(ctx, &mk, a.k_pages, s, box_rows);
    if (st == MLC_OK) st = pool_map(ctx, &mv, a.v_pages, s, box_rows);
    if (st != MLC_OK) return st;
    bool& opted = ctx->tree_smem_set[(D == 128 ? 2 : 0) + (EXACT ? 1 : 0)];
    if (!opted) {
        if (EXACT && C::ctas == 2) {   // a split that asks for more than the launch has would wait for ever
            cudaFuncAttributes attr{};
            MLCB_CUDA(ctx, cudaFuncGetAttributes(&attr, paged_tree_tcgen05_kernel<D, EXACT>));
            if ((attr.numRegs + 7) / 8 * 8 < static_cast<int>(kRegsSoftmax + kRegsOther) / 2)
                return ctx->fail(MLC_ERR_CUDA, "the tree attention kernel was compiled for %d registers a thread", attr.numRegs);
        }
        MLCB_CUDA(ctx, cudaFuncSetAttribute(paged_tree_tcgen05_kernel<D, EXACT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            static_cast<int>(smem)));
        opted = true;
    }
    TreeParams p{};
    p.q = a.q;
    p.v_pages = static_cast<const __half*>(a.v_pages);
    p.o = a.o;
    if (w.n_slots) {
        p.part_o = static_cast<float*>(ctx->tree_scratch.dev);
        p.part_ml = reinterpret_cast<float2*>(p.part_o + static_cast<size_t>(w.n_slots) * w.slot_rows * D);
    }
    p.pieces = w.pieces;
    p.pt_flat = v.pt_flat;
    p.mask = v.mask;
    p.err = ctx->d_err;
    p.H = static_cast<uint32_t>(s.H);
    p.KVH = static_cast<uint32_t>(s.KVH);
    p.G = static_cast<uint32_t>(s.H / s.KVH);
    p.P = static_cast<uint32_t>(s.P);
    p.mask_words = static_cast<uint32_t>(s.mask_words);
    p.slot_rows = w.slot_rows;
    p.box_rows = box_rows;
    p.boxes = kTreeTile / box_rows;
    p.scale_log2 = a.scale * 1.4426950408889634f;
    p.q_f32 = a.q_dtype == MLC_F32;
    p.o_f32 = a.o_dtype == MLC_F32;
    MLCB_CUDA(ctx, launch_dependent(ctx, paged_tree_tcgen05_kernel<D, EXACT>, dim3(w.n_cta), kThreads, smem, mk, mv, p));
    ++ctx->launches;
    if (!w.n_slots) return MLC_OK;
    if (a.o_dtype == MLC_F32) MLCB_CUDA(ctx, (merge_launch<D, float>(ctx, s, w, p.part_o, p.part_ml, a.o)));
    else MLCB_CUDA(ctx, (merge_launch<D, __half>(ctx, s, w, p.part_o, p.part_ml, a.o)));
    ++ctx->launches;
    return MLC_OK;
}

}  // namespace

bool tree_tcgen05_shape(const TreeShape& s) {
    const bool pages = s.P % kTreeTile == 0 || s.P == 32 || s.P == 16;
    return (s.D == 64 || s.D == 128) && pages && s.capacity > 0 && s.capacity < (size_t(1) << 31) && s.P < (size_t(1) << 31) &&
           s.KVH < (size_t(1) << 31) && s.P * s.KVH * s.D * 2 < (size_t(1) << 40);
}

bool tree_tcgen05_buffers(const TreeArgs& a) {
    return aligned_to(a.q, 16) && aligned_to(a.o, 16) && aligned_to(a.k_pages, 16) && aligned_to(a.v_pages, 16);
}

size_t tree_scratch_bytes(const TreeShape& s, uint32_t n_slots, uint32_t slot_rows) {
    return static_cast<size_t>(n_slots) * slot_rows * (s.D * sizeof(float) + sizeof(float2));
}

int launch_tree_tcgen05(mlc_ctx* ctx, const TreeShape& s, const TreeView& v, const TreeArgs& a) {
    const bool exact = a.q_dtype == MLC_F32 || a.o_dtype == MLC_F32;
    if (s.D == 64) return exact ? launch_t<64, true>(ctx, s, v, a) : launch_t<64, false>(ctx, s, v, a);
    return exact ? launch_t<128, true>(ctx, s, v, a) : launch_t<128, false>(ctx, s, v, a);
}

}  // namespace mlcb
