// mla_prefill.cu — causal MLA attention of prompt chunks, expanded form, on
// the 5th-generation tensor cores.
//
// For every sequence (cache rows 0 .. L-1, of which the last T are the chunk's
// own) and head h, with c = c_kv and q = [q_nope | q_rope]:
//   K_h[t] = W_UK[h] c[t]  (128),   V_h[t] = W_UV[h] c[t]  (128)
//   s[i,t] = (q_nope[i] . K_h[t] + q_rope[i] . k_rope[t]) * scale,  t <= L - T + i
//   out[i] = sum_t softmax_t(s[i,t]) V_h[t]
// which is mla_absorbed_attention (weights/store.rs:1179-1327) with the
// products reassociated: 2 x 320 flops per attended pair and head instead of
// the absorbed form's 2 x 1088, for 2 x 512 x 256 flops per cache row and head
// spent once on K and V.
//
// Two launches:
//   1. mla_expand_kernel  K (row-major) and V (transposed) of every head into
//      fp16 workspace rows, each sequence padded to whole 128-row blocks
//      (zeros); the key parts converted to fp16 beside them.
//   2. mla_prefill_kernel flash attention, one CTA per (256 query rows, head).
//
// Operands are fp16 (11 significant bits; bf16 K, V and P would triple the
// error of the output): a query, key part, K or V of magnitude >= 65504 or
// non-finite latches PBMOE_DEV_ERR_F16_RANGE. V is then stored as the nearest
// finite value (0 for NaN) and K as it is, so that a NaN row reaches exactly
// the queries that attend to it: masked scores are selected away, and
// 0 * V stays 0.

#include <cuda.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "kernels.h"
#include "pipe.cuh"
#include "umma.cuh"

namespace pbmoe {

constexpr uint32_t kPfLatent = 512, kPfNope = 128, kPfRope = 64, kPfV = 128, kPfQk = kPfNope + kPfRope;
constexpr uint32_t kPfBlock = 128;              // cache rows per key tile; sequences are padded to it
constexpr uint32_t kPfChunk = kPfBlock * 128;   // [128 rows][64] 16-bit, 128-byte-swizzled: 16 KB

__device__ __forceinline__ uint32_t pf_f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// An f16x2 with an infinity or NaN in either half.
__device__ __forceinline__ bool f16x2_bad(uint32_t v) {
    return (v & 0x7c00u) == 0x7c00u || (v & 0x7c000000u) == 0x7c000000u;
}
// Finite stand-ins of a V pair: +-65504 for overflows, 0 for NaN.
__device__ __forceinline__ uint32_t f16x2_finite(float lo, float hi) {
    lo = lo == lo ? fminf(fmaxf(lo, -65504.f), 65504.f) : 0.f;
    hi = hi == hi ? fminf(fmaxf(hi, -65504.f), 65504.f) : 0.f;
    return pf_f16x2(lo, hi);
}

// Instruction descriptor of kind::f16 with bf16 A and B (format 1).
__host__ __device__ constexpr uint32_t idesc_bf16_f32(uint32_t M, uint32_t N) {
    return idesc_f16_f32(M, N) | (1u << 7) | (1u << 10);
}

// Four tcgen05.ld of 32 columns each with one wait.
__device__ __forceinline__ void tmem_ld32_nowait(uint32_t taddr, uint32_t* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
          "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
          "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr)
        : "memory");
}
// The wait, tied to 32 of the registers so that no use moves above it.
__device__ __forceinline__ void tmem_ld_wait(uint32_t* v) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                   "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]),
                   "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]),
                   "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]),
                   "+r"(v[29]), "+r"(v[30]), "+r"(v[31])
                 :
                 : "memory");
}

// ---------------------------------------------------------------- 1. expand
// D = A B^T over k = 512 in eight 64-wide steps; 128 x 256 output tiles:
//   K tiles  A = 128 cache rows of one block, B = 256 rows of W_UK (two heads)
//   V tiles  A = W_UV[h] (128 rows), B = 256 cache rows (two blocks)
// Persistent CTAs, six warps: loader, MMA issuer, four epilogue warps;
// accumulators double-buffered in TMEM. Both operands bf16 through TMA.
constexpr uint32_t kExThreads = 192, kExStages = 4, kExN = 256, kExSteps = kPfLatent / 64;
constexpr uint32_t kExStage = kPfChunk + 2 * kPfChunk;  // A [128][64], B [256][64]
constexpr size_t kExSmem = 1024 + size_t(kExStages) * kExStage;

// Block index -> its sequence and first row there; false past the last block.
__device__ __forceinline__ bool pf_block(const MlaPrefillSeqs& q, uint32_t blk, uint32_t& seq, uint32_t& row) {
    if (blk >= q.first_block[q.batch]) return false;
    uint32_t b = 0;
    while (q.first_block[b + 1] <= blk) ++b;
    seq = b;
    row = (blk - q.first_block[b]) * kPfBlock;
    return true;
}

__global__ void __launch_bounds__(kExThreads, 1) mla_expand_kernel(const __grid_constant__ MlaExpandParams p) {
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t full[kExStages], empty[kExStages], tfull[2], tempty[2], drain;
    __shared__ uint32_t tmem_base_sh, abort_sh;
    unsigned char* smem =
        reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    volatile uint32_t* abort_flag = &abort_sh;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t blocks = p.seqs.first_block[p.seqs.batch], rows = blocks * kPfBlock;
    const uint32_t pairs = (p.heads + 1) / 2, blk2 = (blocks + 1) / 2;
    const uint32_t k_tiles = blocks * pairs, num_tiles = k_tiles + blk2 * p.heads;

    if (tid == 0) {
        for (uint32_t i = 0; i < kExStages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&tfull[i], 1);
            mbar_init(&tempty[i], 4);
        }
        mbar_init(&drain, 1);
        abort_sh = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(&tmem_base_sh, 2 * kExN);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_sh;

    if (warp == 0) {
        if (lane == 0) {
            uint32_t gs = 0;
            bool ok = true;
            for (uint32_t t = blockIdx.x; ok && t < num_tiles; t += gridDim.x) {
                const bool is_k = t < k_tiles;
                const uint32_t u = is_k ? t : t - k_tiles;
                // K: block u / pairs, head pair u % pairs; V: blocks 2 (u / heads), +1, head u % heads
                uint32_t s0 = 0, r0 = 0, s1 = 0, r1 = 0;
                const uint32_t b0 = is_k ? u / pairs : 2 * (u / p.heads);
                pf_block(p.seqs, b0, s0, r0);
                const bool two = !is_k && pf_block(p.seqs, b0 + 1, s1, r1);
                const int32_t w0 = static_cast<int32_t>(is_k ? (u % pairs) * kExN : (u % p.heads) * kPfV);
                for (uint32_t i = 0; i < kExSteps; ++i, ++gs) {
                    const uint32_t st = gs % kExStages;
                    if (gs >= kExStages && !wait_or_abort(&empty[st], ((gs / kExStages) - 1) & 1, abort_flag, p.status)) {
                        ok = false;
                        break;
                    }
                    unsigned char* a = smem + st * kExStage;
                    const int32_t k0 = static_cast<int32_t>(i * 64);
                    if (is_k) {
                        mbar_arrive_expect_tx(&full[st], 3 * kPfChunk);
                        tma_load_2d(a, &p.tm_c[s0], k0, static_cast<int32_t>(r0), &full[st]);
                        tma_load_2d(a + kPfChunk, &p.tm_uk, k0, w0, &full[st]);
                        tma_load_2d(a + 2 * kPfChunk, &p.tm_uk, k0, w0 + 128, &full[st]);
                    } else {
                        mbar_arrive_expect_tx(&full[st], (two ? 3 : 2) * kPfChunk);
                        tma_load_2d(a, &p.tm_uv, k0, w0, &full[st]);
                        tma_load_2d(a + kPfChunk, &p.tm_c[s0], k0, static_cast<int32_t>(r0), &full[st]);
                        if (two) tma_load_2d(a + 2 * kPfChunk, &p.tm_c[s1], k0, static_cast<int32_t>(r1), &full[st]);
                    }
                }
            }
            if (!ok) {  // give the loads in flight time to land before the CTA exits
                const uint64_t t0 = global_ns();
                while (global_ns() - t0 < 100000ull) __nanosleep(1000);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0) {
            uint32_t gs = 0, lt = 0;
            bool ok = true;
            for (uint32_t t = blockIdx.x; ok && t < num_tiles; t += gridDim.x, ++lt) {
                const uint32_t acc = lt & 1;
                if (lt >= 2 && !wait_or_abort(&tempty[acc], ((lt >> 1) - 1) & 1, abort_flag, p.status)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t d = tmem + acc * kExN;
                for (uint32_t i = 0; i < kExSteps; ++i, ++gs) {
                    const uint32_t st = gs % kExStages;
                    if (!wait_or_abort(&full[st], (gs / kExStages) & 1, abort_flag, p.status)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a = smem_u32(smem + st * kExStage), b = a + kPfChunk;
#pragma unroll
                    for (uint32_t kk = 0; kk < 4; ++kk)
                        umma_f16(d, sw128_kmajor_desc(a + kk * 32), sw128_kmajor_desc(b + kk * 32),
                                 idesc_bf16_f32(128, kExN), (i | kk) != 0u);
                    umma_commit(&empty[st]);
                }
                if (!ok) break;
                umma_commit(&tfull[acc]);
            }
            if (!ok) {
                umma_commit(&drain);
                const uint64_t t0 = global_ns();
                while (!mbar_try_wait_hint(&drain, 0, 20000u) && global_ns() - t0 < kPipeWaitNs) {
                }
            }
        }
        __syncwarp();
    } else {
        bool bad = false;
        // key parts to fp16, zeros in the padding: 8 values a thread and step
        const uint32_t n8 = rows * (kPfRope / 8);
        for (uint32_t i = blockIdx.x * 128 + tid - 64; i < n8; i += gridDim.x * 128) {
            const uint32_t row = i / (kPfRope / 8), c = i % (kPfRope / 8);
            uint32_t s = 0, r = 0;
            pf_block(p.seqs, row / kPfBlock, s, r);
            r += row % kPfBlock;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (r < p.seqs.len[s])
                v = *reinterpret_cast<const uint4*>(p.k_rope[s] + static_cast<size_t>(r) * kPfRope + c * 8);
            const uint32_t in[4] = {v.x, v.y, v.z, v.w};
            uint32_t o[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                o[k] = pf_f16x2(__uint_as_float(in[k] << 16), __uint_as_float(in[k] & 0xffff0000u));
                bad |= f16x2_bad(o[k]);
            }
            reinterpret_cast<uint4*>(p.rope16)[i] = make_uint4(o[0], o[1], o[2], o[3]);
        }
        const uint32_t q = warp & 3, r = 32 * q + lane;
        uint32_t lt = 0;
        for (uint32_t t = blockIdx.x; t < num_tiles; t += gridDim.x, ++lt) {
            const uint32_t acc = lt & 1;
            if (!warp_wait<false>(&tfull[acc], (lt >> 1) & 1, abort_flag, p.status)) break;
            tc_fence_after();
            const bool is_k = t < k_tiles;
            const uint32_t u = is_k ? t : t - k_tiles;
            const uint32_t taddr = tmem + acc * kExN + ((32u * q) << 16);
#pragma unroll 1
            for (uint32_t c0 = 0; c0 < kExN; c0 += 32) {
                uint32_t v[32];
                tmem_ld32(taddr + c0, v);
                uint32_t* dst;
                bool store = true;
                if (is_k) {  // row of block u / pairs, head 2 (u % pairs) + c0 / 128
                    const uint32_t h = 2 * (u % pairs) + c0 / 128;
                    store = h < p.heads;
                    dst = reinterpret_cast<uint32_t*>(
                        p.k16 + (static_cast<size_t>(h) * rows + (u / pairs) * kPfBlock + r) * kPfNope + c0 % 128);
                } else {  // dim r of head u % heads, cache rows 256 (u / heads) + c0 ..
                    const uint32_t col = (u / p.heads) * kExN + c0;
                    store = col < rows;
                    dst = reinterpret_cast<uint32_t*>(
                        p.vt16 + (static_cast<size_t>(u % p.heads) * kPfV + r) * rows + col);
                }
                uint32_t o[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    const float lo = __uint_as_float(v[2 * k]), hi = __uint_as_float(v[2 * k + 1]);
                    o[k] = pf_f16x2(lo, hi);
                    if (store && f16x2_bad(o[k])) {
                        bad = true;
                        if (!is_k) o[k] = f16x2_finite(lo, hi);
                    }
                }
                if (store) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        reinterpret_cast<uint4*>(dst)[k] = make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&tempty[acc]);
        }
        if (bad) latch_status(p.status, PBMOE_DEV_ERR_F16_RANGE);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 2 * kExN);
    }
}

// ---------------------------------------------------------------- 2. attention
// grid (heads, query tiles), 320 threads, one CTA per SM. A CTA takes 256
// query rows of one head as two 128-row halves that share every key tile.
//   warp 0      loader: 16 KB chunks (K: two of K_h, one of the key part; V: two
//               of V_h^T, 64 keys each) through a ring of eight.
//   warp 1      MMA issuer. Half w: S_w = Q_w K^T (TMEM columns 128w ..), then
//               O_w += P_w V with P_w from TMEM (over S_w's first 64 columns).
//               The halves alternate, so one half's softmax runs under the
//               other's MMAs.
//   warps 2-5, 6-9  the halves' softmax, one thread a row: the row's 128 scores
//               in registers, p = 2^(s k - m k) in f32, P to TMEM in fp16. m moves
//               only when the maximum has grown by 2^8 (p then fits fp16 with room),
//               and only then is O_w rescaled.
constexpr uint32_t kPfThreads = 320, kPfRing = 8;
constexpr uint32_t kPfQTile = 128, kPfQBytes = 3 * kPfChunk;
constexpr size_t kPfSmem = 1024 + 2 * size_t(kPfQBytes) + size_t(kPfRing) * kPfChunk;
constexpr float kPfSlack = 8.0f;

// One half's query rows to fp16 in the swizzled K-major layout (three boxes of
// 64 columns), zeros past the chunk; 128 threads, 8 values a step.
template <typename QT>
__device__ __forceinline__ bool pf_load_q(const QT* q, uint32_t stride, uint32_t valid, unsigned char* dst, uint32_t t) {
    bool bad = false;
#pragma unroll 4
    for (uint32_t i = t; i < kPfQTile * (kPfQk / 8); i += 128) {
        const uint32_t row = i / (kPfQk / 8), c = i % (kPfQk / 8);
        float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (row < valid) {
            const QT* src = q + static_cast<size_t>(row) * stride + c * 8;
            if constexpr (sizeof(QT) == 4) {
                const float4 a = reinterpret_cast<const float4*>(src)[0], b = reinterpret_cast<const float4*>(src)[1];
                f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
            } else {
                const uint4 a = *reinterpret_cast<const uint4*>(src);
                const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    f[2 * k] = __uint_as_float(w[k] << 16);
                    f[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
                }
            }
        }
        uint32_t o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            o[k] = pf_f16x2(f[2 * k], f[2 * k + 1]);
            bad |= f16x2_bad(o[k]);
        }
        *reinterpret_cast<uint4*>(dst + (c / 8) * kPfChunk + sw128_offset(row, c % 8)) = make_uint4(o[0], o[1], o[2], o[3]);
    }
    return bad;
}

template <typename QT, typename OT>
__global__ void __launch_bounds__(kPfThreads, 1) mla_prefill_kernel(const __grid_constant__ MlaPrefillParams p) {
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t kvfull[kPfRing], kvempty[kPfRing], qfull[2], sfull[2], pfull[2], pvdone[2], drain;
    __shared__ uint32_t tmem_base_sh, abort_sh;
    unsigned char* smem =
        reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char* ring = smem + 2 * kPfQBytes;
    volatile uint32_t* abort_flag = &abort_sh;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t head = blockIdx.x;
    // query tile -> sequence, the longest rows of a sequence first
    uint32_t b = 0;
    while (p.first_tile[b + 1] <= blockIdx.y) ++b;
    const uint32_t q0 = (p.first_tile[b + 1] - 1 - blockIdx.y) * (2 * kPfQTile);
    const uint32_t qlen = p.q_len[b], ctx = p.seqs.len[b] - qlen;
    // key tiles of each half (the second may have no rows)
    uint32_t nk[2];
#pragma unroll
    for (uint32_t w = 0; w < 2; ++w) {
        const uint32_t first = q0 + w * kPfQTile;
        nk[w] = first < qlen ? (ctx + min(qlen, first + kPfQTile) + kPfBlock - 1) / kPfBlock : 0;
    }
    const uint32_t n = max(nk[0], nk[1]);

    if (tid == 0) {
        for (uint32_t i = 0; i < kPfRing; ++i) {
            mbar_init(&kvfull[i], 1);
            mbar_init(&kvempty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&qfull[i], 4);
            mbar_init(&sfull[i], 1);
            mbar_init(&pfull[i], 4);
            mbar_init(&pvdone[i], 1);
        }
        mbar_init(&drain, 1);
        abort_sh = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(&tmem_base_sh, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_sh;

    if (warp == 0) {
        if (lane == 0) {
            const int32_t row0 = static_cast<int32_t>(p.seqs.first_block[b] * kPfBlock);
            bool ok = true;
            for (uint32_t c = 0; ok && c < 5 * n; ++c) {
                const uint32_t slot = c % kPfRing, j = c / 5, part = c % 5;
                if (c >= kPfRing && !wait_or_abort(&kvempty[slot], ((c / kPfRing) - 1) & 1, abort_flag, p.status)) {
                    ok = false;
                    break;
                }
                unsigned char* dst = ring + slot * kPfChunk;
                const int32_t row = row0 + static_cast<int32_t>(j * kPfBlock);
                mbar_arrive_expect_tx(&kvfull[slot], kPfChunk);
                if (part < 2)
                    tma_load_3d(dst, &p.tm_k, static_cast<int32_t>(part * 64), row, static_cast<int32_t>(head), &kvfull[slot]);
                else if (part == 2)
                    tma_load_2d(dst, &p.tm_rope, 0, row, &kvfull[slot]);
                else
                    tma_load_3d(dst, &p.tm_vt, row + static_cast<int32_t>((part - 3) * 64), 0, static_cast<int32_t>(head),
                                &kvfull[slot]);
            }
            if (!ok) {
                const uint64_t t0 = global_ns();
                while (global_ns() - t0 < 100000ull) __nanosleep(1000);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0) {
            const uint32_t qbase = smem_u32(smem), rbase = smem_u32(ring);
            bool ok = true;
            // chunk c landed (waiting again for a chunk the other half has used is free)
            auto chunk = [&](uint32_t c) {
                ok = ok && wait_or_abort(&kvfull[c % kPfRing], (c / kPfRing) & 1, abort_flag, p.status);
                return rbase + (c % kPfRing) * kPfChunk;
            };
            auto qk = [&](uint32_t w, uint32_t j, bool last_user) {
                for (uint32_t x = 0; x < 3; ++x) {
                    const uint32_t kb = chunk(5 * j + x);
                    if (!ok) return;
                    tc_fence_after();
                    const uint32_t qb = qbase + w * kPfQBytes + x * kPfChunk;
#pragma unroll
                    for (uint32_t kk = 0; kk < 4; ++kk)
                        umma_f16(tmem + w * 128, sw128_kmajor_desc(qb + kk * 32), sw128_kmajor_desc(kb + kk * 32),
                                 idesc_f16_f32(128, 128), (x | kk) != 0u);
                    if (last_user) umma_commit(&kvempty[(5 * j + x) % kPfRing]);
                }
                umma_commit(&sfull[w]);
            };
            // keys past the shorter half's range are used by the other alone
            auto last_user = [&](uint32_t w, uint32_t j) { return w == 1 || j >= nk[1]; };
            for (uint32_t w = 0; ok && w < 2; ++w)
                if (nk[w] > 0) {
                    ok = wait_or_abort(&qfull[w], 0, abort_flag, p.status);
                    if (ok) qk(w, 0, last_user(w, 0));
                }
            for (uint32_t j = 0; ok && j < n; ++j)
                for (uint32_t w = 0; ok && w < 2; ++w) {
                    if (j >= nk[w]) {
                        // K of the next tile and V of this one have no user here; a
                        // tile that only the first half uses is released there
                        continue;
                    }
                    ok = wait_or_abort(&pfull[w], j & 1, abort_flag, p.status);
                    for (uint32_t x = 0; ok && x < 2; ++x) {
                        const uint32_t vb = chunk(5 * j + 3 + x);
                        if (!ok) break;
                        tc_fence_after();
#pragma unroll
                        for (uint32_t kk = 0; kk < 4; ++kk)
                            umma_f16_ts(tmem + 256 + w * 128, tmem + w * 128 + x * 32 + kk * 8,
                                        sw128_kmajor_desc(vb + kk * 32), idesc_f16_f32(128, 128), (j | x | kk) != 0u);
                        if (last_user(w, j)) umma_commit(&kvempty[(5 * j + 3 + x) % kPfRing]);
                    }
                    if (!ok) break;
                    umma_commit(&pvdone[w]);
                    if (j + 1 < nk[w]) {
                        // S_w's next scores overwrite P_w: its readers must be done
                        ok = wait_or_abort(&pvdone[w], j & 1, abort_flag, p.status);
                        if (ok) qk(w, j + 1, last_user(w, j + 1));
                    }
                }
            if (!ok) {
                umma_commit(&drain);
                const uint64_t t0 = global_ns();
                while (!mbar_try_wait_hint(&drain, 0, 20000u) && global_ns() - t0 < kPipeWaitNs) {
                }
            }
        }
        __syncwarp();
    } else {
        const uint32_t w = warp >= 6 ? 1 : 0, quarter = warp & 3, r = 32 * quarter + lane;
        const uint32_t first = q0 + w * kPfQTile;
        if (nk[w] > 0) {
            const uint32_t t = (tid - 64) & 127, valid = min(kPfQTile, qlen - first);
            const QT* q = static_cast<const QT*>(p.query) +
                          (static_cast<size_t>(p.q_first[b] + first) * p.heads + head) * kPfQk;
            const bool bad = pf_load_q(q, p.heads * kPfQk, valid, smem + w * kPfQBytes, t);
            if (bad) latch_status(p.status, PBMOE_DEV_ERR_F16_RANGE);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&qfull[w]);
            const uint32_t lanes = (32u * quarter) << 16;
            const uint32_t ts = tmem + w * 128 + lanes, to = tmem + 256 + w * 128 + lanes;
            const uint32_t limit = ctx + first + r;  // last key this row sees
            const float k = p.scale_log2;
            float m = 0.f, l = 0.f;
            bool ok = true;
            for (uint32_t j = 0; j < nk[w]; ++j) {
                if (!(ok = warp_wait<false>(&sfull[w], j & 1, abort_flag, p.status))) break;
                tc_fence_after();
                uint32_t sr[128];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld32_nowait(ts + 32 * c, sr + 32 * c);
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld_wait(sr + 32 * c);
                float* s = reinterpret_cast<float*>(sr);
                const uint32_t key0 = j * kPfBlock;
                if (key0 + kPfBlock - 1 > ctx + first) {  // some row of the half does not see the whole tile
#pragma unroll
                    for (uint32_t c = 0; c < 128; ++c)
                        if (key0 + c > limit) s[c] = -INFINITY;
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (uint32_t c = 0; c < 128; ++c) mx[c & 3] = fmaxf(mx[c & 3], s[c]);
                const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * k;
                if (j == 0) {
                    m = top > -INFINITY ? top : 0.f;
                } else {
                    const bool over = top > m + kPfSlack;
                    if (__any_sync(kFull, over)) {
                        const float m2 = over ? top : m, alpha = exp2f(m - m2);
                        m = m2;
                        l *= alpha;
#pragma unroll 1
                        for (int c = 0; c < 4; ++c) {
                            uint32_t o[32];
                            tmem_ld32(to + 32 * c, o);
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                            tmem_st32_wait(to + 32 * c, o);
                        }
                    }
                }
                float sum[2] = {0.f, 0.f};
                uint32_t pk[64];
#pragma unroll
                for (int c = 0; c < 64; ++c) {
                    const float p0 = exp2f(fmaf(s[2 * c], k, -m)), p1 = exp2f(fmaf(s[2 * c + 1], k, -m));
                    sum[0] += p0;
                    sum[1] += p1;
                    pk[c] = pf_f16x2(p0, p1);
                }
                l += sum[0] + sum[1];
                tmem_st32_wait(ts, *reinterpret_cast<const uint32_t(*)[32]>(pk));
                tmem_st32_wait(ts + 32, *reinterpret_cast<const uint32_t(*)[32]>(pk + 32));
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&pfull[w]);
            }
            if (ok && warp_wait<false>(&pvdone[w], (nk[w] - 1) & 1, abort_flag, p.status)) {
                tc_fence_after();
                const float inv = 1.0f / l;
                OT* out = static_cast<OT*>(p.out) + (static_cast<size_t>(p.q_first[b] + first + r) * p.heads + head) * kPfV;
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    uint32_t o[32];
                    tmem_ld32(to + 32 * c, o);
                    if (r < valid) {
                        if constexpr (sizeof(OT) == 4) {
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                reinterpret_cast<float4*>(out + 32 * c)[i] =
                                    make_float4(__uint_as_float(o[4 * i]) * inv, __uint_as_float(o[4 * i + 1]) * inv,
                                                __uint_as_float(o[4 * i + 2]) * inv, __uint_as_float(o[4 * i + 3]) * inv);
                        } else {
                            uint32_t h[16];
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                asm("cvt.rn.bf16x2.f32 %0, %1, %2;"
                                    : "=r"(h[i])
                                    : "f"(__uint_as_float(o[2 * i + 1]) * inv), "f"(__uint_as_float(o[2 * i]) * inv));
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                reinterpret_cast<uint4*>(out + 32 * c)[i] =
                                    make_uint4(h[4 * i], h[4 * i + 1], h[4 * i + 2], h[4 * i + 3]);
                        }
                    }
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// ---------------------------------------------------------------- launch
MlaPrefillWs mla_prefill_ws(uint32_t heads, uint32_t blocks) {
    MlaPrefillWs w{};
    const size_t rows = size_t(blocks) * kPfBlock;
    w.k16 = 0;
    w.vt16 = w.k16 + rows * heads * kPfNope * 2;  // multiples of 256 bytes
    w.rope16 = w.vt16 + rows * heads * kPfV * 2;
    w.total = w.rope16 + rows * kPfRope * 2;
    return w;
}

uint32_t mla_prefill_blocks(uint32_t len) { return len / kPfBlock + (len % kPfBlock != 0); }

cudaError_t mla_prefill_launch(const MlaPrefillLaunch& a, int num_sms, cudaStream_t s) {
    const uint32_t blocks = a.seqs.first_block[a.seqs.batch];
    if (blocks == 0) return cudaSuccess;
    const uint64_t rows = uint64_t(blocks) * kPfBlock;
    const MlaPrefillWs w = mla_prefill_ws(a.heads, blocks);
    char* base = static_cast<char*>(a.workspace);
    uint16_t* k16 = reinterpret_cast<uint16_t*>(base + w.k16);
    uint16_t* vt16 = reinterpret_cast<uint16_t*>(base + w.vt16);
    uint16_t* rope16 = reinterpret_cast<uint16_t*>(base + w.rope16);
    cudaError_t e;
    {
        MlaExpandParams p{};
        p.seqs = a.seqs;
        p.heads = a.heads;
        p.k16 = k16;
        p.vt16 = vt16;
        p.rope16 = rope16;
        p.status = a.status;
        for (uint32_t b = 0; b < a.seqs.batch; ++b) {
            p.k_rope[b] = a.k_rope[b];
            if (a.seqs.len[b] == 0) continue;
            if ((e = make_map_16(&p.tm_c[b], true, a.c_kv[b], 2, kPfLatent, a.seqs.len[b], 1, kPfBlock)) != cudaSuccess)
                return e;
        }
        if ((e = make_map_16(&p.tm_uk, true, a.w_uk, 2, kPfLatent, uint64_t(a.heads) * kPfNope, 1, kPfBlock)) != cudaSuccess ||
            (e = make_map_16(&p.tm_uv, true, a.w_uv, 2, kPfLatent, uint64_t(a.heads) * kPfV, 1, kPfBlock)) != cudaSuccess)
            return e;
        if ((e = cudaFuncSetAttribute(mla_expand_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      static_cast<int>(kExSmem))) != cudaSuccess)
            return e;
        const uint64_t tiles = uint64_t(blocks) * ((a.heads + 1) / 2) + uint64_t((blocks + 1) / 2) * a.heads;
        const uint32_t grid = static_cast<uint32_t>(std::min<uint64_t>(tiles, static_cast<uint64_t>(num_sms)));
        mla_expand_kernel<<<grid, kExThreads, kExSmem, s>>>(p);
        if ((e = cudaGetLastError()) != cudaSuccess) return e;
    }
    MlaPrefillParams p{};
    p.seqs = a.seqs;
    p.heads = a.heads;
    p.query = a.query;
    p.out = a.out;
    p.scale_log2 = a.scale * 1.4426950408889634f;
    p.status = a.status;
    uint32_t first = 0;
    uint32_t tiles = 0;
    for (uint32_t b = 0; b < a.seqs.batch; ++b) {
        p.q_len[b] = a.q_len[b];
        p.q_first[b] = first;
        p.first_tile[b] = tiles;
        first += a.q_len[b];
        tiles += a.q_len[b] / (2 * kPfQTile) + (a.q_len[b] % (2 * kPfQTile) != 0);
    }
    for (uint32_t b = a.seqs.batch; b <= kMlaMaxBatch; ++b) p.first_tile[b] = tiles;
    if (tiles == 0) return cudaSuccess;
    if ((e = make_map_16(&p.tm_k, false, k16, 3, kPfNope, rows, a.heads, kPfBlock)) != cudaSuccess ||
        (e = make_map_16(&p.tm_vt, false, vt16, 3, rows, kPfV, a.heads, kPfV)) != cudaSuccess ||
        (e = make_map_16(&p.tm_rope, false, rope16, 2, kPfRope, rows, 1, kPfBlock)) != cudaSuccess)
        return e;
    auto go = [&](auto kernel) {
        cudaError_t r = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kPfSmem));
        if (r != cudaSuccess) return r;
        kernel<<<dim3(a.heads, tiles), kPfThreads, kPfSmem, s>>>(p);
        return cudaGetLastError();
    };
    if (a.q_dtype == PBMOE_F32)
        return a.out_dtype == PBMOE_F32 ? go(mla_prefill_kernel<float, float>) : go(mla_prefill_kernel<float, uint16_t>);
    return a.out_dtype == PBMOE_F32 ? go(mla_prefill_kernel<uint16_t, float>) : go(mla_prefill_kernel<uint16_t, uint16_t>);
}

}  // namespace pbmoe
