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
// Two launches (three where query tiles are cut):
//   1. mla_expand_kernel  K and V of every head into fp16 workspace rows, each
//      sequence padded to whole 128-row blocks (zeros); the key parts converted
//      to fp16 beside them.
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

// Two f32 operations in one instruction (fma.rn.f32x2, add.rn.f32x2).
__device__ __forceinline__ uint64_t f32x2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 f32x2_get(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// 2^x by the special function unit, results below 2^-126 flushed to 0 (a
// weight that fp16 would not keep either).
__device__ __forceinline__ float ex2_ftz(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// 2^x of a pair in the FMA units, for a share of the weights (the special
// function unit's 4 lanes a cycle and scheduler bound a softmax of this size):
// x = n + f with n the nearest integer, 2^f for |f| <= 1/2 by the cubic of
// least relative error (fitted by the Remez exchange: 7.5e-5 = 2^-13.7, below
// the 2^-11 of p's rounding to fp16), times 2^n from n's bits. x is held at
// -126, where the weight rounds to 0 in fp16.
__device__ __forceinline__ float2 exp2_poly(uint64_t x) {
    const float2 v = f32x2_get(x);
    x = f32x2(max_nan(v.x, -126.f), max_nan(v.y, -126.f));
    const uint64_t magic = f32x2(12582912.f, 12582912.f), mone = f32x2(-1.f, -1.f);  // 1.5 * 2^23
    const uint64_t t = add2(x, magic);
    const uint64_t f = fma2(add2(t, f32x2(-12582912.f, -12582912.f)), mone, x);
    uint64_t p = fma2(f32x2(0.0551716685295105f, 0.0551716685295105f), f,
                      f32x2(0.2426111251115799f, 0.2426111251115799f));
    p = fma2(p, f, f32x2(0.6932609677314758f, 0.6932609677314758f));
    p = fma2(p, f, f32x2(0.9999280571937561f, 0.9999280571937561f));
    const float2 ti = f32x2_get(t);  // low bits: n; 2^n as a factor, so that NaN stays NaN
    return f32x2_get(mul2(p, f32x2(__uint_as_float((__float_as_uint(ti.x) << 23) + 0x3f800000u),
                                   __uint_as_float((__float_as_uint(ti.y) << 23) + 0x3f800000u))));
}
// Maximum of three (NaN operands are dropped, as fmaxf does).
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// 16 consecutive 32-bit TMEM columns of this thread's lane, not waited for.
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
            taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
        "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Bounded wait of the attention kernel's roles: polls that each suspend for up
// to 20 us, 100000 of them (2 s of a wait that takes microseconds), given up
// early when another role has. Short on purpose: the roles share instruction
// caches, and a loop that is not resident costs more than the wait.
__device__ __forceinline__ bool pf_wait(uint64_t* bar, uint32_t parity, volatile uint32_t* abort_flag,
                                        uint32_t* status) {
    if (mbar_try_wait(bar, parity)) return true;
#pragma unroll 1
    for (uint32_t i = 0; i < 100000u && *abort_flag == 0; ++i)
        if (mbar_try_wait_hint(bar, parity, 20000u)) return true;
    *abort_flag = 1u;
    latch_status(status, PBMOE_DEV_ERR_PIPE_TIMEOUT);
    return false;
}

// ---------------------------------------------------------------- 1. expand
// One unit = one 128 x 128 output over k = 512: K or V of a head for a 128-row
// block of the cache (A = cache rows, B = W_UK[h] or W_UV[h]). A CTA takes a run
// of units in block order and keeps the block's rows (128 KB) in shared memory,
// so that only W streams, through a ring of four 16 KB places; a unit is eight
// places, so that slots, phases and operand addresses are constants of the
// unrolled loops (with them computed, the issuer's loop took 430 cycles a step
// beside 256 of MMAs). Roles: loader, MMA issuer, two groups of four epilogue
// warps that take turns (one group took 5500 cycles a unit); four accumulators
// in TMEM; outputs go through a staging box a group and TMA stores.
// Measured, 8192 rows x 16 heads: 42 us, 34 GFLOP, 0.82 PFLOP/s: the MMAs' operand
// reads, W's arrival and the outputs share the shared memory.
constexpr uint32_t kExThreads = 320, kExRing = 4, kExAcc = 4, kExN = 128, kExSteps = kPfLatent / 64;
static_assert(kExSteps == 2 * kExRing, "a unit goes round the ring twice");
constexpr size_t kExSmem = 1024 + size_t(kExSteps + kExRing + 2) * kPfChunk;  // rows, W, two staging boxes

// Block index -> its sequence and first row there.
__device__ __forceinline__ void pf_block(const MlaPrefillSeqs& q, uint32_t blk, uint32_t& seq, uint32_t& row) {
    uint32_t b = 0;
    while (q.first_block[b + 1] <= blk) ++b;
    seq = b;
    row = (blk - q.first_block[b]) * kPfBlock;
}

// TMA store of one box, and the waits for a thread's own stores.
__device__ __forceinline__ void tma_store_3d(const void* tmap, const void* src, int32_t c0, int32_t c1, int32_t c2) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(
                     reinterpret_cast<uint64_t>(tmap)),
                 "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(src))
                 : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

__global__ void __launch_bounds__(kExThreads, 1) mla_expand_kernel(const __grid_constant__ MlaExpandParams p) {
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t afull, aempty, full[kExRing], empty[kExRing], tfull[kExAcc], tempty[kExAcc], drain;
    __shared__ uint32_t tmem_base_sh, abort_sh;
    unsigned char* smem =
        reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char* ring = smem + kExSteps * kPfChunk;
    unsigned char* stage = ring + kExRing * kPfChunk;
    volatile uint32_t* abort_flag = &abort_sh;
    const uint32_t tid = threadIdx.x, lane = tid & 31;
    const uint32_t warp = __shfl_sync(kFull, tid >> 5, 0);  // warp-uniform for the compiler too
    const uint32_t blocks = p.seqs.first_block[p.seqs.batch], rows = blocks * kPfBlock;
    const uint32_t per = 2 * p.heads;  // units of a block: K of every head, then V
    const uint64_t units = uint64_t(blocks) * per;
    const uint64_t u0 = units * blockIdx.x / gridDim.x, u1 = units * (blockIdx.x + 1) / gridDim.x;

    if (tid == 0) {
        mbar_init(&afull, 1);
        mbar_init(&aempty, 1);
        for (uint32_t i = 0; i < kExRing; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (uint32_t i = 0; i < kExAcc; ++i) {
            mbar_init(&tfull[i], 1);
            mbar_init(&tempty[i], 4);
        }
        mbar_init(&drain, 1);
        abort_sh = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(&tmem_base_sh, kExAcc * kExN);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // (every thread: the workspace is free, the cache rows are written; what the
    // attention kernel reads before its own wait is older still)
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t tmem = tmem_base_sh;

    if (warp == 0) {
        if (lane == 0) {
            uint32_t loads = 0, have = 0xffffffffu;
            bool ok = true;
            for (uint64_t u = u0; ok && u < u1; ++u) {
                const uint32_t blk = static_cast<uint32_t>(u / per), j = static_cast<uint32_t>(u % per);
                if (blk != have) {
                    have = blk;
                    if (loads > 0) ok = pf_wait(&aempty, (loads - 1) & 1, abort_flag, p.status);
                    if (!ok) break;
                    ++loads;
                    uint32_t s, r;
                    pf_block(p.seqs, blk, s, r);
                    mbar_arrive_expect_tx(&afull, kExSteps * kPfChunk);
                    for (uint32_t i = 0; i < kExSteps; ++i)
                        tma_load_2d(smem + i * kPfChunk, &p.tm_c[s], static_cast<int32_t>(i * 64), static_cast<int32_t>(r),
                                    &afull);
                }
                const void* map = j < p.heads ? &p.tm_uk : &p.tm_uv;
                const int32_t w0 = static_cast<int32_t>(j % p.heads * kExN);
#pragma unroll
                for (uint32_t i = 0; i < kExSteps; ++i) {
                    uint64_t* f = &full[i % kExRing];
                    if (ok && (u > u0 || i >= kExRing))
                        ok = pf_wait(&empty[i % kExRing], (i / kExRing + 1) & 1, abort_flag, p.status);
                    if (ok) {
                        mbar_arrive_expect_tx(f, kPfChunk);
                        tma_load_2d(ring + (i % kExRing) * kPfChunk, map, static_cast<int32_t>(i * 64), w0, f);
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
        const bool leader = elect_one();
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t parity) {
            return __all_sync(kFull, pf_wait(bar, parity, abort_flag, p.status)) != 0;
        };
        // units to the block's end (broadcast: the loops then have warp-uniform
        // bounds, and the operands stay in uniform registers)
        uint32_t left = __shfl_sync(kFull, per - static_cast<uint32_t>(u0 % per), 0);
        const uint32_t total = __shfl_sync(kFull, static_cast<uint32_t>(u1 - u0), 0);
        const uint32_t tmem = __shfl_sync(kFull, tmem_base_sh, 0);
        const uint32_t a0 = smem_u32(smem), w0 = smem_u32(ring);
        uint32_t loads = 0;
        bool fresh = true;
        for (uint32_t lt = 0; ok && lt < total; ++lt) {
            const uint32_t acc = lt % kExAcc, d = tmem + acc * kExN;
            if (fresh) ok = wait(&afull, loads++ & 1);
            fresh = --left == 0 || lt + 1 == total;  // the block's last unit here
            if (ok && lt >= kExAcc) ok = wait(&tempty[acc], ((lt / kExAcc) - 1) & 1);
            tc_fence_after();
#pragma unroll
            for (uint32_t i = 0; i < kExSteps; ++i) {
                ok = ok && wait(&full[i % kExRing], (i / kExRing) & 1);
                if (ok && leader) {
#pragma unroll
                    for (uint32_t kk = 0; kk < 4; ++kk)
                        umma_f16(d, sw128_kmajor_desc(a0 + i * kPfChunk + kk * 32),
                                 sw128_kmajor_desc(w0 + (i % kExRing) * kPfChunk + kk * 32), idesc_bf16_f32(128, kExN),
                                 (i | kk) != 0u);
                    umma_commit(&empty[i % kExRing]);
                    if (i + 1 == kExSteps) {
                        umma_commit(&tfull[acc]);
                        if (fresh) umma_commit(&aempty);
                    }
                }
                __syncwarp();
            }
            if (left == 0) left = per;
        }
        if (!ok && leader) {
            umma_commit(&drain);
            const uint64_t t0 = global_ns();
            while (!mbar_try_wait_hint(&drain, 0, 20000u) && global_ns() - t0 < kPipeWaitNs) {
            }
        }
        __syncwarp();
    } else {
        bool bad = false;
        // key parts to fp16, zeros in the padding: 8 values a thread and step
        const uint32_t n8 = rows * (kPfRope / 8);
        for (uint32_t i = blockIdx.x * 256 + tid - 64; i < n8; i += gridDim.x * 256) {
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
        const uint32_t group = (tid - 64) / 128;
        const bool issuer = (tid - 64) % 128 == 0;
        const int bar = 1 + 2 * static_cast<int>(group);
        unsigned char* st = stage + group * kPfChunk;
        uint32_t lt = group;
        for (uint64_t u = u0 + group; u < u1; u += 2, lt += 2) {
            const uint32_t blk = static_cast<uint32_t>(u / per), j = static_cast<uint32_t>(u % per), acc = lt % kExAcc;
            const bool is_k = j < p.heads;
            const bool ok = warp_wait<false>(&tfull[acc], (lt / kExAcc) & 1, abort_flag, p.status);
            tc_fence_after();
            if (issuer) bulk_wait_read();  // the staging box is free
            if (named_sync_or(bar, 128, !ok)) break;  // all four warps leave together
            for (uint32_t x = 0; x < 2; ++x) {  // 64 columns
                if (x == 1) {
                    if (issuer) bulk_wait_read();
                    named_sync(bar, 128);
                }
#pragma unroll
                for (uint32_t c0 = 0; c0 < 64; c0 += 32) {
                    uint32_t v[32], o[16];
                    tmem_ld32(tmem + acc * kExN + x * 64 + ((32u * q) << 16) + c0, v);
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const float lo = __uint_as_float(v[2 * k]), hi = __uint_as_float(v[2 * k + 1]);
                        o[k] = pf_f16x2(lo, hi);
                        if (f16x2_bad(o[k])) {
                            bad = true;
                            if (!is_k) o[k] = f16x2_finite(lo, hi);
                        }
                    }
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k)
                        *reinterpret_cast<uint4*>(st + sw128_offset(r, c0 / 8 + k)) =
                            make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
                }
                fence_proxy_async_smem();
                named_sync(bar + 1, 128);
                if (issuer) {
                    tma_store_3d(is_k ? &p.tm_k : &p.tm_v, st, static_cast<int32_t>(64 * x),
                                 static_cast<int32_t>(blk * kPfBlock), static_cast<int32_t>(j % p.heads));
                    bulk_commit();
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&tempty[acc]);
        }
        if (issuer) bulk_wait();
        if (bad) latch_status(p.status, PBMOE_DEV_ERR_F16_RANGE);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, kExAcc * kExN);
    }
}

// ---------------------------------------------------------------- 2. attention
// grid (heads, query tiles), 384 threads, one CTA per SM. A CTA takes 256
// query rows of one head as two 128-row halves that share every key tile of 64
// cache rows.
//   warp 0      loader: K tiles ([64 rows][64] boxes: two of K_h, one of the key
//               part) and V tiles (two [64 rows][64 dims] boxes), a ring of three
//               each.
//   warps 1, 2  MMA issuers, one a half: S = Q K_t^T (TMEM, 64 columns), then
//               O += P_t V_t with P_t from TMEM (32 columns of its own: S of tile t+1
//               is issued as soon as the softmax has S of tile t in registers, and
//               runs under it).
//   warps 4-7, 8-11  the halves' softmax, one thread a row: p = 2^(s k - m k) in
//               f32, P to TMEM in fp16. m moves only when the maximum has grown by
//               2^8 (p then fits fp16 with room), and only then is O rescaled.
// Measured, 8192 tokens x 16 heads: 300 us, 344 GFLOP, 1.15 PFLOP/s of 1.65. Bound by
// shared memory: a score product of 64 keys takes 49 cycles for 32 of tensor work, since
// it reads 128 rows of Q beside 64 of K each time (128 keys would take 64 cycles for 64,
// but their scores and P do not fit TMEM beside both halves' O with S and P apart, and
// with P over S the next scores wait for the softmax: 400 us).
constexpr uint32_t kPfThreads = 384, kPfHalfThreads = 128, kPfRing = 3, kPfKeys = 64;
constexpr uint32_t kPfQTile = 128, kPfQBytes = 3 * kPfChunk;
constexpr uint32_t kPfKBox = kPfKeys * 128, kPfKBytes = 3 * kPfKBox, kPfVBytes = kPfV * 128;
constexpr size_t kPfSmem = 1024 + 2 * size_t(kPfQBytes) + size_t(kPfRing) * (kPfKBytes + kPfVBytes);
constexpr float kPfSlack = 8.0f;
constexpr float kPfFloor = -1e38f;  // m of a row that has seen only -inf or NaN: below every finite score
constexpr int kPfPoly = 2, kPfPolyOf = 8;  // share of the weights that exp2_poly takes

// One half's query rows to fp16 in the swizzled K-major layout (three boxes of
// 64 columns), zeros past the chunk; 128 threads, 8 values a step.
template <typename QT>
__device__ __forceinline__ bool pf_load_q(const QT* q, uint32_t stride, uint32_t valid, unsigned char* dst, uint32_t t) {
    constexpr uint32_t kChunks = kPfQk / 8, kBatch = sizeof(QT) == 4 ? 12 : 24, kVec = sizeof(QT) / 2;
    static_assert(kPfQTile * kChunks % (kPfHalfThreads * kBatch) == 0, "whole batches");
    bool bad = false;
#pragma unroll 1
    for (uint32_t i0 = t; i0 < kPfQTile * kChunks; i0 += kPfHalfThreads * kBatch) {
        uint4 v[kBatch][kVec];  // a batch's loads in flight together
#pragma unroll
        for (uint32_t j = 0; j < kBatch; ++j) {
            const uint32_t i = i0 + kPfHalfThreads * j, row = i / kChunks, c = i % kChunks;
            const uint4* src = reinterpret_cast<const uint4*>(q + static_cast<size_t>(row) * stride + c * 8);
#pragma unroll
            for (uint32_t k = 0; k < kVec; ++k) v[j][k] = row < valid ? __ldg(src + k) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (uint32_t j = 0; j < kBatch; ++j) {
            const uint32_t i = i0 + kPfHalfThreads * j, row = i / kChunks, c = i % kChunks;
            uint32_t o[4];
            if constexpr (kVec == 2) {
                const uint4 a = v[j][0], b = v[j][1];
                o[0] = pf_f16x2(__uint_as_float(a.x), __uint_as_float(a.y));
                o[1] = pf_f16x2(__uint_as_float(a.z), __uint_as_float(a.w));
                o[2] = pf_f16x2(__uint_as_float(b.x), __uint_as_float(b.y));
                o[3] = pf_f16x2(__uint_as_float(b.z), __uint_as_float(b.w));
            } else {
                const uint32_t w[4] = {v[j][0].x, v[j][0].y, v[j][0].z, v[j][0].w};
#pragma unroll
                for (int k = 0; k < 4; ++k) o[k] = pf_f16x2(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xffff0000u));
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) bad |= f16x2_bad(o[k]);
            *reinterpret_cast<uint4*>(dst + (c / 8) * kPfChunk + sw128_offset(row, c % 8)) = make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
    return bad;
}

template <typename QT, typename OT>
__global__ void __launch_bounds__(kPfThreads, 1) mla_prefill_kernel(const __grid_constant__ MlaPrefillParams p) {
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t kfull[kPfRing], kempty[kPfRing], vfull[kPfRing], vempty[kPfRing], qfull[2],
        sfull[2], sfree[2], pfull[2], pvdone[2], drain[2];
    __shared__ uint32_t tmem_base_sh, abort_sh;
    unsigned char* smem =
        reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char* kring = smem + 2 * kPfQBytes;
    unsigned char* vring = kring + kPfRing * kPfKBytes;
    volatile uint32_t* abort_flag = &abort_sh;
    const uint32_t tid = threadIdx.x, lane = tid & 31;
    const uint32_t warp = __shfl_sync(kFull, tid >> 5, 0);  // warp-uniform for the compiler too
    const uint32_t head = blockIdx.x;
    // work item -> sequence, query tile and the key tiles kt0 .. kt1 of it
    uint32_t b = 0, tile, slot = 0, part = 0, parts = 1;
    if (p.items) {
        const MlaPrefillItem it = p.item[blockIdx.y];
        b = it.seq, tile = it.tile, slot = it.slot, part = it.part, parts = it.parts;
    } else {  // every query tile whole, the longest rows of a sequence first
        while (p.first_tile[b + 1] <= blockIdx.y) ++b;
        tile = p.first_tile[b + 1] - 1 - blockIdx.y;
    }
    const uint32_t q0 = tile * (2 * kPfQTile);
    const uint32_t qlen = p.q_len[b], ctx = p.seqs.len[b] - qlen;
    const uint32_t keys = (ctx + min(qlen, q0 + 2 * kPfQTile) + kPfKeys - 1) / kPfKeys;
    const uint32_t kt0 = keys * part / parts, kt1 = keys * (part + 1) / parts;
    // key tiles of each half from kt0 (none where the second has no rows, or
    // the half sees nothing of this part)
    uint32_t nk[2];
#pragma unroll
    for (uint32_t w = 0; w < 2; ++w) {
        const uint32_t first = q0 + w * kPfQTile;
        const uint32_t end =
            first < qlen ? min(kt1, (ctx + min(qlen, first + kPfQTile) + kPfKeys - 1) / kPfKeys) : 0;
        nk[w] = end > kt0 ? end - kt0 : 0;
    }
    const uint32_t n = max(nk[0], nk[1]);

    if (tid == 0) {
        for (uint32_t i = 0; i < kPfRing; ++i) {
            mbar_init(&kfull[i], 1);
            mbar_init(&kempty[i], 2);  // both halves
            mbar_init(&vfull[i], 1);
            mbar_init(&vempty[i], 2);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&qfull[i], 4);
            mbar_init(&sfull[i], 1);
            mbar_init(&sfree[i], 4);
            mbar_init(&pfull[i], 4);
            mbar_init(&pvdone[i], 1);
            mbar_init(&drain[i], 1);
        }
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
            pdl_wait();  // K, V and key parts; the queries were written before the expansion began
            pdl_launch_dependents();
            const int32_t row0 = static_cast<int32_t>(p.seqs.first_block[b] * kPfBlock), h = static_cast<int32_t>(head);
            bool ok = true;
            for (uint32_t t = 0; ok && t < n; ++t) {
                const uint32_t slot = t % kPfRing;
                const int32_t row = row0 + static_cast<int32_t>((kt0 + t) * kPfKeys);
                if (t >= kPfRing && !pf_wait(&kempty[slot], ((t / kPfRing) - 1) & 1, abort_flag, p.status)) {
                    ok = false;
                    break;
                }
                unsigned char* k = kring + slot * kPfKBytes;
                mbar_arrive_expect_tx(&kfull[slot], kPfKBytes);
                tma_load_3d(k, &p.tm_k, 0, row, h, &kfull[slot]);
                tma_load_3d(k + kPfKBox, &p.tm_k, 64, row, h, &kfull[slot]);
                tma_load_2d(k + 2 * kPfKBox, &p.tm_rope, 0, row, &kfull[slot]);
                if (t >= kPfRing && !pf_wait(&vempty[slot], ((t / kPfRing) - 1) & 1, abort_flag, p.status)) {
                    ok = false;
                    break;
                }
                mbar_arrive_expect_tx(&vfull[slot], kPfVBytes);
                unsigned char* v = vring + slot * kPfVBytes;
                tma_load_3d(v, &p.tm_v, 0, row, h, &vfull[slot]);
                tma_load_3d(v + kPfKBox, &p.tm_v, 64, row, h, &vfull[slot]);
            }
            if (!ok) {
                const uint64_t t0 = global_ns();
                while (global_ns() - t0 < 100000ull) __nanosleep(1000);
            }
        }
        __syncwarp();
    } else if (warp < 3) {
        const uint32_t w = warp - 1;
        const bool leader = elect_one();
        const uint32_t qb = smem_u32(smem) + w * kPfQBytes, kb0 = smem_u32(kring), vb0 = smem_u32(vring);
        // (broadcasts: warp-uniform bounds and operands)
        const uint32_t mine = __shfl_sync(kFull, nk[w], 0), n = __shfl_sync(kFull, max(nk[0], nk[1]), 0);
        const uint32_t tmem = __shfl_sync(kFull, tmem_base_sh, 0);
        const uint32_t ts = tmem + w * 128, tp = ts + kPfKeys, to = tmem + 256 + w * 128;
        auto wait = [&](uint64_t* bar, uint32_t parity) {
            const bool ok = __all_sync(kFull, pf_wait(bar, parity, abort_flag, p.status));
            tc_fence_after();
            return ok;
        };
        auto wait2 = [&](uint64_t* bar, uint32_t parity, uint64_t* bar2, uint32_t parity2) {
            const bool ok = __all_sync(kFull, pf_wait(bar, parity, abort_flag, p.status) &&
                                                  pf_wait(bar2, parity2, abort_flag, p.status));
            tc_fence_after();
            return ok;
        };
        // ring places of the next K and V tile, and their phases
        uint32_t ks = 0, kp = 0, vs = 0, vp = 0;
        auto next = [](uint32_t& s, uint32_t& p) {
            if (++s == kPfRing) s = 0, p ^= 1u;
        };
        auto qk = [&]() {
            if (leader) {
                const uint32_t kb = kb0 + ks * kPfKBytes;
#pragma unroll
                for (uint32_t x = 0; x < 3; ++x)
#pragma unroll
                    for (uint32_t kk = 0; kk < 4; ++kk)
                        umma_f16(ts, sw128_kmajor_desc(qb + x * kPfChunk + kk * 32),
                                 sw128_kmajor_desc(kb + x * kPfKBox + kk * 32), idesc_f16_f32(128, kPfKeys), (x | kk) != 0u);
                umma_commit(&sfull[w]);
                umma_commit(&kempty[ks]);
            }
            __syncwarp();
            next(ks, kp);
        };
        bool ok = true;
        if (mine > 0) {
            ok = wait(&qfull[w], 0) && wait(&kfull[0], 0);
            if (ok) qk();
        }
        for (uint32_t t = 0; ok && t < mine; ++t) {
            if (t + 1 < mine) {
                // the softmax holds the scores of t in registers
                ok = wait2(&kfull[ks], kp, &sfree[w], t & 1);
                if (!ok) break;
                qk();
            }
            ok = wait2(&vfull[vs], vp, &pfull[w], t & 1);
            if (!ok) break;
            if (leader) {
                const uint32_t vb = vb0 + vs * kPfVBytes;
#pragma unroll
                for (uint32_t kk = 0; kk < 4; ++kk)
                    umma_f16_ts(to, tp + kk * 8, sw128_nmajor_desc(vb + kk * 16 * 128, kPfKBox),
                                idesc_f16_f32(128, 128) | kIdescBNMajor, (t | kk) != 0u);
                umma_commit(&pvdone[w]);
                umma_commit(&vempty[vs]);
            }
            __syncwarp();
            next(vs, vp);
        }
        // key tiles of the other half alone: released once they have landed (so
        // that no arrival runs ahead of its barrier's phase)
        for (uint32_t t = mine; ok && t < n; ++t) {
            ok = wait(&kfull[ks], kp);
            if (ok && leader) mbar_arrive(&kempty[ks]);
            ok = ok && wait(&vfull[vs], vp);
            if (ok && leader) mbar_arrive(&vempty[vs]);
            __syncwarp();
            next(ks, kp);
            next(vs, vp);
        }
        if (!ok && leader && mine > 0) {
            umma_commit(&drain[w]);
            const uint64_t t0 = global_ns();
            while (!mbar_try_wait_hint(&drain[w], 0, 20000u) && global_ns() - t0 < kPipeWaitNs) {
            }
        }
        __syncwarp();
    } else if (warp >= 4) {
        const uint32_t w = (warp - 4) >> 2, quarter = warp & 3, r = 32 * quarter + lane;
        const uint32_t first = q0 + w * kPfQTile;
        const size_t at = (static_cast<size_t>(slot) * p.heads + head) * (2 * kPfQTile) + w * kPfQTile + r;  // of a part
        if (nk[w] == 0 && parts > 1) p.stats[at] = make_float2(-INFINITY, 0.f);
        if (nk[w] > 0) {
            const uint32_t valid = min(kPfQTile, qlen - first);
            const QT* q = static_cast<const QT*>(p.query) +
                          (static_cast<size_t>(p.q_first[b] + first) * p.heads + head) * kPfQk;
            const bool bad =
                pf_load_q(q, p.heads * kPfQk, valid, smem + w * kPfQBytes, (tid - 128) % kPfHalfThreads);
            if (bad) latch_status(p.status, PBMOE_DEV_ERR_F16_RANGE);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&qfull[w]);
            const uint32_t lanes = (32u * quarter) << 16;
            const uint32_t ts = tmem + w * 128 + lanes, tp = ts + kPfKeys, to = tmem + 256 + w * 128 + lanes;
            const uint32_t limit = ctx + first + r;  // last key this row sees
            const float k = p.scale_log2;
            float m = 0.f, l = 0.f;
            bool ok = true;
            for (uint32_t t = 0; t < nk[w]; ++t) {
                ok = __all_sync(kFull, pf_wait(&sfull[w], t & 1, abort_flag, p.status));
                if (!ok) break;
                tc_fence_after();
                uint32_t s[64];
                tmem_ld32_nowait(ts, s);
                tmem_ld32_nowait(ts + 32, s + 32);
                tmem_ld_wait(s);
                tmem_ld_wait(s + 32);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sfree[w]);
                const uint32_t key0 = (kt0 + t) * kPfKeys;
                if (key0 + kPfKeys - 1 > ctx + first) {  // some row of the half does not see the whole tile
                    const uint32_t vis = limit < key0 ? 0 : limit - key0 + 1;
#pragma unroll
                    for (uint32_t c = 0; c < 64; ++c)
                        if (c >= vis) s[c] = 0xff800000u;
                }
                float mx[4];
#pragma unroll
                for (uint32_t c = 0; c < 4; ++c) mx[c] = __uint_as_float(s[c]);
#pragma unroll
                for (uint32_t c = 4; c < 64; c += 2)
                    mx[(c >> 1) & 3] = max3(mx[(c >> 1) & 3], __uint_as_float(s[c]), __uint_as_float(s[c + 1]));
                const float top = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]) * k;
                if (t == 0) {
                    m = top > -INFINITY ? top : kPfFloor;
                } else {
                    const bool over = top > m + kPfSlack;
                    // the product of the tile before has read its P (written over below) and
                    // completed O; the next waits for this tile's P
                    ok = __all_sync(kFull, pf_wait(&pvdone[w], (t - 1) & 1, abort_flag, p.status));
                    if (!ok) break;
                    tc_fence_after();
                    if (__any_sync(kFull, over)) {
                        const float m2 = over ? top : m, alpha = ex2_ftz(m - m2);
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
                uint64_t sum[2] = {0, 0};
                const uint64_t k2 = f32x2(k, k), m2 = f32x2(-m, -m);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t pk[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int e = 32 * c + 2 * i;
                        const uint64_t y = fma2(f32x2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), k2, m2);
                        float2 pv;
                        if (i % kPfPolyOf < kPfPoly) {
                            pv = exp2_poly(y);
                        } else {
                            pv = f32x2_get(y);
                            pv = make_float2(ex2_ftz(pv.x), ex2_ftz(pv.y));
                        }
                        sum[i & 1] = add2(sum[i & 1], f32x2(pv.x, pv.y));
                        pk[i] = pf_f16x2(pv.x, pv.y);
                    }
                    tmem_st16(tp + 16 * c, pk);
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&pfull[w]);
                const float2 s2 = f32x2_get(add2(sum[0], sum[1]));
                l += s2.x + s2.y;
            }
            // a row that scored -inf everywhere has summed what exp2_poly makes of its lower
            // end: nothing, so that softmax's NaN comes out (0 / 0), or an empty part
            if (m == kPfFloor && l == l) l = 0.f;
            if (ok && __all_sync(kFull, pf_wait(&pvdone[w], (nk[w] - 1) & 1, abort_flag, p.status))) {
                tc_fence_after();
                const bool whole = parts == 1;
                const float f = whole ? 1.0f / l : 1.0f;  // parts stay unnormalised
                if (!whole) p.stats[at] = make_float2(l == 0.f ? -INFINITY : m, l);
                // 32 columns at a time through the warp's own part of Q's place (every
                // MMA that reads it is done): a row a lane in, whole rows out
                float* st = reinterpret_cast<float*>(smem + w * kPfQBytes + quarter * (kPfQBytes / 4));
                constexpr uint32_t kRow = 36;  // floats: 16-byte lanes of eight rows on distinct banks
#pragma unroll 1
                for (uint32_t i = 0; i < 4; ++i) {
                    uint32_t o[32];
                    tmem_ld32(to + 32 * i, o);
#pragma unroll
                    for (int v = 0; v < 8; ++v)
                        reinterpret_cast<float4*>(st + lane * kRow)[v] =
                            make_float4(__uint_as_float(o[4 * v]) * f, __uint_as_float(o[4 * v + 1]) * f,
                                        __uint_as_float(o[4 * v + 2]) * f, __uint_as_float(o[4 * v + 3]) * f);
                    __syncwarp();
#pragma unroll
                    for (uint32_t v = 0; v < 8; ++v) {  // 4 rows of 8 lanes, 4 columns each
                        const uint32_t rr = 4 * v + lane / 8, row = 32 * quarter + rr, col = 4 * (lane % 8);
                        const float4 x = *reinterpret_cast<const float4*>(st + rr * kRow + col);
                        if (!whole) {
                            *reinterpret_cast<float4*>(p.partial + (at - r + row) * kPfV + 32 * i + col) = x;
                        } else if (row < valid) {
                            OT* dst = static_cast<OT*>(p.out) +
                                      (static_cast<size_t>(p.q_first[b] + first + row) * p.heads + head) * kPfV + 32 * i + col;
                            if constexpr (sizeof(OT) == 4) {
                                *reinterpret_cast<float4*>(dst) = x;
                            } else {
                                uint2 h;
                                asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(h.x) : "f"(x.y), "f"(x.x));
                                asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(h.y) : "f"(x.w), "f"(x.z));
                                *reinterpret_cast<uint2*>(dst) = h;
                            }
                        }
                    }
                    __syncwarp();
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

// ---------------------------------------------------------------- join
// Parts of a query tile: out = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s, a
// warp a (row, head), four dims a lane. grid (tiles, heads, 256 / 8).
constexpr uint32_t kPfJoinThreads = 256;
template <typename OT>
__global__ void __launch_bounds__(kPfJoinThreads) mla_prefill_join_kernel(const __grid_constant__ MlaPrefillJoin p) {
    const uint32_t head = blockIdx.y, lane = threadIdx.x & 31;
    const MlaPrefillItem it = p.tile[blockIdx.x];
    const uint32_t b = it.seq, parts = it.parts, r = blockIdx.z * (kPfJoinThreads / 32) + (threadIdx.x >> 5);
    const uint32_t row = it.tile * (2 * kPfQTile) + r;
    if (row >= p.q_len[b]) return;
    pdl_wait();
    const size_t at0 = (static_cast<size_t>(it.slot) * p.heads + head) * (2 * kPfQTile) + r;
    const size_t step = static_cast<size_t>(p.heads) * (2 * kPfQTile);
    // statistics of 32 parts a round, a part a lane; an empty part (no visible
    // key there) has weight 0 and its output, which is not written, is not read
    float M = -INFINITY, l = 0.f;
    for (uint32_t s0 = 0; s0 < parts; s0 += 32)
        M = fmaxf(M, s0 + lane < parts ? p.stats[at0 + (s0 + lane) * step].x : -INFINITY);
    M = warp_max(M);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (uint32_t s0 = 0; s0 < parts; s0 += 32) {
        const float2 st = s0 + lane < parts ? p.stats[at0 + (s0 + lane) * step] : make_float2(-INFINITY, 0.f);
        const float f = st.x == -INFINITY ? 0.f : exp2f(st.x - M);
        l += f * st.y;
        const unsigned used = __ballot_sync(kFull, st.x != -INFINITY);
        for (uint32_t s1 = 0; s1 < min(32u, parts - s0); s1 += 8) {
            float4 o[8];  // eight parts' loads in flight together
#pragma unroll
            for (uint32_t s = 0; s < 8; ++s)
                o[s] = (used >> (s1 + s) & 1u)
                           ? reinterpret_cast<const float4*>(p.partial + (at0 + (s0 + s1 + s) * step) * kPfV)[lane]
                           : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (uint32_t s = 0; s < 8; ++s) {
                const float fs = __shfl_sync(kFull, f, s1 + s);
                acc.x = fmaf(fs, o[s].x, acc.x);
                acc.y = fmaf(fs, o[s].y, acc.y);
                acc.z = fmaf(fs, o[s].z, acc.z);
                acc.w = fmaf(fs, o[s].w, acc.w);
            }
        }
    }
    const float inv = 1.0f / warp_sum(l);
    OT* out = static_cast<OT*>(p.out) + (static_cast<size_t>(p.q_first[b] + row) * p.heads + head) * kPfV + 4 * lane;
    if constexpr (sizeof(OT) == 4) {
        *reinterpret_cast<float4*>(out) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    } else {
        uint2 h;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(h.x) : "f"(acc.y * inv), "f"(acc.x * inv));
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(h.y) : "f"(acc.w * inv), "f"(acc.z * inv));
        *reinterpret_cast<uint2*>(out) = h;
    }
}

// ---------------------------------------------------------------- launch
MlaPrefillWs mla_prefill_ws(uint32_t heads, uint32_t blocks, int num_sms) {
    MlaPrefillWs w{};
    const size_t rows = size_t(blocks) * kPfBlock, slots = kMlaPrefillSlots * size_t(num_sms);  // slots x heads
    w.k16 = 0;
    w.v16 = w.k16 + rows * heads * kPfNope * 2;  // multiples of 256 bytes
    w.rope16 = w.v16 + rows * heads * kPfV * 2;
    w.partial = w.rope16 + rows * kPfRope * 2;
    w.stats = w.partial + slots * 2 * kPfQTile * kPfV * 4;
    w.total = w.stats + slots * 2 * kPfQTile * 8;
    return w;
}

namespace {

// The work list of one call. A CTA's time goes by its key tiles, and a call's
// by its slowest SM, so query tiles may be cut into parts: with few rows over a
// long context there would be one CTA a head, and a single prompt's last rows
// take twice its mean. The longest tile is cut into 1, 2, 3, ... parts and the
// others to the same size, and the size is taken whose estimate is least: the
// longest item, the mean load of an SM, or, when there are more CTAs than SMs,
// the two that share one, whichever is largest (in key tiles, 0.7 us each; an
// item costs kStart more, joining kJoin once). Lists that would not fit stay
// whole, in grid order: they have several CTAs an SM, which balance by
// themselves. The two constants are fitted to 154 shapes (1 to 128 heads, 1 to
// 8192 tokens, contexts up to 16000, each timed whole and in up to 48 parts): the
// choice is 0.6% slower than the best of them on average and 10% at most. Whole
// and cut, 16 heads: 2048 tokens 53 us and 64 in three parts (stays whole), 500
// after 1000 rows 42.5 and 34.0, 61 after 4035 rows 75 and 40.
void prefill_items(const MlaPrefillLaunch& a, int num_sms, MlaPrefillParams& p, MlaPrefillJoin& j) {
    constexpr uint32_t kStart = 14, kJoin = 10, kLeast = 4;
    p.items = 0;
    j.tiles = 0;
    struct Tile {
        uint32_t keys, seq, index;
    };
    Tile tile[kMlaPrefillItems];
    uint32_t tiles = 0;
    for (uint32_t b = 0; b < a.seqs.batch; ++b)
        for (uint32_t row = 0; row < a.q_len[b]; row += 2 * kPfQTile) {
            if (tiles == kMlaPrefillItems) return;
            const uint64_t seen = uint64_t(a.seqs.len[b]) - a.q_len[b] + std::min(a.q_len[b], row + 2 * kPfQTile);
            tile[tiles++] = {static_cast<uint32_t>((seen + kPfKeys - 1) / kPfKeys), b, row / (2 * kPfQTile)};
        }
    uint32_t longest = 0;
    for (uint32_t i = 0; i < tiles; ++i) longest = std::max(longest, tile[i].keys);
    const uint32_t max_slots = kMlaPrefillSlots * static_cast<uint32_t>(num_sms) / a.heads;
    uint64_t best = ~uint64_t(0);
    uint32_t size = longest;
    for (uint32_t cut = 1; cut <= 255 && (cut == 1 || longest / cut >= kLeast); ++cut) {
        const uint32_t part = (longest + cut - 1) / cut;
        uint64_t load = 0, items = 0, slots = 0;
        // the items at the SMs' last and next place, longest first, by counting
        uint32_t most = 0, count[3] = {0, 0, 0};  // items above 3/4, 1/2 and 1/4 of a part
        for (uint32_t i = 0; i < tiles; ++i) {
            const uint32_t parts = (tile[i].keys + part - 1) / part, each = (tile[i].keys + parts - 1) / parts;
            items += parts;
            slots += parts > 1 ? parts : 0;
            load += tile[i].keys + uint64_t(parts) * kStart;
            most = std::max(most, each);
            for (uint32_t q = 0; q < 3; ++q) count[q] += each * 4 > part * (3 - q) ? parts : 0;
        }
        if (items > kMlaPrefillItems || slots > max_slots) break;
        uint64_t t = std::max<uint64_t>(most + kStart, (load * a.heads + num_sms - 1) / num_sms);
        for (uint32_t q = 0; q < 3; ++q)  // two items of at least this length share an SM
            if (uint64_t(count[q]) * a.heads > static_cast<uint64_t>(num_sms)) {
                t = std::max<uint64_t>(t, 2 * (part * (3 - q) / 4 + kStart));
                break;
            }
        if (cut > 1) t += kJoin;
        if (t < best) {
            best = t;
            size = part;
        }
    }
    struct Item {
        uint32_t keys;
        MlaPrefillItem it;
    };
    Item list[kMlaPrefillItems];
    uint32_t n = 0, slots = 0;
    for (uint32_t i = 0; i < tiles; ++i) {
        const uint32_t parts = (tile[i].keys + size - 1) / size;
        MlaPrefillItem it{static_cast<uint16_t>(tile[i].index), static_cast<uint16_t>(parts > 1 ? slots : 0),
                          static_cast<uint8_t>(tile[i].seq), 0, static_cast<uint8_t>(parts)};
        if (parts > 1) j.tile[j.tiles++] = it;
        for (uint32_t s = 0; s < parts; ++s) {
            it.part = static_cast<uint8_t>(s);
            it.slot = static_cast<uint16_t>(parts > 1 ? slots++ : 0);
            list[n++] = {(tile[i].keys + parts - 1) / parts, it};
        }
    }
    std::stable_sort(list, list + n, [](const Item& x, const Item& y) { return x.keys > y.keys; });
    for (uint32_t i = 0; i < n; ++i) p.item[i] = list[i].it;
    p.items = n;
}

}  // namespace

uint32_t mla_prefill_blocks(uint32_t len) { return len / kPfBlock + (len % kPfBlock != 0); }

// The kernels' shared memory, once per device (set where the workspace is).
cudaError_t mla_prefill_prepare() {
    cudaError_t e = cudaSuccess;
    auto set = [&](auto kernel, size_t bytes) {
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    };
    set(mla_expand_kernel, kExSmem);
    set(mla_prefill_kernel<float, float>, kPfSmem);
    set(mla_prefill_kernel<float, uint16_t>, kPfSmem);
    set(mla_prefill_kernel<uint16_t, float>, kPfSmem);
    set(mla_prefill_kernel<uint16_t, uint16_t>, kPfSmem);
    return e;
}

cudaError_t mla_prefill_launch(const MlaPrefillLaunch& a, int num_sms, cudaStream_t s) {
    const uint32_t blocks = a.seqs.first_block[a.seqs.batch];
    if (blocks == 0) return cudaSuccess;
    const uint64_t rows = uint64_t(blocks) * kPfBlock;
    const MlaPrefillWs w = mla_prefill_ws(a.heads, blocks, num_sms);
    char* base = static_cast<char*>(a.workspace);
    uint16_t* k16 = reinterpret_cast<uint16_t*>(base + w.k16);
    uint16_t* v16 = reinterpret_cast<uint16_t*>(base + w.v16);
    uint16_t* rope16 = reinterpret_cast<uint16_t*>(base + w.rope16);
    cudaError_t e;
    {
        MlaExpandParams p{};
        p.seqs = a.seqs;
        p.heads = a.heads;
        p.rope16 = rope16;
        p.status = a.status;
        for (uint32_t b = 0; b < a.seqs.batch; ++b) {
            p.k_rope[b] = a.k_rope[b];
            if (a.seqs.len[b] == 0) continue;
            if ((e = make_map_16(&p.tm_c[b], true, a.c_kv[b], 2, kPfLatent, a.seqs.len[b], 1, kPfBlock)) != cudaSuccess)
                return e;
        }
        if ((e = make_map_16(&p.tm_uk, true, a.w_uk, 2, kPfLatent, uint64_t(a.heads) * kPfNope, 1, kPfBlock)) != cudaSuccess ||
            (e = make_map_16(&p.tm_uv, true, a.w_uv, 2, kPfLatent, uint64_t(a.heads) * kPfV, 1, kPfBlock)) != cudaSuccess ||
            (e = make_map_16(&p.tm_k, false, k16, 3, kPfNope, rows, a.heads, kPfBlock)) != cudaSuccess ||
            (e = make_map_16(&p.tm_v, false, v16, 3, kPfV, rows, a.heads, kPfBlock)) != cudaSuccess)
            return e;
        const uint32_t grid = static_cast<uint32_t>(
            std::min<uint64_t>(uint64_t(blocks) * 2 * a.heads, static_cast<uint64_t>(num_sms)));
        if ((e = launch_pdl_kernel(mla_expand_kernel, dim3(grid), dim3(kExThreads), kExSmem, s, p)) != cudaSuccess) return e;
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
    if ((e = make_map_16(&p.tm_k, false, k16, 3, kPfNope, rows, a.heads, kPfKeys)) != cudaSuccess ||
        (e = make_map_16(&p.tm_v, false, v16, 3, kPfV, rows, a.heads, kPfKeys)) != cudaSuccess ||
        (e = make_map_16(&p.tm_rope, false, rope16, 2, kPfRope, rows, 1, kPfKeys)) != cudaSuccess)
        return e;
    MlaPrefillJoin j{};
    prefill_items(a, num_sms, p, j);
    p.partial = reinterpret_cast<float*>(base + w.partial);
    p.stats = reinterpret_cast<float2*>(base + w.stats);
    auto go = [&](auto kernel) {
        return launch_pdl_kernel(kernel, dim3(a.heads, p.items ? p.items : tiles), dim3(kPfThreads), kPfSmem, s, p);
    };
    const bool f32 = a.out_dtype == PBMOE_F32;
    if (a.q_dtype == PBMOE_F32)
        e = f32 ? go(mla_prefill_kernel<float, float>) : go(mla_prefill_kernel<float, uint16_t>);
    else
        e = f32 ? go(mla_prefill_kernel<uint16_t, float>) : go(mla_prefill_kernel<uint16_t, uint16_t>);
    if (e != cudaSuccess || j.tiles == 0) return e;
    for (uint32_t b = 0; b < kMlaMaxBatch; ++b) {
        j.q_len[b] = p.q_len[b];
        j.q_first[b] = p.q_first[b];
    }
    j.heads = a.heads;
    j.partial = p.partial;
    j.stats = p.stats;
    j.out = a.out;
    const dim3 grid(j.tiles, a.heads, 2 * kPfQTile / (kPfJoinThreads / 32));
    return f32 ? launch_pdl_kernel(mla_prefill_join_kernel<float>, grid, dim3(kPfJoinThreads), 0, s, j)
               : launch_pdl_kernel(mla_prefill_join_kernel<uint16_t>, grid, dim3(kPfJoinThreads), 0, s, j);
}

}  // namespace pbmoe
