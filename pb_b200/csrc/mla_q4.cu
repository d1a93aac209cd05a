// mla_q4.cu — the MLA latent cache held in 4 bits: rows quantised as they are
// written, read back, and attended over (absorbed decode attention).
//
// A row of the cache (one token; no counterpart in the reference, whose
// KvCache::mla_records keeps f32 rows, state/kv_cache.rs:414-450) is
//   codes   512 x 4 bits, column c in byte c/2 (low nibble = even c), the
//           stored nibble u = q + 8 with q in -7..7
//   scales  one bf16 per 64 columns, s = bf16(max|x| / 7)
//   k_rope  64 x bf16, the rotated key part, not quantised: it enters every
//           score undiluted, and its 128 of 400 bytes buy no more than 1.3x
// and stands for v = q * s: 400 bytes where the bf16 cache row has 1152. The
// code is symmetric so that a group's sum needs no per-token bias:
//   sum_c x_c v_c = s * (sum_c x_c u_c - 8 sum_c x_c),
// with sum_c x_c known once per query (scores) or one extra MMA column
// (context).

#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "mma_sync.cuh"

namespace pbmoe {

constexpr uint32_t kQ4Latent = 512, kQ4Rope = 64, kQ4Group = 64;
constexpr uint32_t kQ4Groups = kQ4Latent / kQ4Group;  // 8 scales per row
constexpr uint32_t kQ4CodeBytes = kQ4Latent / 2;

__device__ __forceinline__ uint32_t cvt_f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// ---------------------------------------------------------------- append
// CTAs of 8 warps: first those of the cache rows, a CTA or (many tokens) a warp a row,
// then 16 heads of a token's query a CTA, two a warp (lane p: pair p), their loads
// before the position is known and before any store, so the query may be rotated in
// place. The mean square is summed in f64: a code next to a rounding border is then
// the same whatever the order of the sum.
// A decode step's rows are bound by the launch and one chain of loads (32 tokens: 2.2
// us in a graph; a warp a row 4.3, its sums one after another), a prompt's by the
// memory (8190 tokens, bf16 rows, f32 queries of 16 x 192 into bf16: 30.5 us, 164 MB,
// 5.4 TB/s; a CTA a row 37.6: eight warps reduce and wait for one another, and the
// issue slots run out; CTAs that stay and load the next heads under the stores of
// these 43-61, since fewer are resident). The two forms, a CTA and a warp a row: 512
// tokens 3.4 and 4.9 us, 768 4.4 and 6.6, 1024 5.3 and 5.0, 2048 8.4 and 6.5.
constexpr int kQ4AppendThreads = 256;
constexpr uint32_t kQ4AppendWarpRows = 1024;  // tokens from which a row is a warp's
template <typename KT>
__device__ __forceinline__ float2 load_pair(const KT* p);
template <>
__device__ __forceinline__ float2 load_pair<float>(const float* p) {
    return *reinterpret_cast<const float2*>(p);
}
template <>
__device__ __forceinline__ float2 load_pair<uint16_t>(const uint16_t* p) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
    return make_float2(bf16_lo(w), bf16_hi(w));
}
__device__ __forceinline__ void store_one(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_one(uint16_t* p, float v) {
    *p = static_cast<uint16_t>(cvt_bf16x2(v, 0.f) & 0xffffu);
}
__device__ __forceinline__ void store_pair(float* p, float2 v) { *reinterpret_cast<float2*>(p) = v; }
__device__ __forceinline__ void store_pair(uint16_t* p, float2 v) {
    *reinterpret_cast<uint32_t*>(p) = cvt_bf16x2(v.x, v.y);
}

// Up to kQ4AppendHeads heads of one token, h0, h0 + kQ4AppendWarps, ... <
// heads: loaded, then rotated (and, out of place, their nope parts copied).
constexpr uint32_t kQ4AppendHeads = 2, kQ4AppendWarps = kQ4AppendThreads / 32;
struct HeadPairs {
    float2 v[kQ4AppendHeads], n0[kQ4AppendHeads], n1[kQ4AppendHeads];
};
template <typename QT>
__device__ __forceinline__ void load_heads(HeadPairs& x, const QT* q, uint32_t h0, uint32_t heads, uint32_t nope,
                                           bool copy_nope) {
    const uint32_t lane = threadIdx.x & 31, qk = nope + kQ4Rope, i0 = 2 * lane, i1 = 64 + 2 * lane;  // nope <= 128
#pragma unroll
    for (uint32_t j = 0; j < kQ4AppendHeads; ++j) {
        const uint32_t h = h0 + j * kQ4AppendWarps;
        if (h >= heads) continue;
        x.v[j] = load_pair(q + h * qk + nope + 2 * lane);
        if (copy_nope && i0 < nope) x.n0[j] = load_pair(q + h * qk + i0);
        if (copy_nope && i1 < nope) x.n1[j] = load_pair(q + h * qk + i1);
    }
}
template <typename OT>
__device__ __forceinline__ void store_heads(const HeadPairs& x, OT* out, uint32_t h0, uint32_t heads, uint32_t nope,
                                            float2 cs, bool copy_nope) {
    const uint32_t lane = threadIdx.x & 31, qk = nope + kQ4Rope, i0 = 2 * lane, i1 = 64 + 2 * lane;
    __syncwarp();  // every pair read
#pragma unroll
    for (uint32_t j = 0; j < kQ4AppendHeads; ++j) {
        const uint32_t h = h0 + j * kQ4AppendWarps;
        if (h >= heads) continue;
        OT* o = out + h * qk;
        store_one(o + nope + lane, __fsub_rn(__fmul_rn(x.v[j].x, cs.x), __fmul_rn(x.v[j].y, cs.y)));
        store_one(o + nope + 32 + lane, __fadd_rn(__fmul_rn(x.v[j].y, cs.x), __fmul_rn(x.v[j].x, cs.y)));
        if (copy_nope && i0 < nope) store_pair(o + i0, x.n0[j]);
        if (copy_nope && i1 < nope) store_pair(o + i1, x.n1[j]);
    }
}

// rint(x / s) in -7..7. x * (1 / s) is within 2e-6 of the quotient (of at most
// 7.1): where it lies that far from a border it rounds to the same integer, and
// the quotient is only taken next to one (or where 1 / s overflows).
__device__ __forceinline__ int q4_code(float x, float s, float rs) {
    float t = x * rs;
    if (!(fabsf(t - rintf(t)) <= 0.4999f)) t = __fdiv_rn(x, s);
    return max(-7, min(7, __float2int_rn(t)));
}

__device__ __forceinline__ bool q4_place(const MlaQ4Append& a, uint32_t tok, uint32_t& seq, uint32_t& pos) {
    seq = a.sequences ? a.sequences[tok] : tok;
    pos = a.positions[tok];
    return seq < a.batch && pos < a.max_positions && pos < a.seqs.len[min(seq, kMlaMaxBatch - 1)];
}

// A cache row by a CTA: thread i holds columns 2i and 2i+1, warp g is group g.
template <typename KT>
__device__ __forceinline__ void q4_row_by_cta(const MlaQ4Append& a, uint32_t tok) {
    __shared__ double red[kQ4AppendThreads / 32];
    __shared__ float scale_sh;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const KT* kv = static_cast<const KT*>(a.kv) + static_cast<size_t>(tok) * (kQ4Latent + kQ4Rope);
    float2 x = load_pair(kv + 2 * tid), key = make_float2(0.f, 0.f), nw = key;  // in flight while the position arrives
    if (warp == 0) key = load_pair(kv + kQ4Latent + 2 * lane);
    if (a.latent_norm_w) nw = *reinterpret_cast<const float2*>(a.latent_norm_w + 2 * tid);
    uint32_t seq, pos;
    if (!q4_place(a, tok, seq, pos)) {
        if (tid == 0) latch_status(a.status, PBMOE_DEV_ERR_POSITION);
        return;
    }
    const float2 cs = a.table[static_cast<size_t>(pos) * (kQ4Rope / 2) + lane];
    if (a.latent_norm_w) {
        double ss = static_cast<double>(x.x) * x.x + static_cast<double>(x.y) * x.y;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(kFull, ss, o);
        if (lane == 0) red[warp] = ss;
        __syncthreads();
        if (warp == 0) {  // (once: the f64 root and quotient are long)
            double tot = lane < kQ4AppendThreads / 32 ? red[lane] : 0.0;
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) tot += __shfl_xor_sync(kFull, tot, o);
            if (lane == 0) scale_sh = static_cast<float>(1.0 / sqrt(tot / kQ4Latent + static_cast<double>(a.eps)));
        }
        __syncthreads();
        const float scale = scale_sh;
        x.x = __fmul_rn(__fmul_rn(x.x, scale), nw.x);
        x.y = __fmul_rn(__fmul_rn(x.y, scale), nw.y);
    }
    // the group's scale; a non-finite value makes it NaN, and with it every
    // value that the group stands for
    const bool bad = !(fabsf(x.x) < INFINITY) || !(fabsf(x.y) < INFINITY);
    const float amax = warp_max(fmaxf(fabsf(x.x), fabsf(x.y)));
    const bool group_bad = __any_sync(kFull, bad);
    uint32_t s16 = cvt_bf16x2(__fdiv_rn(amax, 7.0f), 0.f) & 0xffffu;
    if (group_bad) s16 = 0x7fc0u;
    const float s = bf16_bits_to_f32(s16);
    int q0 = 0, q1 = 0;
    if (s > 0.f) {
        const float rs = __frcp_rn(s);
        q0 = q4_code(x.x, s, rs);
        q1 = q4_code(x.y, s, rs);
    }
    const size_t row = pos;
    const uint32_t byte = static_cast<uint32_t>(q0 + 8) | (static_cast<uint32_t>(q1 + 8) << 4);
    // four lanes' bytes to one word
    uint32_t word = byte << (8 * (lane & 3));
    word |= __shfl_xor_sync(kFull, word, 1);
    word |= __shfl_xor_sync(kFull, word, 2);
    if ((lane & 3) == 0) *reinterpret_cast<uint32_t*>(a.seqs.codes[seq] + row * kQ4CodeBytes + tid) = word;
    if (lane == 0) {
        a.seqs.scales[seq][row * kQ4Groups + warp] = static_cast<uint16_t>(s16);
        if (group_bad) latch_status(a.status, PBMOE_DEV_ERR_CACHE_RANGE);
    }
    if (warp == 0) {
        uint16_t* kr = a.seqs.k_rope[seq] + row * kQ4Rope;
        store_one(kr + lane, __fsub_rn(__fmul_rn(key.x, cs.x), __fmul_rn(key.y, cs.y)));
        store_one(kr + 32 + lane, __fadd_rn(__fmul_rn(key.y, cs.x), __fmul_rn(key.x, cs.y)));
    }
}

// A cache row by a warp: lane l holds columns 64g + 2l and the next of every group g.
template <typename KT>
__device__ __forceinline__ void q4_row_by_warp(const MlaQ4Append& a, uint32_t tok) {
    const uint32_t lane = threadIdx.x & 31;
    const KT* kv = static_cast<const KT*>(a.kv) + static_cast<size_t>(tok) * (kQ4Latent + kQ4Rope);
    float2 x[kQ4Groups];
#pragma unroll
    for (uint32_t g = 0; g < kQ4Groups; ++g) x[g] = load_pair(kv + kQ4Group * g + 2 * lane);
    const float2 key = load_pair(kv + kQ4Latent + 2 * lane);
    uint32_t seq, pos;
    if (!q4_place(a, tok, seq, pos)) {
        if (lane == 0) latch_status(a.status, PBMOE_DEV_ERR_POSITION);
        return;
    }
    const float2 cs = a.table[static_cast<size_t>(pos) * (kQ4Rope / 2) + lane];
    const size_t row = pos;
    {
        uint16_t* kr = a.seqs.k_rope[seq] + row * kQ4Rope;
        store_one(kr + lane, __fsub_rn(__fmul_rn(key.x, cs.x), __fmul_rn(key.y, cs.y)));
        store_one(kr + 32 + lane, __fadd_rn(__fmul_rn(key.y, cs.x), __fmul_rn(key.x, cs.y)));
    }
    if (a.latent_norm_w) {
        double ss = 0.0, st = 0.0;
#pragma unroll
        for (uint32_t g = 0; g < kQ4Groups; ++g) {
            ss = fma(static_cast<double>(x[g].x), static_cast<double>(x[g].x), ss);
            st = fma(static_cast<double>(x[g].y), static_cast<double>(x[g].y), st);
        }
        ss += st;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(kFull, ss, o);
        const float scale = static_cast<float>(1.0 / sqrt(ss / kQ4Latent + static_cast<double>(a.eps)));
#pragma unroll
        for (uint32_t g = 0; g < kQ4Groups; ++g) {
            const float2 w = *reinterpret_cast<const float2*>(a.latent_norm_w + kQ4Group * g + 2 * lane);
            x[g].x = __fmul_rn(__fmul_rn(x[g].x, scale), w.x);
            x[g].y = __fmul_rn(__fmul_rn(x[g].y, scale), w.y);
        }
    }
    uint8_t* codes = a.seqs.codes[seq] + row * kQ4CodeBytes + lane;
    uint32_t scales[kQ4Groups / 2] = {};
    bool bad = false;
#pragma unroll
    for (uint32_t g = 0; g < kQ4Groups; ++g) {
        // the group's scale from its largest magnitude (as bits: ordered like the
        // values, infinity and NaN above all); a non-finite value makes it NaN, and
        // with it every value that the group stands for
        const uint32_t amax = __reduce_max_sync(
            kFull, max(__float_as_uint(x[g].x) & 0x7fffffffu, __float_as_uint(x[g].y) & 0x7fffffffu));
        uint32_t s16 = cvt_bf16x2(__fdiv_rn(__uint_as_float(amax), 7.0f), 0.f) & 0xffffu;
        if (amax >= 0x7f800000u) s16 = 0x7fc0u, bad = true;
        scales[g / 2] |= s16 << (16 * (g & 1));
        const float s = bf16_bits_to_f32(s16);
        int q0 = 0, q1 = 0;
        if (s > 0.f) {
            const float rs = __frcp_rn(s);
            q0 = q4_code(x[g].x, s, rs);
            q1 = q4_code(x[g].y, s, rs);
        }
        codes[kQ4Group / 2 * g] = static_cast<uint8_t>(static_cast<uint32_t>(q0 + 8) | (static_cast<uint32_t>(q1 + 8) << 4));
    }
    if (lane == 0) {
        *reinterpret_cast<uint4*>(a.seqs.scales[seq] + row * kQ4Groups) = make_uint4(scales[0], scales[1], scales[2], scales[3]);
        if (bad) latch_status(a.status, PBMOE_DEV_ERR_CACHE_RANGE);
    }
}

template <typename KT, typename QT, typename OT, bool kWarpRow>
__global__ void __launch_bounds__(kQ4AppendThreads, kWarpRow ? 6 : 8)
    mla_q4_append_kernel(const __grid_constant__ MlaQ4Append a, uint32_t cache_ctas, uint32_t groups) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_wait();
    pdl_launch_dependents();
    if (blockIdx.x < cache_ctas) {
        if constexpr (kWarpRow) {
            const uint32_t tok = blockIdx.x * kQ4AppendWarps + warp;
            if (tok < a.tokens) q4_row_by_warp<KT>(a, tok);
        } else {
            q4_row_by_cta<KT>(a, blockIdx.x);
        }
        return;
    }
    const uint32_t i = blockIdx.x - cache_ctas, tok = i / groups;
    const uint32_t h0 = i % groups * (kQ4AppendHeads * kQ4AppendWarps) + warp;
    const size_t at = static_cast<size_t>(tok) * a.heads * (a.nope + kQ4Rope);
    HeadPairs hp{};  // in flight while the position arrives
    load_heads(hp, static_cast<const QT*>(a.query) + at, h0, a.heads, a.nope, a.query_out != a.query);
    uint32_t seq, pos;
    if (!q4_place(a, tok, seq, pos)) return;
    const float2 cs = a.table[static_cast<size_t>(pos) * (kQ4Rope / 2) + lane];
    store_heads(hp, static_cast<OT*>(a.query_out) + at, h0, a.heads, a.nope, cs, a.query_out != a.query);
}

namespace {
template <typename KT, typename QT, typename OT>
cudaError_t append_go(const MlaQ4Append& a, cudaStream_t s) {
    constexpr uint32_t kHeads = kQ4AppendHeads * kQ4AppendWarps;  // a CTA
    const uint32_t groups = a.query ? (a.heads + kHeads - 1) / kHeads : 0;
    if (a.tokens < kQ4AppendWarpRows)
        return launch_pdl_kernel(mla_q4_append_kernel<KT, QT, OT, false>, dim3(a.tokens * (1 + groups)),
                                 dim3(kQ4AppendThreads), 0, s, a, a.tokens, groups);
    const uint32_t cache_ctas = (a.tokens + kQ4AppendWarps - 1) / kQ4AppendWarps;
    return launch_pdl_kernel(mla_q4_append_kernel<KT, QT, OT, true>, dim3(cache_ctas + a.tokens * groups),
                             dim3(kQ4AppendThreads), 0, s, a, cache_ctas, groups);
}
template <typename KT, typename QT>
cudaError_t append_out(const MlaQ4Append& a, cudaStream_t s) {
    return a.query_out_dtype == PBMOE_F32 ? append_go<KT, QT, float>(a, s) : append_go<KT, QT, uint16_t>(a, s);
}
template <typename KT>
cudaError_t append_query(const MlaQ4Append& a, cudaStream_t s) {
    return a.query_dtype == PBMOE_F32 ? append_out<KT, float>(a, s) : append_out<KT, uint16_t>(a, s);
}
}  // namespace

cudaError_t mla_q4_append_launch(const MlaQ4Append& a, cudaStream_t s) {
    if (a.tokens == 0) return cudaSuccess;
    return a.kv_dtype == PBMOE_F32 ? append_query<float>(a, s) : append_query<uint16_t>(a, s);
}

// ---------------------------------------------------------------- read back
// Rows [begin, begin + count) of each sequence as bf16, packed one sequence
// after another: v = q * s in f32, one rounding. grid (row blocks, batch),
// 256 threads; a warp takes whole rows: lane l turns codes 16l .. 16l+15
// (8 bytes) into 32 bytes, lanes 0-7 copy the key part. Bound by memory: 155 MB
// (eight sequences, about 100000 rows) in 33 us with the launch, 4.7 TB/s; four
// rows' loads in flight a warp.
constexpr uint32_t kQ4ReadThreads = 256, kQ4ReadRows = 64;
__global__ void __launch_bounds__(kQ4ReadThreads) mla_q4_read_kernel(const __grid_constant__ MlaQ4Read a) {
    const uint32_t b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t count = a.count[b];
    const uint32_t r0 = blockIdx.x * kQ4ReadRows;
    if (r0 >= count) return;
    const uint32_t r1 = min(count, r0 + kQ4ReadRows);
    const uint8_t* codes = a.seqs.codes[b];
    const uint16_t* scales = a.seqs.scales[b];
    const uint16_t* krope = a.seqs.k_rope[b];
    constexpr uint32_t kRows = 4, kWarps = kQ4ReadThreads / 32;
    for (uint32_t r = r0 + warp; r < r1; r += kRows * kWarps) {
        uint2 w[kRows];
        uint32_t s16[kRows];
        uint4 key[kRows];
#pragma unroll
        for (uint32_t i = 0; i < kRows; ++i) {  // the rows' loads in flight together
            const bool ok = r + i * kWarps < r1;
            const size_t row = static_cast<size_t>(a.begin[b]) + (ok ? r + i * kWarps : r);
            w[i] = ld_stream_u2(codes + row * kQ4CodeBytes + 8 * lane);
            s16[i] = scales[row * kQ4Groups + lane / 4];
            key[i] = make_uint4(0, 0, 0, 0);
            if (a.k_rope && lane < 8) key[i] = *reinterpret_cast<const uint4*>(krope + row * kQ4Rope + 8 * lane);
        }
#pragma unroll
        for (uint32_t i = 0; i < kRows; ++i) {
            if (r + i * kWarps >= r1) break;
            const size_t dst = static_cast<size_t>(a.offset[b]) + r + i * kWarps;
            const float s = bf16_bits_to_f32(s16[i]);
            uint32_t o[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint32_t u = (k < 4 ? w[i].x : w[i].y) >> (8 * (k & 3));
                o[k] = cvt_bf16x2(static_cast<float>(static_cast<int>(u & 15u) - 8) * s,
                                  static_cast<float>(static_cast<int>((u >> 4) & 15u) - 8) * s);
            }
            uint4* out = reinterpret_cast<uint4*>(a.c_kv + dst * kQ4Latent + 16 * lane);
            out[0] = make_uint4(o[0], o[1], o[2], o[3]);
            out[1] = make_uint4(o[4], o[5], o[6], o[7]);
            if (a.k_rope && lane < 8) *reinterpret_cast<uint4*>(a.k_rope + dst * kQ4Rope + 8 * lane) = key[i];
        }
    }
}

cudaError_t mla_q4_read_launch(const MlaQ4Read& a, uint32_t max_count, cudaStream_t s) {
    if (max_count == 0) return cudaSuccess;
    const dim3 grid((max_count + kQ4ReadRows - 1) / kQ4ReadRows, a.batch);
    return launch_pdl_kernel(mla_q4_read_kernel, grid, dim3(kQ4ReadThreads), 0, s, a);
}

// ---------------------------------------------------------------- decode attention
// grid (splits of all sequences, heads / 16), 256 threads (8 warps), two CTAs
// per SM. 64-token tiles of the packed rows, two stages of cp.async; the 4-bit
// codes become MMA operands in registers and never pass through shared memory
// unpacked.
//
//   scores   warp w takes latent columns 128c .. 128c+127 (c = w % 4, two groups)
//            for tokens 32h .. 32h+31 (h = w / 4): S[16 heads x 8 tokens] per
//            n-tile, Q' as fp16 A fragments held in registers (a power of two per
//            head keeps its largest value in [2^11, 2^12): 11 significant bits
//            each), codes as B. A 32-bit word of codes gives four B registers by
//            masks alone: nibbles 0 and 4 masked by 0x000f000f are the fp16
//            subnormals u * 2^-24, nibbles 1 and 5 masked by 0x00f000f0 are
//            u * 2^-20 (Q' / 16 there). Accumulators start at -8 sum Q', and each
//            group's is scaled by its tokens' s. The four partial sums meet in
//            shared memory.
//   softmax  warp w adds the rope part (bf16, Q' as hi + lo, for its own tokens
//            8w .. 8w+7: eight MMAs in a row, since a bf16 MMA between two f16 ones
//            costs more than itself) to the sums of its tokens and takes p = 2^(z - M), z = S + e, where
//            2^e bounds the token's scales: p s 2^-e is then at most p. M is set 7
//            below the maximum of z and moves only when that exceeds M by 15 (then O,
//            l are rescaled): most tiles skip the exchange. p is then at most 2^15,
//            which fp16 holds, and weights down to 2^-31 of the largest count (2^-24
//            of it with M at the maximum: 2^18 rows at 2^-25.5 weigh 0.5%, and were
//            lost). l sums p 2^-e in f32.
//   context  warp w owns group w's 64 columns: O[16 x 64] += (p . s 2^-e) U with p,
//            s 2^-e and their product in fp16 (11 bits each), B = code pairs of two
//            tokens from a byte permute and the same masks; a column of ones
//            collects the sum of the weights, whose eightfold is taken off every
//            four tiles: the sums then stay near the size of the result. (The MMAs'
//            f32 sums are truncated; 8 times the weights of a whole split in them
//            cost 0.06 of an output of random signs after 512 tiles.)
// Scales are spread by group once a tile (f32 for the scores, fp16 s 2^-e for the
// context) by the threads that copied them.
//
// Measured, 8 x 32768 rows of 16 heads: 50 us of the call's 62, 105 MB read at 2.1
// TB/s; 1 x 4096: 20 us for the call's three launches. No unit is the bound: of the
// active cycles the tensor pipe works in 37%, an instruction issues in 43%, shared
// memory moves data in 53%, DRAM in 23%. A tile's copy wait, scores, softmax and context
// follow one another in all eight warps, and the 16 warps that an SM holds do not fill
// the gaps: of the 8.4 cycles from one instruction of a warp to its next, 1.5 are fixed
// latencies, 1.3 wait for the tensor pipe, 1.1 for shared memory, 0.8 at barriers.
// (With eight partial sums a score, f32 p and scales read row by row, 27 wavefronts of
// shared memory a token instead of 17: 58 us.)
constexpr uint32_t kQ4Heads = 16, kQ4Tile = 64, kQ4Warps = 8, kQ4Threads = 256, kQ4Stages = 2;
constexpr uint32_t kQ4RopeRow = kQ4Rope * 2 + 16;  // bytes; 9 x 16: eight rows' words on distinct banks
constexpr uint32_t kQ4SRow = kQ4Tile + 8;          // floats; rows 8 banks apart
constexpr uint32_t kQ4PRow = kQ4Tile * 2 + 16;     // bytes of a row of p, against ldmatrix conflicts
constexpr uint32_t kQ4Parts = 4;                   // partial sums of a score
constexpr uint32_t kQ4BiasTiles = 4;               // tiles between two corrections of the context's sums
constexpr uint32_t kQ4ScaleOff = kQ4Tile * kQ4CodeBytes, kQ4RopeOff = kQ4ScaleOff + kQ4Tile * 16;
constexpr uint32_t kQ4StageBytes = kQ4RopeOff + kQ4Tile * kQ4RopeRow;
constexpr uint32_t kQ4PartialFloats = 2 + kQ4Latent;
// stages | partial sums | p | per buffer: scales f32 [8][64], s 2^-e fp16 [8][64], e f32 [64] | rope Q' | maxima
constexpr uint32_t kQ4SpreadBytes = kQ4Groups * kQ4Tile * 6 + kQ4Tile * 4;
constexpr size_t kQ4Smem = size_t(kQ4Stages) * kQ4StageBytes + kQ4Parts * kQ4Heads * kQ4SRow * 4 + kQ4Heads * kQ4PRow +
                           2 * kQ4SpreadBytes + 2 * kQ4Heads * kQ4RopeRow + kQ4Warps * kQ4Heads * 4;
static_assert(kMlaCtasPerSm * (kQ4Smem + 1024) <= 228 * 1024, "two attention CTAs per SM");
static_assert(kQ4Warps == kQ4Groups && kQ4Tile == 8 * kQ4Warps, "a warp: one group, eight tokens of the softmax");
constexpr float kQ4Lift = 7.0f, kQ4Slack = 15.0f;  // M below the maximum when set, and at most

__device__ __forceinline__ void mma16816_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 16-byte chunk c of a tile's code row: chunks are spread so that the score
// reads (8 rows x 4 neighbouring words) and the context reads (rows 0, 2, 4, 6
// or 1, 3, 5, 7 x 8 words) are both free of bank conflicts.
__device__ __forceinline__ uint32_t q4_swz(uint32_t row) { return (row & 6u) ^ ((row & 1u) << 2); }
__global__ void __launch_bounds__(kQ4Threads, kMlaCtasPerSm)
    mla_q4_attn_kernel(const float* __restrict__ qp, const __grid_constant__ MlaQ4Seqs seqs,
                       const __grid_constant__ MlaSplits splits, uint32_t heads, float* __restrict__ partial) {
    extern __shared__ __align__(128) unsigned char smem[];
    float* spart = reinterpret_cast<float*>(smem + kQ4Stages * kQ4StageBytes);  // [parts][16][kQ4SRow]
    unsigned char* pbuf = reinterpret_cast<unsigned char*>(spart + kQ4Parts * kQ4Heads * kQ4SRow);  // [16][kQ4PRow]
    unsigned char* spread = pbuf + kQ4Heads * kQ4PRow;
    unsigned char* qrope = spread + 2 * kQ4SpreadBytes;                          // [2][16][kQ4RopeRow]
    float* wmax = reinterpret_cast<float*>(qrope + 2 * kQ4Heads * kQ4RopeRow);  // [warps][16]
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t g = lane >> 2, t = lane & 3;
    const uint32_t h0 = blockIdx.y * kQ4Heads;
    uint32_t b = 0;
    while (splits.first[b + 1] <= blockIdx.x) ++b;
    const uint32_t t0 = (blockIdx.x - splits.first[b]) * splits.tokens, t1 = min(seqs.len[b], t0 + splits.tokens);
    float* out = partial + (static_cast<size_t>(blockIdx.x) * heads + h0) * kQ4PartialFloats;
    const float NEG_INF = -INFINITY;
    const uint8_t* codes = seqs.codes[b];
    const uint8_t* scales = reinterpret_cast<const uint8_t*>(seqs.scales[b]);
    const uint8_t* krope = reinterpret_cast<const uint8_t*>(seqs.k_rope[b]);
    const uint32_t ntiles = (t1 - t0 + kQ4Tile - 1) / kQ4Tile;

    // thread i copies code chunk i % 16 of rows i / 16 + 16j, rope chunk i % 8 of
    // rows i / 8 + 32j and, below 64, the scales of row i; rows past the split
    // are zero-filled
    auto issue_tile = [&](uint32_t tile) {
        unsigned char* st = smem + (tile % kQ4Stages) * kQ4StageBytes;
        const uint32_t tb = t0 + tile * kQ4Tile;
        const uint32_t cr = tid >> 4, cc = tid & 15;
        unsigned char* cdst = st + cr * kQ4CodeBytes + ((cc ^ q4_swz(cr)) << 4);
        const uint8_t* csrc = codes + static_cast<size_t>(tb + cr) * kQ4CodeBytes + cc * 16;
        const uint32_t rr = tid >> 3, rc = tid & 7;
        unsigned char* rdst = st + kQ4RopeOff + rr * kQ4RopeRow + rc * 16;
        const uint8_t* rsrc = krope + static_cast<size_t>(tb + rr) * (kQ4Rope * 2) + rc * 16;
        const uint8_t* ssrc = scales + static_cast<size_t>(tb + tid) * 16;
        if (tb + kQ4Tile <= t1) {
#pragma unroll
            for (uint32_t j = 0; j < kQ4Tile / 16; ++j) cp16(cdst + j * 16 * kQ4CodeBytes, csrc + j * 16 * kQ4CodeBytes);
#pragma unroll
            for (uint32_t j = 0; j < kQ4Tile / 32; ++j) cp16(rdst + j * 32 * kQ4RopeRow, rsrc + j * 32 * (kQ4Rope * 2));
            if (tid < kQ4Tile) cp16(st + kQ4ScaleOff + tid * 16, ssrc);
        } else {
            for (uint32_t j = 0; j < kQ4Tile / 16; ++j) {
                const bool ok = tb + cr + 16 * j < t1;
                cp16_zfill(cdst + j * 16 * kQ4CodeBytes, ok ? csrc + j * 16 * kQ4CodeBytes : codes, ok ? 16u : 0u);
            }
            for (uint32_t j = 0; j < kQ4Tile / 32; ++j) {
                const bool ok = tb + rr + 32 * j < t1;
                cp16_zfill(rdst + j * 32 * kQ4RopeRow, ok ? rsrc + j * 32 * (kQ4Rope * 2) : krope, ok ? 16u : 0u);
            }
            if (tid < kQ4Tile) {
                const bool ok = tb + tid < t1;
                cp16_zfill(st + kQ4ScaleOff + tid * 16, ok ? ssrc : scales, ok ? 16u : 0u);
            }
        }
    };
    // every attended row was written before this call, whose first launch has
    // waited for it: the first tile is requested before this kernel's wait
    issue_tile(0);
    cp_commit();
    pdl_wait();
    pdl_launch_dependents();

    // Q' fragments of this warp's columns: step (group j, word v, half u) holds
    // at k = 2t, 2t+1 columns c0 + 2u, c0 + 2u + 4 and at k = 2t+8, 2t+9 columns
    // c0 + 2u + 1, c0 + 2u + 5 (divided by 16), c0 = 128 (w % 4) + 64j + 16t + 8v
    const uint32_t cols = warp & 3;
    uint32_t qa[2][4][4];
    float qinit[2][2];  // -8 * 2^-24 * sum of the group's Q', rows g and g+8
    float qscale[2];    // back to true units
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const float* qr = qp + (static_cast<size_t>(b) * heads + h0 + g + 8 * r) * (kQ4Latent + kQ4Rope) + 128 * cols;
        float v[2][16];
        float mx = 0.f;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 x = __ldcg(reinterpret_cast<const float4*>(qr + 64 * j + 16 * t + 4 * i));
                v[j][4 * i] = x.x, v[j][4 * i + 1] = x.y, v[j][4 * i + 2] = x.z, v[j][4 * i + 3] = x.w;
            }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, fabsf(v[j][i]));
        mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 2));
        // 2^(11 - exponent of mx), exponent clamped so that both factors are normal
        const int ex = max(40, min(220, static_cast<int>(__float_as_uint(mx) >> 23)));
        const float up = __uint_as_float(static_cast<uint32_t>(265 - ex) << 23);
        qscale[r] = __uint_as_float(static_cast<uint32_t>(ex - 11 + 24) << 23);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float sum = 0.f;
#pragma unroll
            for (int wd = 0; wd < 2; ++wd)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int c = 8 * wd + 2 * u;
                    const uint32_t lo = cvt_f16x2(v[j][c] * up, v[j][c + 4] * up);
                    const uint32_t hi = cvt_f16x2(v[j][c + 1] * up * 0.0625f, v[j][c + 5] * up * 0.0625f);
                    qa[j][2 * wd + u][r] = lo;
                    qa[j][2 * wd + u][2 + r] = hi;
                    const float2 fl = __half22float2(*reinterpret_cast<const __half2*>(&lo));
                    const float2 fh = __half22float2(*reinterpret_cast<const __half2*>(&hi));
                    sum += (fl.x + fl.y) + 16.0f * (fh.x + fh.y);
                }
            sum += __shfl_xor_sync(kFull, sum, 1);
            sum += __shfl_xor_sync(kFull, sum, 2);
            qinit[j][r] = sum * (-8.0f / 16777216.0f);
        }
    }
    {  // the rope part's A operands, bf16 hi and the rest, in shared memory
        const uint32_t row = tid >> 4, c = (tid & 15) * 4;
        const float4 v = __ldcg(reinterpret_cast<const float4*>(
            qp + (static_cast<size_t>(b) * heads + h0 + row) * (kQ4Latent + kQ4Rope) + kQ4Latent + c));
        const uint2 hi = make_uint2(cvt_bf16x2(v.x, v.y), cvt_bf16x2(v.z, v.w));
        *reinterpret_cast<uint2*>(qrope + row * kQ4RopeRow + c * 2) = hi;
        *reinterpret_cast<uint2*>(qrope + (kQ4Heads + row) * kQ4RopeRow + c * 2) =
            make_uint2(cvt_bf16x2(v.x - bf16_lo(hi.x), v.y - bf16_hi(hi.x)),
                       cvt_bf16x2(v.z - bf16_lo(hi.y), v.w - bf16_hi(hi.y)));
    }

    float M[2] = {NEG_INF, NEG_INF}, l[2] = {0.f, 0.f};
    float o[8][4], ones[4] = {0.f, 0.f, 0.f, 0.f};  // context columns of nibble n; sums of p s
#pragma unroll
    for (int n = 0; n < 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    // the lane's places in a tile: codes of token row g (scores), of tokens
    // 2t + e (context), both for whole groups of 8 rows by fixed steps
    const uint32_t tok_q = 32 * (warp >> 2);  // first token of the warp's scores
    const uint32_t sc_code = (tok_q + g) * kQ4CodeBytes + (((4 * cols + (t >> 1)) ^ q4_swz(g)) << 4) + (t & 1) * 8;
    const uint32_t sc_code2 = (tok_q + g) * kQ4CodeBytes + (((4 * cols + 2 + (t >> 1)) ^ q4_swz(g)) << 4) + (t & 1) * 8;
    uint32_t pv_code[2];
#pragma unroll
    for (uint32_t e = 0; e < 2; ++e)
        pv_code[e] = (2 * t + e) * kQ4CodeBytes + (((2 * warp + (g >> 2)) ^ q4_swz(2 * t + e)) << 4) + (g & 3) * 4;

    // the eightfold of the weights off the sums of stored nibbles (u 2^-24, odd n u 2^-20)
    auto take_bias = [&]() {
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n][i] = fmaf(ones[i], (n & 1) ? -8.0f / 1048576.0f : -8.0f / 16777216.0f, o[n][i]);
        ones[0] = ones[1] = ones[2] = ones[3] = 0.f;
    };

    for (uint32_t tile = 0; tile < ntiles; ++tile) {
        cp_wait<0>();
        const unsigned char* st = smem + (tile % kQ4Stages) * kQ4StageBytes;
        float* sq = reinterpret_cast<float*>(spread + (tile & 1) * kQ4SpreadBytes);  // [8][64]
        __half* sp = reinterpret_cast<__half*>(sq + kQ4Groups * kQ4Tile);            // [8][64]
        float* eb = reinterpret_cast<float*>(sp + kQ4Groups * kQ4Tile);              // [64]
        if (tid < kQ4Tile) {  // the scales that this thread copied, by group
            const uint4 q = *reinterpret_cast<const uint4*>(st + kQ4ScaleOff + tid * 16);
            uint32_t m = __vmaxu2(__vmaxu2(q.x, q.y), __vmaxu2(q.z, q.w));
            m = max(m & 0xffffu, m >> 16);
            // 2^e > every scale of the token (a NaN scale counts as the largest)
            const int e = max(-40, min(100, static_cast<int>(m >> 7) - 126));
            const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float lo = bf16_lo(w[i]), hi = bf16_hi(w[i]);
                sq[(2 * i) * kQ4Tile + tid] = lo;
                sq[(2 * i + 1) * kQ4Tile + tid] = hi;
                sp[(2 * i) * kQ4Tile + tid] = __float2half_rn(lo * down);
                sp[(2 * i + 1) * kQ4Tile + tid] = __float2half_rn(hi * down);
            }
            eb[tid] = static_cast<float>(e);
        }
        __syncthreads();  // tile landed; everyone is done with the previous one
        if (tile + 1 < ntiles) issue_tile(tile + 1);
        cp_commit();
        if (tile % kQ4BiasTiles == 0 && tile) take_bias();  // (right after the MMAs it would wait for them: 63.4 us for 62.7)
        // ---- partial scores over this warp's columns, 8 tokens at a time
        float* sw = spart + cols * kQ4Heads * kQ4SRow + tok_q + 2 * t;
        const float* sg = sq + 2 * cols * kQ4Tile + tok_q + 2 * t;
#pragma unroll
        for (uint32_t n = 0; n < 4; ++n) {
            const uint2 w0 = *reinterpret_cast<const uint2*>(st + sc_code + n * 8 * kQ4CodeBytes);
            const uint2 w1 = *reinterpret_cast<const uint2*>(st + sc_code2 + n * 8 * kQ4CodeBytes);
            const float2 s0 = *reinterpret_cast<const float2*>(sg + n * 8);
            const float2 s1 = *reinterpret_cast<const float2*>(sg + kQ4Tile + n * 8);
            float acc[2][4];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                acc[j][0] = acc[j][1] = qinit[j][0];
                acc[j][2] = acc[j][3] = qinit[j][1];
            }
            const uint32_t wd[2][2] = {{w0.x, w0.y}, {w1.x, w1.y}};
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t x = wd[j][i] >> (8 * u);
                        mma16816_f16(acc[j], qa[j][2 * i + u], x & 0x000f000fu, x & 0x00f000f0u);
                    }
            *reinterpret_cast<float2*>(sw + g * kQ4SRow + n * 8) =
                make_float2(qscale[0] * fmaf(s0.x, acc[0][0], s1.x * acc[1][0]),
                            qscale[0] * fmaf(s0.y, acc[0][1], s1.y * acc[1][1]));
            *reinterpret_cast<float2*>(sw + (g + 8) * kQ4SRow + n * 8) =
                make_float2(qscale[1] * fmaf(s0.x, acc[0][2], s1.x * acc[1][2]),
                            qscale[1] * fmaf(s0.y, acc[0][3], s1.y * acc[1][3]));
        }
        // the rope part of this warp's own tokens 8w .. 8w+7
        float ra[2][4] = {};  // hi, rest
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            uint32_t rb[4];
            ldsm_x4(rb, st + kQ4RopeOff + (8 * warp + (lane & 7)) * kQ4RopeRow + ((lane >> 3) * 8 + 32 * m) * 2);
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint32_t qf[4];
                    ldsm_x4(qf, qrope + (i * kQ4Heads + (lane & 15)) * kQ4RopeRow + ((2 * m + u) * 16 + (lane >> 4) * 8) * 2);
                    mma16816(ra[i], qf, rb[2 * u], rb[2 * u + 1]);
                }
        }
        __syncthreads();  // every warp's partial scores written
        // ---- softmax of tokens 8w .. 8w+7: z[r][e] = head g + 8r, token 8w + 2t + e
        float z[2][2], zmax[2];
        const uint32_t tok = 8 * warp + 2 * t, tb = t0 + tile * kQ4Tile;
        const float2 e2 = *reinterpret_cast<const float2*>(eb + tok);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float2 v[kQ4Parts];
#pragma unroll
            for (uint32_t w = 0; w < kQ4Parts; ++w)
                v[w] = *reinterpret_cast<const float2*>(spart + (w * kQ4Heads + g + 8 * r) * kQ4SRow + tok);
            z[r][0] = tb + tok < t1 ? ((v[0].x + v[1].x) + (v[2].x + v[3].x)) + (ra[0][2 * r] + ra[1][2 * r]) + e2.x : NEG_INF;
            z[r][1] = tb + tok + 1 < t1 ? ((v[0].y + v[1].y) + (v[2].y + v[3].y)) + (ra[0][2 * r + 1] + ra[1][2 * r + 1]) + e2.y : NEG_INF;
            zmax[r] = fmaxf(z[r][0], z[r][1]);
        }
        const float2 down = make_float2(__uint_as_float(static_cast<uint32_t>(127 - static_cast<int>(e2.x)) << 23),
                                        __uint_as_float(static_cast<uint32_t>(127 - static_cast<int>(e2.y)) << 23));
        float lt[2];
        auto write_p = [&]() {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float p0 = exp2f(z[r][0] - M[r]), p1 = exp2f(z[r][1] - M[r]);
                lt[r] = fmaf(p0, down.x, p1 * down.y);
                *reinterpret_cast<uint32_t*>(pbuf + (g + 8 * r) * kQ4PRow + tok * 2) = cvt_f16x2(p0, p1);
            }
        };
        const bool over = M[0] == NEG_INF || zmax[0] > M[0] + kQ4Slack || zmax[1] > M[1] + kQ4Slack;
        write_p();
        if (__syncthreads_or(over)) {  // P complete, unless the maximum moved
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                zmax[r] = fmaxf(zmax[r], __shfl_xor_sync(kFull, zmax[r], 1));
                zmax[r] = fmaxf(zmax[r], __shfl_xor_sync(kFull, zmax[r], 2));
                if (t == 0) wmax[warp * kQ4Heads + g + 8 * r] = zmax[r];
            }
            __syncthreads();
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float m = M[r];
#pragma unroll
                for (uint32_t w = 0; w < kQ4Warps; ++w) m = fmaxf(m, wmax[w * kQ4Heads + g + 8 * r] - kQ4Lift);
                if (m == NEG_INF) m = -1e38f;  // only -inf or NaN so far: finite, so that NaN alone stays NaN, and below every score
                const float alpha = exp2f(M[r] - m);
                M[r] = m;
                l[r] *= alpha;
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    o[n][2 * r] *= alpha;
                    o[n][2 * r + 1] *= alpha;
                }
                ones[2 * r] *= alpha;
                ones[2 * r + 1] *= alpha;
            }
            write_p();
            __syncthreads();  // P complete
        }
        l[0] += lt[0];
        l[1] += lt[1];
        // ---- context: 16 tokens a step
#pragma unroll
        for (uint32_t kb = 0; kb < kQ4Tile / 16; ++kb) {
            const uint32_t tk = kb * 16 + 2 * t;  // tokens tk, tk+1, tk+8, tk+9
            uint32_t w[4], pa[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                w[e] = *reinterpret_cast<const uint32_t*>(st + pv_code[e & 1] + (kb * 16 + 8 * (e >> 1)) * kQ4CodeBytes);
            ldsm_x4(pa, pbuf + (lane & 15) * kQ4PRow + (kb * 16 + (lane >> 4) * 8) * 2);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const __half2 f = *reinterpret_cast<const __half2*>(sp + warp * kQ4Tile + tk + 8 * e);
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    __half2& x = *reinterpret_cast<__half2*>(&pa[2 * e + r]);
                    x = __hmul2(x, f);
                }
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {  // nibbles 0-3 and 4-7
                const uint32_t x0 = __byte_perm(w[0], w[1], half ? 0x7632 : 0x5410);
                const uint32_t x1 = __byte_perm(w[2], w[3], half ? 0x7632 : 0x5410);
                const uint32_t y0 = x0 >> 8, y1 = x1 >> 8;
                mma16816_f16(o[4 * half], pa, x0 & 0x000f000fu, x1 & 0x000f000fu);
                mma16816_f16(o[4 * half + 1], pa, x0 & 0x00f000f0u, x1 & 0x00f000f0u);
                mma16816_f16(o[4 * half + 2], pa, y0 & 0x000f000fu, y1 & 0x000f000fu);
                mma16816_f16(o[4 * half + 3], pa, y0 & 0x00f000f0u, y1 & 0x00f000f0u);
            }
            mma16816_f16(ones, pa, 0x3c003c00u, 0x3c003c00u);
        }
    }
    take_bias();
    cp_wait<0>();

    // ---- split partial: maximum, sum, O
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(kFull, l[r], 1);
        l[r] += __shfl_xor_sync(kFull, l[r], 2);
        if (t == 0) wmax[warp * kQ4Heads + g + 8 * r] = l[r];  // this warp's tokens
    }
    __syncthreads();
    if (tid < kQ4Heads) {
        float sum = 0.f;
#pragma unroll
        for (uint32_t w = 0; w < kQ4Warps; ++w) sum += wmax[w * kQ4Heads + tid];
        out[tid * kQ4PartialFloats + 1] = sum;
    }
    if (warp == 0 && t == 0) {
        out[g * kQ4PartialFloats] = M[0];
        out[(g + 8) * kQ4PartialFloats] = M[1];
    }
    // column of accumulator n, element e: 64w + 8(2t + e) + n
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float v[8];
#pragma unroll
            for (int n = 0; n < 8; ++n)
                v[n] = o[n][2 * r + e] * ((n & 1) ? 1048576.0f : 16777216.0f);
            float* dst = out + (g + 8 * r) * kQ4PartialFloats + 2 + 64 * warp + 8 * (2 * t + e);
#pragma unroll
            for (int n = 0; n < 8; n += 2) *reinterpret_cast<float2*>(dst + n) = make_float2(v[n], v[n + 1]);
        }
}

// Splits: the fewest whole tiles a CTA for which the splits of all sequences and
// head blocks still fit one wave of the two CTAs an SM runs (a sequence of any
// length has one at least), so that a batch of mixed lengths shares the SMs by
// its rows.
void mla_q4_plan_splits(uint32_t batch, uint32_t heads, const uint32_t* lens, int num_sms, MlaSplits& s) {
    const uint64_t wave = std::max<uint64_t>(kMlaCtasPerSm * static_cast<uint64_t>(num_sms) / (heads / kQ4Heads), batch);
    auto count = [&](uint64_t tokens) {
        uint64_t n = 0;
        for (uint32_t b = 0; b < batch; ++b) n += (lens[b] + tokens - 1) / tokens;
        return n;
    };
    uint64_t lo = 1, hi = 1;  // tiles a split
    while (count(hi * kQ4Tile) > wave) hi *= 2;
    while (lo < hi) {
        const uint64_t mid = (lo + hi) / 2;
        if (count(mid * kQ4Tile) > wave)
            lo = mid + 1;
        else
            hi = mid;
    }
    s.tokens = static_cast<uint32_t>(std::min<uint64_t>(hi * kQ4Tile, 0xffffffc0u));
    s.first[0] = 0;
    for (uint32_t b = 0; b < kMlaMaxBatch; ++b)
        s.first[b + 1] =
            s.first[b] + (b < batch ? static_cast<uint32_t>((uint64_t(lens[b]) + s.tokens - 1) / s.tokens) : 0);
}

// The kernels' shared memory, once per device (set where the workspace is).
cudaError_t mla_q4_prepare() {
    cudaError_t e = cudaFuncSetAttribute(mla_q4_attn_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(kQ4Smem));
    return e != cudaSuccess ? e : mla_merge_out_prepare();
}

cudaError_t mla_q4_decode_launch(const MlaLaunch& a, const MlaQ4Seqs& seqs, const MlaSplits& splits, uint32_t heads,
                                 cudaStream_t s) {
    cudaError_t e = mla_absorb_launch(a, heads, s);
    if (e != cudaSuccess) return e;
    if ((e = launch_pdl_kernel(mla_q4_attn_kernel, dim3(splits.first[kMlaMaxBatch], heads / kQ4Heads), dim3(kQ4Threads),
                               kQ4Smem, s, a.qp, seqs, splits, heads, a.partial)) != cudaSuccess)
        return e;
    return mla_merge_out_launch(a, splits, heads, s);
}

}  // namespace pbmoe
