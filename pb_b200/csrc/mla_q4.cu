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

#include "common.cuh"
#include "kernels.h"
#include "mma_sync.cuh"

namespace pbmoe {

constexpr uint32_t kQ4Latent = 512, kQ4Rope = 64, kQ4Group = 64;
constexpr uint32_t kQ4Groups = kQ4Latent / kQ4Group;  // 8 scales per row
constexpr uint32_t kQ4CodeBytes = kQ4Latent / 2;

// f32 pair -> bf16x2 bits (round to nearest even, NaN stays NaN).
__device__ __forceinline__ uint32_t cvt_bf16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t cvt_f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// ---------------------------------------------------------------- append
// One CTA per token, 256 threads. Thread i holds latent columns 2i and 2i+1
// (one byte of codes), so warp g is quantisation group g and the group's
// maximum is a warp reduction. The mean square is summed in f64: a code next
// to a rounding border is then the same whatever the order of the sum. A warp
// rotates whole heads of the query (lane p: pair p), reading a head's pairs
// before it writes any, so the query may be rotated in place.
constexpr int kQ4AppendThreads = 256;
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

// The head's rotated part (and, out of place, its nope part) of one token.
template <typename QT, typename OT>
__device__ __forceinline__ void rotate_head(const QT* q, OT* out, uint32_t nope, float2 cs, bool copy_nope) {
    const uint32_t lane = threadIdx.x & 31;
    const float2 v = load_pair(q + nope + 2 * lane);
    if (copy_nope)
        for (uint32_t i = 2 * lane; i < nope; i += 64) store_pair(out + i, load_pair(q + i));
    const float r0 = __fsub_rn(__fmul_rn(v.x, cs.x), __fmul_rn(v.y, cs.y));
    const float r1 = __fadd_rn(__fmul_rn(v.y, cs.x), __fmul_rn(v.x, cs.y));
    __syncwarp();  // every pair of the head read
    store_one(out + nope + lane, r0);
    store_one(out + nope + 32 + lane, r1);
}

template <typename KT, typename QT, typename OT>
__global__ void __launch_bounds__(kQ4AppendThreads) mla_q4_append_kernel(const __grid_constant__ MlaQ4Append a) {
    __shared__ double red[kQ4AppendThreads / 32];
    const uint32_t tok = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t seq = a.sequences ? a.sequences[tok] : tok;
    const uint32_t pos = a.positions[tok];
    if (seq >= a.batch || pos >= a.max_positions || pos >= a.seqs.len[min(seq, kMlaMaxBatch - 1)]) {
        if (tid == 0) latch_status(a.status, PBMOE_DEV_ERR_POSITION);
        return;
    }
    const KT* kv = static_cast<const KT*>(a.kv) + static_cast<size_t>(tok) * (kQ4Latent + kQ4Rope);
    const float2 cs = a.table[static_cast<size_t>(pos) * (kQ4Rope / 2) + lane];
    float2 x = load_pair(kv + 2 * tid);
    float2 key = make_float2(0.f, 0.f);
    if (warp == 0) key = load_pair(kv + kQ4Latent + 2 * lane);
    if (a.query) {
        const uint32_t qk = a.nope + kQ4Rope;
        const QT* q = static_cast<const QT*>(a.query) + static_cast<size_t>(tok) * a.heads * qk;
        OT* qo = static_cast<OT*>(a.query_out) + static_cast<size_t>(tok) * a.heads * qk;
        const bool copy = a.query_out != a.query;
        for (uint32_t h = warp; h < a.heads; h += kQ4AppendThreads / 32)
            rotate_head(q + h * qk, qo + h * qk, a.nope, cs, copy);
    }
    if (a.latent_norm_w) {
        double ss = static_cast<double>(x.x) * x.x + static_cast<double>(x.y) * x.y;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(kFull, ss, o);
        if (lane == 0) red[warp] = ss;
        __syncthreads();
        double tot = 0;
#pragma unroll
        for (int w = 0; w < kQ4AppendThreads / 32; ++w) tot += red[w];
        const float scale = static_cast<float>(1.0 / sqrt(tot / kQ4Latent + static_cast<double>(a.eps)));
        const float2 w = *reinterpret_cast<const float2*>(a.latent_norm_w + 2 * tid);
        x.x = __fmul_rn(__fmul_rn(x.x, scale), w.x);
        x.y = __fmul_rn(__fmul_rn(x.y, scale), w.y);
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
        q0 = max(-7, min(7, __float2int_rn(__fdiv_rn(x.x, s))));
        q1 = max(-7, min(7, __float2int_rn(__fdiv_rn(x.y, s))));
    }
    const size_t row = pos;
    const uint32_t byte = static_cast<uint32_t>(q0 + 8) | (static_cast<uint32_t>(q1 + 8) << 4);
    // four lanes' bytes to one word
    uint32_t word = byte << (8 * (lane & 3));
    word |= __shfl_xor_sync(kFull, word, 1);
    word |= __shfl_xor_sync(kFull, word, 2);
    if ((lane & 3) == 0)
        *reinterpret_cast<uint32_t*>(a.seqs.codes[seq] + row * kQ4CodeBytes + 2 * tid / 2) = word;
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

namespace {
template <typename KT, typename QT>
cudaError_t append_out(const MlaQ4Append& a, cudaStream_t s) {
    const dim3 g(a.tokens), b(kQ4AppendThreads);
    if (a.query_out_dtype == PBMOE_F32)
        return launch_pdl_kernel(mla_q4_append_kernel<KT, QT, float>, g, b, 0, s, a);
    return launch_pdl_kernel(mla_q4_append_kernel<KT, QT, uint16_t>, g, b, 0, s, a);
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
// (8 bytes) into 32 bytes, lanes 0-7 copy the key part.
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
    for (uint32_t r = r0 + warp; r < r1; r += kQ4ReadThreads / 32) {
        const size_t row = static_cast<size_t>(a.begin[b]) + r, dst = static_cast<size_t>(a.offset[b]) + r;
        const uint2 w = ld_stream_u2(codes + row * kQ4CodeBytes + 8 * lane);
        const float s = bf16_bits_to_f32(scales[row * kQ4Groups + lane / 4]);
        uint4 key = make_uint4(0, 0, 0, 0);
        if (a.k_rope && lane < 8) key = *reinterpret_cast<const uint4*>(krope + row * kQ4Rope + 8 * lane);
        uint32_t o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t u = (i < 4 ? w.x : w.y) >> (8 * (i & 3));
            o[i] = cvt_bf16x2(static_cast<float>(static_cast<int>(u & 15u) - 8) * s,
                              static_cast<float>(static_cast<int>((u >> 4) & 15u) - 8) * s);
        }
        uint4* out = reinterpret_cast<uint4*>(a.c_kv + dst * kQ4Latent + 16 * lane);
        out[0] = make_uint4(o[0], o[1], o[2], o[3]);
        out[1] = make_uint4(o[4], o[5], o[6], o[7]);
        if (a.k_rope && lane < 8) *reinterpret_cast<uint4*>(a.k_rope + dst * kQ4Rope + 8 * lane) = key;
    }
}

cudaError_t mla_q4_read_launch(const MlaQ4Read& a, uint32_t max_count, cudaStream_t s) {
    if (max_count == 0) return cudaSuccess;
    const dim3 grid((max_count + kQ4ReadRows - 1) / kQ4ReadRows, a.batch);
    return launch_pdl_kernel(mla_q4_read_kernel, grid, dim3(kQ4ReadThreads), 0, s, a);
}

// ---------------------------------------------------------------- decode attention
// grid (splits, batch, heads / 16), 128 threads (4 warps), two CTAs per SM.
// 64-token tiles of the packed rows, three stages of cp.async; the 4-bit
// codes become MMA operands in registers and never pass through shared
// memory unpacked.
//
// Warp w owns latent columns 128w .. 128w+127 (two groups) in both products.
//   scores   S[16 heads x 8 tokens] per n-tile: Q' as fp16 A fragments held in
//            registers (a power of two per head keeps its largest value in
//            [2^11, 2^12): 11 significant bits each), codes as B. A 32-bit word
//            of codes gives four B registers by masks alone: nibbles 0 and 4
//            masked by 0x000f000f are the fp16 subnormals u * 2^-24, nibbles
//            1 and 5 masked by 0x00f000f0 are u * 2^-20 (Q' / 16 there).
//            Accumulators start at -8 sum Q', and each group's is scaled by
//            its tokens' s. The rope part adds one k16 step a warp (Q' as bf16
//            hi + lo). Partial sums of the four warps meet in shared memory.
//   softmax  warp w sums tokens 16w .. 16w+15 and takes p = 2^(S - M) in f32.
//            M follows the maximum of S + log2(bound of the token's scales),
//            so that p * s fits fp16, and moves only when it is exceeded by
//            2^8 (then O, l are rescaled): most tiles skip the exchange.
//   context  O[16 x 128] += (p s_g) U: P s as fp16 A fragments, B = code pairs
//            of two tokens from a byte permute and the same masks; a column of
//            ones collects sum p s, whose eightfold is taken off at the end.
constexpr uint32_t kQ4Heads = 16, kQ4Tile = 64, kQ4Warps = 4, kQ4Threads = 128, kQ4Stages = 3;
constexpr uint32_t kQ4RopeRow = kQ4Rope * 2 + 16;  // bytes; 9 x 16: eight rows' words on distinct banks
constexpr uint32_t kQ4SRow = kQ4Tile + 8;          // floats; rows 8 banks apart
constexpr uint32_t kQ4ScaleOff = kQ4Tile * kQ4CodeBytes, kQ4RopeOff = kQ4ScaleOff + kQ4Tile * 16;
constexpr uint32_t kQ4StageBytes = kQ4RopeOff + kQ4Tile * kQ4RopeRow;
constexpr uint32_t kQ4PartialFloats = 2 + kQ4Latent;
constexpr size_t kQ4Smem = size_t(kQ4Stages) * kQ4StageBytes + (kQ4Warps + 1) * kQ4Heads * kQ4SRow * 4 +
                           kQ4Warps * kQ4Heads * 4;
static_assert(kMlaCtasPerSm * (kQ4Smem + 1024) <= 228 * 1024, "two attention CTAs per SM");
constexpr float kQ4Slack = 8.0f;  // M may lag the maximum by 2^8: p s <= 2^9 in fp16

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
    mla_q4_attn_kernel(const float* __restrict__ qp, const __grid_constant__ MlaQ4Seqs seqs, uint32_t heads,
                       uint32_t split_tokens, uint32_t splits, float* __restrict__ partial) {
    extern __shared__ __align__(128) unsigned char smem[];
    float* spart = reinterpret_cast<float*>(smem + kQ4Stages * kQ4StageBytes);  // [warps][16][kQ4SRow]
    float* pbuf = spart + kQ4Warps * kQ4Heads * kQ4SRow;                       // [16][kQ4SRow]
    float* wmax = pbuf + kQ4Heads * kQ4SRow;                                   // [warps][16]
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t g = lane >> 2, t = lane & 3;
    const uint32_t b = blockIdx.y, sp = blockIdx.x, h0 = blockIdx.z * kQ4Heads;
    const uint32_t L = seqs.len[b];
    const uint32_t t0 = sp * split_tokens, t1 = min(L, t0 + split_tokens);
    float* out = partial + ((static_cast<size_t>(b) * splits + sp) * heads + h0) * kQ4PartialFloats;
    const float NEG_INF = -INFINITY;
    if (t0 >= t1) {  // empty split: contributes nothing
        pdl_wait();
        pdl_launch_dependents();
        for (uint32_t i = tid; i < kQ4Heads * kQ4PartialFloats; i += kQ4Threads)
            out[i] = (i % kQ4PartialFloats == 0) ? NEG_INF : 0.f;
        return;
    }
    const uint8_t* codes = seqs.codes[b];
    const uint8_t* scales = reinterpret_cast<const uint8_t*>(seqs.scales[b]);
    const uint8_t* krope = reinterpret_cast<const uint8_t*>(seqs.k_rope[b]);
    const uint32_t ntiles = (t1 - t0 + kQ4Tile - 1) / kQ4Tile;

    // thread i copies code chunk i % 16 of rows i / 16 + 8j, rope chunk i % 8 of
    // rows i / 8 + 16j and, below 64, the scales of row i; rows past the split
    // are zero-filled
    auto issue_tile = [&](uint32_t tile) {
        unsigned char* st = smem + (tile % kQ4Stages) * kQ4StageBytes;
        const uint32_t tb = t0 + tile * kQ4Tile;
        const uint32_t cr = tid >> 4, cc = tid & 15;
        unsigned char* cdst = st + cr * kQ4CodeBytes + ((cc ^ q4_swz(cr)) << 4);
        const uint8_t* csrc = codes + static_cast<size_t>(tb + cr) * kQ4CodeBytes + cc * 16;
#pragma unroll
        for (uint32_t j = 0; j < kQ4Tile / 8; ++j) {
            const bool ok = tb + cr + 8 * j < t1;
            cp16_zfill(cdst + j * 8 * kQ4CodeBytes, ok ? csrc + j * 8 * kQ4CodeBytes : codes, ok ? 16u : 0u);
        }
        const uint32_t rr = tid >> 3, rc = tid & 7;
        unsigned char* rdst = st + kQ4RopeOff + rr * kQ4RopeRow + rc * 16;
        const uint8_t* rsrc = krope + static_cast<size_t>(tb + rr) * (kQ4Rope * 2) + rc * 16;
#pragma unroll
        for (uint32_t j = 0; j < kQ4Tile / 16; ++j) {
            const bool ok = tb + rr + 16 * j < t1;
            cp16_zfill(rdst + j * 16 * kQ4RopeRow, ok ? rsrc + j * 16 * (kQ4Rope * 2) : krope, ok ? 16u : 0u);
        }
        if (tid < kQ4Tile) {
            const bool ok = tb + tid < t1;
            cp16_zfill(st + kQ4ScaleOff + tid * 16, ok ? scales + static_cast<size_t>(tb + tid) * 16 : scales,
                       ok ? 16u : 0u);
        }
    };
    // every attended row was written before this call, whose first launch has
    // waited for it: the first tiles are requested before this kernel's wait
#pragma unroll
    for (uint32_t i = 0; i < kQ4Stages - 1; ++i) {
        if (i < ntiles) issue_tile(i);
        cp_commit();
    }
    pdl_wait();
    pdl_launch_dependents();

    // Q' fragments of this warp's columns: step (group j, word v, half u) holds
    // at k = 2t, 2t+1 columns c0 + 2u, c0 + 2u + 4 and at k = 2t+8, 2t+9 columns
    // c0 + 2u + 1, c0 + 2u + 5 (divided by 16), c0 = 128w + 64j + 16t + 8v
    uint32_t qa[2][4][4];
    float qinit[2][2];  // -8 * 2^-24 * sum of the group's Q', rows g and g+8
    float qscale[2];    // back to true units
    {
        const float* qr[2] = {qp + (static_cast<size_t>(b) * heads + h0 + g) * (kQ4Latent + kQ4Rope),
                              qp + (static_cast<size_t>(b) * heads + h0 + g + 8) * (kQ4Latent + kQ4Rope)};
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float v[2][16];
            float mx = 0.f;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float4 x = __ldcg(reinterpret_cast<const float4*>(qr[r] + 128 * warp + 64 * j + 16 * t + 4 * i));
                    v[j][4 * i] = x.x, v[j][4 * i + 1] = x.y, v[j][4 * i + 2] = x.z, v[j][4 * i + 3] = x.w;
                    mx = fmaxf(fmaxf(fmaxf(mx, fabsf(x.x)), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
                }
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
    }
    // rope part, k16 step `warp`, bf16 hi and lo
    uint32_t rh[4], rl[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float* q = qp + (static_cast<size_t>(b) * heads + h0 + g + 8 * (i & 1)) * (kQ4Latent + kQ4Rope) +
                         kQ4Latent + 16 * warp + 2 * t + 8 * (i >> 1);
        const float2 v = __ldcg(reinterpret_cast<const float2*>(q));
        rh[i] = cvt_bf16x2(v.x, v.y);
        rl[i] = cvt_bf16x2(v.x - bf16_lo(rh[i]), v.y - bf16_hi(rh[i]));
    }

    float M[2] = {NEG_INF, NEG_INF}, l[2] = {0.f, 0.f};
    float o[2][8][4], ones[2][4];  // context of group j, columns of nibble n; sums of p s
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int n = 0; n < 8; ++n) o[j][n][0] = o[j][n][1] = o[j][n][2] = o[j][n][3] = 0.f;
        ones[j][0] = ones[j][1] = ones[j][2] = ones[j][3] = 0.f;
    }

    for (uint32_t tile = 0; tile < ntiles; ++tile) {
        cp_wait<kQ4Stages - 2>();
        __syncthreads();  // tile landed; everyone is done with the previous one
        if (tile + kQ4Stages - 1 < ntiles) issue_tile(tile + kQ4Stages - 1);
        cp_commit();
        const unsigned char* st = smem + (tile % kQ4Stages) * kQ4StageBytes;
        const unsigned char* sc = st + kQ4ScaleOff;
        const unsigned char* rt = st + kQ4RopeOff;
        // ---- partial scores over this warp's columns, 8 tokens at a time
        float* sw = spart + warp * kQ4Heads * kQ4SRow;
#pragma unroll 2
        for (uint32_t n = 0; n < kQ4Tile / 8; ++n) {
            const uint32_t row = n * 8 + g;
            float acc[2][4], ra[4] = {0.f, 0.f, 0.f, 0.f};
            const unsigned char* rrow = rt + row * kQ4RopeRow + 32 * warp + 4 * t;
            const uint32_t rb0 = *reinterpret_cast<const uint32_t*>(rrow);
            const uint32_t rb1 = *reinterpret_cast<const uint32_t*>(rrow + 16);
            const uint32_t sa = *reinterpret_cast<const uint32_t*>(sc + (n * 8 + 2 * t) * 16 + 4 * warp);
            const uint32_t sb = *reinterpret_cast<const uint32_t*>(sc + (n * 8 + 2 * t + 1) * 16 + 4 * warp);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t chunk = (4 * warp + 2 * j + (t >> 1)) ^ q4_swz(g);
                const uint2 w = *reinterpret_cast<const uint2*>(st + row * kQ4CodeBytes + chunk * 16 + (t & 1) * 8);
                acc[j][0] = acc[j][1] = qinit[j][0];
                acc[j][2] = acc[j][3] = qinit[j][1];
                const uint32_t wd[2] = {w.x, w.y};
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    mma16816_f16(acc[j], qa[j][2 * i], wd[i] & 0x000f000fu, wd[i] & 0x00f000f0u);
                    const uint32_t hi = wd[i] >> 8;
                    mma16816_f16(acc[j], qa[j][2 * i + 1], hi & 0x000f000fu, hi & 0x00f000f0u);
                }
            }
            mma16816(ra, rh, rb0, rb1);
            mma16816(ra, rl, rb0, rb1);
            const float s00 = bf16_lo(sa), s01 = bf16_hi(sa), s10 = bf16_lo(sb), s11 = bf16_hi(sb);
            const uint32_t col = n * 8 + 2 * t;
            *reinterpret_cast<float2*>(sw + g * kQ4SRow + col) =
                make_float2(fmaf(qscale[0], fmaf(s00, acc[0][0], s01 * acc[1][0]), ra[0]),
                            fmaf(qscale[0], fmaf(s10, acc[0][1], s11 * acc[1][1]), ra[1]));
            *reinterpret_cast<float2*>(sw + (g + 8) * kQ4SRow + col) =
                make_float2(fmaf(qscale[1], fmaf(s00, acc[0][2], s01 * acc[1][2]), ra[2]),
                            fmaf(qscale[1], fmaf(s10, acc[0][3], s11 * acc[1][3]), ra[3]));
        }
        __syncthreads();  // every warp's partial scores written
        // ---- softmax of tokens 16w .. 16w+15: s[i][r][e] = head g + 8r, token 16w + 8i + 2t + e
        float s[2][2][2];
        float zmax[2] = {NEG_INF, NEG_INF};
        const uint32_t tb = t0 + tile * kQ4Tile;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t tok = 16 * warp + 8 * i + 2 * t;
            float ebound[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {  // 2^ebound > every scale of the token
                const uint4 q = *reinterpret_cast<const uint4*>(sc + (tok + e) * 16);
                uint32_t m = __vmaxu2(__vmaxu2(q.x, q.y), __vmaxu2(q.z, q.w));
                m = max(m & 0xffffu, m >> 16);
                ebound[e] = static_cast<float>(max(-40, min(100, static_cast<int>(m >> 7) - 126)));
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float2 acc = make_float2(0.f, 0.f);
#pragma unroll
                for (uint32_t w = 0; w < kQ4Warps; ++w) {
                    const float2 v =
                        *reinterpret_cast<const float2*>(spart + (w * kQ4Heads + g + 8 * r) * kQ4SRow + tok);
                    acc.x += v.x;
                    acc.y += v.y;
                }
                s[i][r][0] = tb + tok < t1 ? acc.x : NEG_INF;
                s[i][r][1] = tb + tok + 1 < t1 ? acc.y : NEG_INF;
                zmax[r] = fmaxf(zmax[r], fmaxf(s[i][r][0] + ebound[0], s[i][r][1] + ebound[1]));
            }
        }
        float lt[2];
        auto write_p = [&]() {
            lt[0] = lt[1] = 0.f;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float2 p = make_float2(exp2f(s[i][r][0] - M[r]), exp2f(s[i][r][1] - M[r]));
                    lt[r] += p.x + p.y;
                    *reinterpret_cast<float2*>(pbuf + (g + 8 * r) * kQ4SRow + 16 * warp + 8 * i + 2 * t) = p;
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
                for (uint32_t w = 0; w < kQ4Warps; ++w) m = fmaxf(m, wmax[w * kQ4Heads + g + 8 * r]);
                if (m == NEG_INF) m = 0.f;  // only NaN scores so far: they are to stay NaN
                const float alpha = exp2f(M[r] - m);
                M[r] = m;
                l[r] *= alpha;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
#pragma unroll
                    for (int n = 0; n < 8; ++n) {
                        o[j][n][2 * r] *= alpha;
                        o[j][n][2 * r + 1] *= alpha;
                    }
                    ones[j][2 * r] *= alpha;
                    ones[j][2 * r + 1] *= alpha;
                }
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
            float2 p[2][2];                       // [row half r][token half]
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    p[r][e] = *reinterpret_cast<const float2*>(pbuf + (g + 8 * r) * kQ4SRow + tk + 8 * e);
            uint32_t sw4[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                sw4[e] = *reinterpret_cast<const uint32_t*>(sc + (tk + (e & 1) + 8 * (e >> 1)) * 16 + 4 * warp);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float f[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) f[e] = j ? bf16_hi(sw4[e]) : bf16_lo(sw4[e]);
                const uint32_t pa[4] = {cvt_f16x2(p[0][0].x * f[0], p[0][0].y * f[1]),
                                        cvt_f16x2(p[1][0].x * f[0], p[1][0].y * f[1]),
                                        cvt_f16x2(p[0][1].x * f[2], p[0][1].y * f[3]),
                                        cvt_f16x2(p[1][1].x * f[2], p[1][1].y * f[3])};
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t row = tk + (e & 1) + 8 * (e >> 1);
                    const uint32_t chunk = (4 * warp + 2 * j + (g >> 2)) ^ q4_swz(row);
                    w[e] = *reinterpret_cast<const uint32_t*>(st + row * kQ4CodeBytes + chunk * 16 + (g & 3) * 4);
                }
#pragma unroll
                for (int half = 0; half < 2; ++half) {  // nibbles 0-3 and 4-7
                    uint32_t x0, x1;
                    x0 = __byte_perm(w[0], w[1], half ? 0x7632 : 0x5410);
                    x1 = __byte_perm(w[2], w[3], half ? 0x7632 : 0x5410);
                    mma16816_f16(o[j][4 * half], pa, x0 & 0x000f000fu, x1 & 0x000f000fu);
                    mma16816_f16(o[j][4 * half + 1], pa, x0 & 0x00f000f0u, x1 & 0x00f000f0u);
                    x0 >>= 8;
                    x1 >>= 8;
                    mma16816_f16(o[j][4 * half + 2], pa, x0 & 0x000f000fu, x1 & 0x000f000fu);
                    mma16816_f16(o[j][4 * half + 3], pa, x0 & 0x00f000f0u, x1 & 0x00f000f0u);
                }
                mma16816_f16(ones[j], pa, 0x3c003c00u, 0x3c003c00u);
            }
        }
    }
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
    // column of accumulator (j, n), element e: 128w + 64j + 8(2t + e) + n
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float v[8];
#pragma unroll
                for (int n = 0; n < 8; ++n)
                    v[n] = fmaf(o[j][n][2 * r + e], (n & 1) ? 1048576.0f : 16777216.0f, -8.0f * ones[j][2 * r]);
                float* dst = out + (g + 8 * r) * kQ4PartialFloats + 2 + 128 * warp + 64 * j + 8 * (2 * t + e);
#pragma unroll
                for (int n = 0; n < 8; n += 2) *reinterpret_cast<float2*>(dst + n) = make_float2(v[n], v[n + 1]);
            }
}

// Splits of the longest cache so that batch x head blocks x splits fill at
// most one wave of the two CTAs an SM runs, each at least one tile.
void mla_q4_plan_splits(uint32_t batch, uint32_t heads, const uint32_t* lens, int num_sms, uint32_t& split_tokens,
                        uint32_t& splits) {
    uint32_t lmax = 1;
    for (uint32_t b = 0; b < batch; ++b) lmax = lens[b] > lmax ? lens[b] : lmax;
    uint32_t want = kMlaCtasPerSm * static_cast<uint32_t>(num_sms) / (batch * (heads / kQ4Heads));
    if (want < 1) want = 1;
    uint32_t st = static_cast<uint32_t>((static_cast<uint64_t>(lmax) + want - 1) / want);
    if (st < kQ4Tile) st = kQ4Tile;
    split_tokens = st;
    splits = static_cast<uint32_t>((static_cast<uint64_t>(lmax) + st - 1) / st);
}

cudaError_t mla_q4_decode_launch(const MlaLaunch& a, const MlaQ4Seqs& seqs, uint32_t heads, cudaStream_t s) {
    cudaError_t e = mla_absorb_launch(a, heads, s);
    if (e != cudaSuccess) return e;
    if ((e = cudaFuncSetAttribute(mla_q4_attn_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  static_cast<int>(kQ4Smem))) != cudaSuccess)
        return e;
    if ((e = launch_pdl_kernel(mla_q4_attn_kernel, dim3(a.splits, a.batch, heads / kQ4Heads), dim3(kQ4Threads), kQ4Smem,
                               s, a.qp, seqs, heads, a.split_tokens, a.splits, a.partial)) != cudaSuccess)
        return e;
    return mla_merge_out_launch(a, heads, s);
}

}  // namespace pbmoe
