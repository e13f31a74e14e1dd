// Attention of many query rows over one run of tokens of the quantised cache: the prefix that the
// sequences of a batch share.  One decode step reads it once for all of them.
//
// For a kv-head the batch has M = B * group query rows, so the scores are a matrix product Q K^T with
// M rows and so are the outputs P V; K and V are decoded once per workgroup and used by all of its
// rows.  Against the step, whose wave has 4 or 8 rows, a tile's decoding is spread over 128 (64) rows
// and every operand is a plain f16 tile.
//
//   S^T[token][row] = sum_d c[token][d] q[row][d]       v_mfma_f32_32x32x16_f16, A = c, B = q
//   O^T[dim][row]  += sum_t V^T[dim][t] P^T[t][row]     the same, A = V's codes less the middle one, B = P x V's scale
//
// With the rows in the columns a lane (c, h) = (lane % 32, lane / 32) has one row's scores (tokens 8 (i / 4) +
// 4 h + i % 4 of its 32): the running maximum and the sum are its own values, the accumulators are
// rescaled by its own factor, and P's registers are the B operand as they stand: k-slot (h, j) of a
// 16-token product is token 8 (j / 4) + 4 h + j % 4, and V^T is laid out in LDS in that order.
//
// A workgroup of WR * WT waves takes WR * 32 rows and tiles of WT * 32 tokens, each wave 32 rows x 32
// tokens of a tile; waves with the same rows join in LDS at the end.  WR = 4, WT = 2: eight waves, one
// workgroup per CU; WR = 2, WT = 1, for up to 64 rows: two waves, four workgroups per CU.  A thread
// decodes 32 elements of K (a quarter of a token) and / or of V (8 dims of 4 tokens) per tile, from
// registers loaded one tile ahead, into one of two LDS tiles (WT = 1: the only one).
//
// What bounds it: the matrix cores at the rate that they keep up under load, and what runs beside them.
// 64 sequences of 4 heads a kv-head, 8 kv-heads, 32768 shared tokens (AoS): 96 to 100 us.  A 64-token tile is 64
// products per SIMD; on zeros one takes 16 ns (2.1 PFLOP/s), on random operands read from LDS with four fma
// beside it 25 ns (1.3 PFLOP/s: the card slows down with the bits that change), so 1.6 us of the 2.5 per tile.
// Leaving out K's decoding saves 24 us, K's scores 24, V's decoding 11, the loads 13: none of them hides
// another.  Orders that hide latencies better change little: every wave on its own 100 us, two workgroups of
// four waves per CU 96, all products of a tile in one stretch with the exponentials between them 88 (but 1 to 4 %
// slower whole calls at 2048 to 8192 tokens).  Start and end cost 11 to 15 us (8192 tokens: 35 us; one tile per
// workgroup: 13): the chain pages, K, decoding, first product, and part rows of 516 bytes (17 MB at 16 splits).
//
// Precision: the centroids and q (times the score scale) are f16 hi + lo, three products c_hi q_hi +
// c_lo q_hi + c_hi q_lo, and the norm multiplies the fp32 score, so scores and the log-sum-exp keep 2^-21
// as the step's do; FP8 keys and 16-bit queries are exact in f16, one product.  (With single f16
// operands the log-sum-exp was off by 1 to 3e-5: a centroid's rounding is the same for every token that
// has it.)  V's codes are exact, p times a token's V scale is the operand, and the sum of p times V's value at the middle
// code is the row's own in fp32.  For bf16 outputs the operand is one f16 (half a step, 2^-11, of the distance from the middle:
// with the codes themselves it would be of twice as much), for fp16 outputs hi + lo (PLO).  Relative errors of 64 x 8192
// tokens in bf16 1.675e-3 where rounding the output alone makes 1.662e-3 (hi + lo: a quarter more matrix products), of 100 x 4000 in
// fp16 2.074e-4, as rounding alone.  (V itself as f16, code * scale + zero: 1.683e-3 and 2.65e-4, infinite past 65504,
// and 0.5 to 1.5 us faster: 65.9 : 67.4 us the whole call for the first, 61.1 : 61.8 for the second.)
#pragma once
#include "prefix_tiles.h"
#include "step.h"

namespace tq4 {
namespace prefix {

using xdl::half8;
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x3a2 __attribute__((ext_vector_type(3), aligned(2)));
typedef uint32_t u32a1 __attribute__((aligned(1)));
typedef uint32_t u32a2 __attribute__((aligned(2)));

// LDS tiles.  K (hi, and lo): token t's 128 dims at kKRow t.  V^T: dim d = 8 e + i in row 16 i + e, the row's
// 16-byte chunk 2 T + h = tokens 16 T + 8 (j / 4) + 4 h + j % 4, j = 0 .. 7.  Rows are 16 bytes longer than their
// contents, so that 16 consecutive ones, which are read (V: also written) together, start in the 16
// different bank quads, and every access is a thread's one address plus a constant.
constexpr int kKRow = 2 * kHeadDim + 16;
template <int WR, int WT, bool KF8> struct Shape {
    static constexpr int threads = 64 * WR * WT;
    static constexpr int tokens = 32 * WT;          // per tile
    static constexpr int vrow = 2 * tokens + 16;
    static constexpr int klo = tokens * kKRow;      // bytes: K hi at 0, K lo, V^T
    static constexpr int v = klo * (KF8 ? 1 : 2);
    static constexpr int tile = v + kHeadDim * vrow;
    static constexpr int bufs = Buffers<WT>::tiles;
    static constexpr int join = WT == 2 ? WR * 64 * 67 * 4 : 0;  // the waves' sums at the end
    static constexpr int bytes = bufs * tile > join ? bufs * tile : join;
    static constexpr bool halves = threads > 4 * tokens;         // threads decode K or V, else both
    static constexpr int k_waves = halves ? WR * WT / 2 : WR * WT;  // that decode K
    static_assert(threads == 4 * tokens * (halves ? 2 : 1), "a unit of 32 elements per thread");
};

// What the softmax takes of a tile's tokens: the score factor (not with FP8 keys), V's scale and V's value at the
// middle code; and, from each wave that decodes K, whether one of its scales is above xdl::kLargeScale.
template <bool V3> constexpr float kMiddle = V3 ? 4.f : 8.f;
template <int TOKENS, int K_WAVES, bool KF8> struct alignas(16) Factors {
    float norm[KF8 ? 4 : TOKENS];
    float2 v[TOKENS];
    uint32_t large[K_WAVES];
};

struct Args {
    const void *query;       // fp32 rows, already rotated; FP8 keys: q_dtype rows
    const float *centroids;  // [16], 3-bit keys [8], FP8 keys null
    const uint8_t *cache;
    const int32_t *pages;    // block table [batch, table_width]
    const int32_t *seq_lens;
    float *parts;            // part rows (stage2.h)
    int64_t block_stride;
    float score_scale_log2;
    int q_dtype, num_q_heads, num_kv_heads, group, rows;  // rows: batch * group, per kv-head
    int total_rows, batch, table_width;  // total_rows: batch * num_q_heads
    int row_tiles, splits;   // splits: part rows per (sequence, head)
    int tokens, tiles;       // of the prefix (tiles of Shape::tokens)
    int block_size_log2, slot_pos, slot_head;
};

__device__ __forceinline__ floatx16 mfma32(half8 a, half8 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ half2v as_half2(uint32_t x) { return __builtin_bit_cast(half2v, x); }
__device__ __forceinline__ uint32_t as_u32(half2v x) { return __builtin_bit_cast(uint32_t, x); }
__device__ __forceinline__ half2v splat(_Float16 x) { return half2v{x, x}; }

// What a thread loads of a tile, unit u: K bytes of token u / 4 (dims 32 (u % 4) ..) and one of its scalars (u % 4:
// norm, V's scale, V's zero; FP8 keys: no norm); V bytes of tokens 4 (u / 16) .. +3 (dims 8 (u % 16) ..), four of each.
struct RawK {
    uint4 k, k2;           // (k2: FP8 keys)
    uint32_t scalar;
};

// Token `t` of a kv-head in block `blk`.
template <int LAYOUT, bool KF8, bool KB3, bool V3> struct Record {
    static constexpr int rec = xdl::record_bytes<LAYOUT, KF8, KB3, V3>(), v0 = xdl::v_offset<LAYOUT, KF8, KB3>();
    static constexpr int kbytes = KF8 ? kHeadDim : KB3 ? xdl::kK3Bytes : kHalfD, vbytes = V3 ? xdl::kK3Bytes : kHalfD;
    static constexpr int nf = KF8 ? 2 : 3;
    const uint8_t *data;
    const uint16_t *meta;  // SoA: field f at meta[f * bs]
    int pos, bs;
    __device__ __forceinline__ Record(const Args &a, int kvh, int t, int blk) {
        bs = 1 << a.block_size_log2;
        const int hk = a.num_kv_heads, off = t & (bs - 1);
        pos = LAYOUT == 0 ? hk * rec : a.slot_pos;
        const uint8_t *b = a.cache + (int64_t)blk * a.block_stride;
        data = b + (int64_t)off * pos + (int64_t)kvh * (LAYOUT == 0 ? rec : a.slot_head);
        meta = reinterpret_cast<const uint16_t *>(b + (int64_t)bs * hk * rec) + (int64_t)kvh * nf * bs + off;
    }
};

template <int LAYOUT, bool KF8, bool KB3, bool V3>
__device__ __forceinline__ void load_k(RawK &r, const Args &a, int kvh, int t, int blk, int u) {
    using R = Record<LAYOUT, KF8, KB3, V3>;
    const R at(a, kvh, t, blk);
    const uint8_t *p = at.data + (u & 3) * (R::kbytes / 4);
    if constexpr (KB3) {
        const u32x3a2 w = *reinterpret_cast<const u32x3a2 *>(p);
        r.k = uint4{w[0], w[1], w[2], 0u};
    } else {
        const u32x4a2 w = *reinterpret_cast<const u32x4a2 *>(p);
        r.k = uint4{w[0], w[1], w[2], w[3]};
        if constexpr (KF8) {
            const u32x4a2 w2 = *reinterpret_cast<const u32x4a2 *>(p + 16);
            r.k2 = uint4{w2[0], w2[1], w2[2], w2[3]};
        }
    }
    const int f = min(u & 3, R::nf - 1), v = KF8 ? f : f - 1;  // (v: -1 norm, 0 scale, 1 zero)
    if constexpr (LAYOUT == 0)
        r.scalar = at.meta[f * at.bs];
    else
        r.scalar = *reinterpret_cast<const uint16_t *>(at.data + (v < 0 ? R::kbytes : R::v0 + R::vbytes + 2 * v));
}
// (t: a multiple of 4, its four tokens in one block)
template <int LAYOUT, bool KF8, bool KB3, bool V3>
__device__ __forceinline__ void load_v(uint4 &r, const Args &a, int kvh, int t, int blk, int u) {
    using R = Record<LAYOUT, KF8, KB3, V3>;
    const R at(a, kvh, t, blk);
    const uint8_t *p = at.data + R::v0 + (V3 ? 3 : 4) * (u & 15);
    auto token = [&](int i) { return *reinterpret_cast<const u32a1 *>(p + (int64_t)i * at.pos); };
    r = uint4{token(0), token(1), token(2), token(3)};  // (3-bit values: the fourth byte is the next field's first)
}

// The unit's K elements into the LDS tile(s) and, from the token's first thread, the token's factors; `wave`: the
// wave's number among those that decode K.
// 4-bit keys: a byte's pair of centroids, hi and lo parts, from a 256-entry table; 3-bit: six bits' from 64.
template <int LAYOUT, bool KF8, bool KB3, bool V3, class F>
__device__ __forceinline__ void store_k(const RawK &r, unsigned char *khi, unsigned char *klo, F &factors,
                                        const uint2 *lut, int u, int wave) {
    const int t = u >> 2, j = u & 3, at = t * kKRow + 64 * j;
    const float own = half_bits_to_float(r.scalar);
    uint32_t e[16], lo[16];
    if constexpr (KF8) {
        const uint32_t w[8] = {r.k.x, r.k.y, r.k.z, r.k.w, r.k2.x, r.k2.y, r.k2.z, r.k2.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const auto x = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false);
            const auto y = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
            e[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x[0], x[1]));  // (exact)
            e[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(y[0], y[1]));
        }
    } else {
        const uint32_t w[4] = {r.k.x, r.k.y, r.k.z, r.k.w};
#pragma unroll
        for (int b = 0; b < 16; ++b) {
            uint32_t v;
            if constexpr (KB3) {
                const int bit = 6 * b, wi = bit >> 5, sh = bit & 31;
                v = w[wi] >> sh;
                if (sh > 26)
                    v |= w[wi + 1] << (32 - sh);
                v &= 63u;
            } else {
                v = (w[b >> 2] >> (8 * (b & 3))) & 0xFFu;
            }
            const uint2 c = lut[v];
            e[b] = c.x;
            lo[b] = c.y;
        }
        float n = own;
        if constexpr (LAYOUT == 1) {  // the raw norm over the norm of the decoded direction (h.h + 2 h.l: see lookup_tile)
            float hh = 0.f, hl = 0.f;
#pragma unroll
            for (int b = 0; b < 16; ++b) {
                const auto h = __builtin_bit_cast(__fp16 __attribute__((ext_vector_type(2))), e[b]);
                const auto l = __builtin_bit_cast(__fp16 __attribute__((ext_vector_type(2))), lo[b]);
                hh = __builtin_amdgcn_fdot2(h, h, hh, false);
                hl = __builtin_amdgcn_fdot2(h, l, hl, false);
            }
            float csq = fmaf(2.f, hl, hh);
            csq += xdl::dppf<0xB1>(csq);  // quad_perm [1, 0, 3, 2]: the token's four threads
            csq += xdl::dppf<0x4E>(csq);  // quad_perm [2, 3, 0, 1]
            n *= __builtin_amdgcn_rsqf(csq + 1e-16f);
        }
        if (j == 0)
            factors.norm[t] = n;
#pragma unroll
        for (int q = 0; q < 4; ++q)
            *reinterpret_cast<uint4 *>(klo + at + 16 * q) = uint4{lo[4 * q], lo[4 * q + 1], lo[4 * q + 2], lo[4 * q + 3]};
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
        *reinterpret_cast<uint4 *>(khi + at + 16 * q) = uint4{e[4 * q], e[4 * q + 1], e[4 * q + 2], e[4 * q + 3]};
    const float scale = xdl::quad_bcast<KF8 ? 0 : 1>(own);
    if (j == (KF8 ? 1 : 2))
        factors.v[t] = float2{scale, fmaf(scale, kMiddle<V3>, own)};
    const bool large = __any(fabsf(scale) > xdl::kLargeScale);
    if ((u & 63) == 0)
        factors.large[wave] = large;
}

// The unit's V codes (8 dims of 4 tokens) less the middle one, transposed into the LDS tile: for dim i the f16
// pairs of tokens (0, 1) and (2, 3).  A code is put into the significand of 1024 and 1024 + the middle taken off.
template <bool V3, int VROW> __device__ __forceinline__ void store_v(const uint4 &r, unsigned char *vtile, int u) {
    const int dg = u & 15, quad = u >> 4;
    const uint32_t v[4] = {r.x, r.y, r.z, r.w};
    const half2v k0 = splat((_Float16)(1024.f + kMiddle<V3>));
    auto value = [&](uint32_t codes) { return as_u32(as_half2(codes | 0x64006400u) - k0); };
    unsigned char *to = vtile + dg * VROW + 16 * (2 * (quad >> 2) + (quad & 1)) + 8 * ((quad >> 1) & 1);
    auto put = [&](int i, uint32_t c01, uint32_t c23) {
        *reinterpret_cast<uint2 *>(to + 16 * i * VROW) = uint2{value(c01), value(c23)};
    };
    if constexpr (V3) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            auto code = [&](int t) { return (v[t] >> (3 * i)) & 7u; };
            put(i, code(0) | (code(1) << 16), code(2) | (code(3) << 16));
        }
    } else {
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const uint32_t sel = (uint32_t)m | 0x0C00u | ((uint32_t)(4 + m) << 16) | 0x0C000000u;
            const uint32_t p01 = __builtin_amdgcn_perm(v[1], v[0], sel), p23 = __builtin_amdgcn_perm(v[3], v[2], sel);
            put(2 * m, p01 & 0x000F000Fu, p23 & 0x000F000Fu);
            put(2 * m + 1, (p01 >> 4) & 0x000F000Fu, (p23 >> 4) & 0x000F000Fu);
        }
    }
}

// The row's q as B operands (dims 16 i + 8 h .. +7).  FP8 keys: q scaled by the power of two that puts its
// largest magnitude in [0.5, 1), exact for 16-bit queries.  Else q times the score scale, hi + lo parts;
// rows whose largest reaches 2^15 are scaled down into f16's range.  Returns what a product has to be
// multiplied by for scores in log2 units.
template <bool KF8>
__device__ __forceinline__ float load_q(half8 (&hi)[8], half8 (&lo)[8], const Args &a, int64_t head_row, int h) {
    float x[8][8];
    if (KF8 && a.q_dtype != kOutF32) {
        const uint16_t *q = static_cast<const uint16_t *>(a.query) + head_row * kHeadDim + 8 * h;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint4 w = *reinterpret_cast<const uint4 *>(q + 16 * i);
            const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t b = (ww[j >> 1] >> (16 * (j & 1))) & 0xFFFFu;
                x[i][j] = a.q_dtype == kOutBf16 ? __builtin_bit_cast(float, b << 16) : half_bits_to_float(b);
            }
        }
    } else {
        const float *q = static_cast<const float *>(a.query) + head_row * kHeadDim + 8 * h;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float4 lo = *reinterpret_cast<const float4 *>(q + 16 * i), hi = *reinterpret_cast<const float4 *>(q + 16 * i + 4);
            const float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
            for (int j = 0; j < 8; ++j)
                x[i][j] = v[j];
        }
    }
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j)
            amax = fmaxf(amax, fabsf(x[i][j]));
    const auto both = __builtin_amdgcn_permlane32_swap(xdl::fbits(amax), xdl::fbits(amax), false, false);
    const uint32_t b0 = both[0], b1 = both[1];
    amax = fmaxf(xdl::bitsf(b0), xdl::bitsf(b1));
    if constexpr (KF8) {
        const int e = (amax > 0.f && amax < __builtin_inff()) ? -__builtin_amdgcn_frexp_expf(amax) : 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                hi[i][j] = (_Float16)__builtin_ldexpf(x[i][j], e);
        return __builtin_ldexpf(a.score_scale_log2, -e);
    }
    amax *= a.score_scale_log2;
    const int e = (amax >= 32768.f && amax < __builtin_inff()) ? 15 - __builtin_amdgcn_frexp_expf(amax) : 0;
    const float scale = __builtin_ldexpf(a.score_scale_log2, e);
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            // (the product stands in a register: folded into one of the two casts, and rounded once there, hi
            // and lo would not belong together where it is next to a tie of f16)
            float v = x[i][j] * scale;
            asm("" : "+v"(v));
            hi[i][j] = (_Float16)v;
            lo[i][j] = (_Float16)(v - (float)hi[i][j]);
        }
    return __builtin_ldexpf(1.f, -e);
}

// (no NaN-quieting copies of the operands, as fmaxf makes; a NaN operand is passed over)
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
__device__ __forceinline__ half8 pinned(half8 x) {
    xdl::u32x4 t = __builtin_bit_cast(xdl::u32x4, x);
    asm volatile("" : "+v"(t));
    return __builtin_bit_cast(half8, t);
}
// The first sequence of at least `tokens` tokens, -1: none.  (Wave-uniform.)
__device__ __forceinline__ int first_as_long(const int32_t *seq_lens, int batch, int tokens, int lane) {
    for (int b0 = 0; b0 < batch; b0 += 64) {
        const uint64_t has = __ballot(b0 + lane < batch && seq_lens[min(b0 + lane, batch - 1)] >= tokens);
        if (has)
            return b0 + __builtin_ctzll(has);
    }
    return -1;
}
// Rows of a lane pair (c, c + 32): max and sum over both.
__device__ __forceinline__ float pair_max(float x) { return xdl::max_xor32(x); }
__device__ __forceinline__ float pair_sum(float x) { return xdl::sum_xor32(x); }

template <int LAYOUT, bool KF8, bool KB3, bool V3, int WR, int WT, bool PLO>
__global__ __launch_bounds__(64 * WR * WT) __attribute__((amdgpu_waves_per_eu(2, 2)))
void prefix_kernel(const Args a) {
    using S = Shape<WR, WT, KF8>;
    using B = Buffers<WT>;
    __shared__ __align__(16) unsigned char mem[S::bytes];
    __shared__ __align__(16) Factors<S::tokens, S::k_waves, KF8> factors[B::factors];
    __shared__ __align__(16) uint2 lut[KF8 ? 1 : KB3 ? 64 : 256];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 31, h = lane >> 5, wr = w % WR, wt = w / WR;
    // Row tiles of one (kv-head, split) read the same tokens: the list of all workgroups, row tiles
    // first, is cut into eight runs, one per XCD (workgroup i runs on XCD i % 8).
    const int per = gridDim.x >> 3, item = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    const int gi = item / a.row_tiles, rt = item - gi * a.row_tiles;
    if (gi >= a.num_kv_heads * a.splits)
        return;
    const int kvh = gi % a.num_kv_heads, sp = gi / a.num_kv_heads;
    const int tile0 = (int)((int64_t)a.tiles * sp / a.splits), tile1 = (int)((int64_t)a.tiles * (sp + 1) / a.splits);

    // this thread's unit of a tile; its tokens are kept inside the prefix (whole blocks: a multiple of 16)
    // (worked out again in every tile: what depends on it alone would be kept from tile to tile, and spill)
    auto unit = [&] {
        int u = tid & (4 * S::tokens - 1);
        asm volatile("" : "+v"(u));
        return u;
    };
    const bool does_k = !S::halves || w < WR * WT / 2, does_v = !S::halves || w >= WR * WT / 2;
    auto k_tok = [&](int i, int u) { return min(S::tokens * i + (u >> 2), a.tokens - 1); };
    auto v_tok = [&](int i, int u) { return min(S::tokens * i + 4 * (u >> 4), a.tokens - 4); };
    const int32_t *pages = a.pages;
    // (a thread that decodes one of the two has the same registers for both)
    int blks[2] = {};
    int &kblk = blks[0], &vblk = blks[S::halves ? 0 : 1];
    RawK rk;
    uint4 rv_own;
    uint4 &rv = S::halves ? rk.k : rv_own;
    // tile i of this workgroup's (past either end: the next one inside)
    const int n_tiles = tile1 - tile0;
    auto within = [&](int i) { return tile0 + max(min(i, n_tiles - 1), 0); };
    auto read_pages = [&](int i) {
        const int u = unit();
        if (does_k)
            kblk = pages[k_tok(within(i), u) >> a.block_size_log2];
        if (does_v)
            vblk = pages[v_tok(within(i - B::behind), u) >> a.block_size_log2];
    };
    auto load = [&](int i) {
        const int u = unit();
        if (does_k)
            load_k<LAYOUT, KF8, KB3, V3>(rk, a, kvh, k_tok(within(i), u), kblk, u);
        if (does_v)
            load_v<LAYOUT, KF8, KB3, V3>(rv, a, kvh, v_tok(within(i - B::behind), u), vblk, u);
    };
    auto store = [&](int i) {
        const int u = unit();
        unsigned char *m = mem + B::tile(i) * S::tile;
        if (does_k)
            store_k<LAYOUT, KF8, KB3, V3>(rk, m, m + S::klo, factors[B::factor(i)], lut, u, w);
        if (does_v)
            store_v<V3, S::vrow>(rv, m + S::v, u);
    };
    read_pages(0);
    if constexpr (!KF8)
        for (int e = tid; e < (KB3 ? 64 : 256); e += S::threads) {
            const uint32_t x = xdl::split_f16(a.centroids[KB3 ? e & 7 : e & 15]), z = xdl::split_f16(a.centroids[KB3 ? e >> 3 : e >> 4]);
            lut[e] = uint2{(x & 0xFFFFu) | (z << 16), (x >> 16) | (z & 0xFFFF0000u)};
        }
    // The shared blocks are named by every sequence that has the prefix, mostly by the first one, whose entries
    // are on their way (in the table whatever they hold); if nobody has it the join reads no row of this kernel.
    if (a.seq_lens[0] < a.tokens) {
        const int b = first_as_long(a.seq_lens, a.batch, a.tokens, lane);
        if (b < 0)
            return;
        pages += (int64_t)b * a.table_width;
        read_pages(0);
    }
    load(0);
    read_pages(1);

    const int row = rt * 32 * WR + 32 * wr + c, row_in = min(row, a.rows - 1);
    const int b = row_in / a.group, hh = row_in - b * a.group;
    const int64_t head_row = (int64_t)b * a.num_q_heads + kvh * a.group + hh;
    half8 q_hi[8], q_lo[8];
    const float f = load_q<KF8>(q_hi, q_lo, a, head_row, h);
    const bool scaled = __any(f != 1.f);

    floatx16 acc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < 16; ++k)
            acc[i][k] = 0.f;
    // -max in log2 units (+FLT_MAX: no token yet), this lane's shares of the sum and of V's middle values
    float negm = __FLT_MAX__, l = 0.f, z = 0.f;

    xdl::lds_barrier();  // the table
    auto fill = [&](int i) {
        store(i);
        load(i + 1);
        read_pages(i + 2);
    };
    const bool late = WT == 2 && w >= WR;
    auto phase_end = [] {
        __builtin_amdgcn_sched_barrier(0);
        xdl::lds_barrier();
        __builtin_amdgcn_sched_barrier(0);
    };
    floatx16 s;
    half8 p[2], p_lo[2];
    const unsigned char *k_from = mem + (32 * wt + c) * kKRow + 16 * h, *v_from = mem + S::v + c * S::vrow + 16 * (4 * wt + h);
    auto scores = [&](int i) {
        const unsigned char *k_hi = k_from + B::tile(i) * S::tile;
#pragma unroll
        for (int k = 0; k < 16; ++k)
            s[k] = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const half8 a_hi = *reinterpret_cast<const half8 *>(k_hi + 32 * k);
            s = mfma32(a_hi, q_hi[k], s);
            if constexpr (!KF8) {
                s = mfma32(*reinterpret_cast<const half8 *>(k_hi + S::klo + 32 * k), q_hi[k], s);
                s = mfma32(a_hi, q_lo[k], s);
            }
        }
    };
    auto outputs = [&](int i) {
        const unsigned char *vt = v_from + B::tile(i) * S::tile;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const half8 v = *reinterpret_cast<const half8 *>(vt + 32 * d * S::vrow + 32 * t);
                acc[d] = mfma32(v, p[t], acc[d]);
                if constexpr (PLO)
                    acc[d] = mfma32(v, p_lo[t], acc[d]);
            }
    };
    auto softmax = [&](int j) {
        const auto &of = factors[B::factor(j)];
        const int tok0 = 32 * wt + 4 * h;  // s[k]: token tok0 + 8 (k / 4) + k % 4 of the tile
        float n[16];
        if constexpr (!KF8) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float4 v = *reinterpret_cast<const float4 *>(of.norm + tok0 + 8 * k);
                n[4 * k] = v.x;
                n[4 * k + 1] = v.y;
                n[4 * k + 2] = v.z;
                n[4 * k + 3] = v.w;
            }
            if (scaled)
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    n[k] *= f;
        } else {
#pragma unroll
            for (int k = 0; k < 16; ++k)
                n[k] = f;
        }
        uint32_t large = 0;
#pragma unroll
        for (int k = 0; k < S::k_waves; ++k)
            large |= of.large[k];
        // V's scales and middles a quarter (four tokens) ahead: there are no registers for all
        float4 v[2][2];
        auto read_v = [&](int q) {
            const float4 *from = reinterpret_cast<const float4 *>(of.v + tok0 + 8 * q);
            v[q & 1][0] = from[0];
            v[q & 1][1] = from[1];
        };
        read_v(0);
        const int first = S::tokens * (tile0 + j);
        if (first + S::tokens > a.tokens) {  // tokens past the prefix (the last tile's)
#pragma unroll
            for (int k = 0; k < 16; ++k)
                if (first + tok0 + 8 * (k >> 2) + (k & 3) >= a.tokens) {
                    s[k] = -INFINITY;
                    n[k] = 1.f;
                }
        }
        // Scores in log2 units; the running maximum moves only when one passes it by more than kRescaleLogX (p
        // stays below 256), with a large scale in the tile whenever one passes it: p times a scale, an f16
        // operand, stays below 2^15, or 65504.  (The three-way maximum reads the multiplications' results, never the matrix
        // core's: its wait states are the compiler's to insert, and it does not see into asm.)
        float mx = -INFINITY;
#pragma unroll
        for (int k = 0; k < 16; k += 2) {
            s[k] = s[k] * n[k];
            s[k + 1] = s[k + 1] * n[k + 1];
            mx = max3(mx, s[k], s[k + 1]);
        }
        const float most = large ? 0.f : xdl::kRescaleLogX;
        if (__any(mx + negm > most)) {
            const float m_row = pair_max(mx);
            const float negm_new = m_row + negm > most ? -m_row : negm;
            const float alpha = __builtin_amdgcn_exp2f(negm_new - negm);  // 0 at the first tile
            negm = negm_new;
            l *= alpha;
            z *= alpha;
#pragma unroll
            for (int d = 0; d < 4; ++d)
                acc[d] *= alpha;
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (q < 3)
                read_v(q + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int k = 4 * q + i;
                const float4 &vv = v[q & 1][i >> 1];
                const float e = __builtin_amdgcn_exp2f(s[k] + negm);
                l += e;
                z = fmaf(e, i & 1 ? vv.w : vv.y, z);
                float x = e * (i & 1 ? vv.z : vv.x);
                if constexpr (PLO)
                    asm("" : "+v"(x));  // (see load_q)
                p[k >> 3][k & 7] = (_Float16)x;
                if constexpr (PLO)
                    p_lo[k >> 3][k & 7] = (_Float16)(x - (float)p[k >> 3][k & 7]);
            }
        }
        // (worked out here: left to itself the compiler moves this into the matrix phase, next to its use)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            p[t] = pinned(p[t]);
            if constexpr (PLO)
                p_lo[t] = pinned(p_lo[t]);
        }
    };
    run_tiles<WT>(n_tiles, late, [] { xdl::lds_barrier(); }, phase_end, fill, scores, softmax, outputs,
                  [](bool up) { up ? __builtin_amdgcn_s_setprio(1) : __builtin_amdgcn_s_setprio(0); });

    l = pair_sum(l);
    z = pair_sum(z);
    if constexpr (WT == 2) {
        // waves wt = 1 leave their sums in LDS, waves wt = 0 join them with theirs
        xdl::lds_barrier();  // the tiles are no longer read
        float *out = reinterpret_cast<float *>(mem) + wr * 64 * 67 + lane;
        if (wt == 1) {
#pragma unroll
            for (int d = 0; d < 4; ++d)
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    out[64 * (16 * d + k)] = acc[d][k];
            out[64 * 64] = negm;
            out[64 * 65] = l;
            out[64 * 66] = z;
        }
        xdl::lds_barrier();
        if (wt == 1)
            return;
        const float negm1 = out[64 * 64], l1 = out[64 * 65];
        // (a half whose tokens all lie past the prefix has l = 0 and -max = FLT_MAX, the other's weight is then 1)
        const float both = fminf(negm, negm1);
        const float w0 = __builtin_amdgcn_exp2f(both - negm), w1 = __builtin_amdgcn_exp2f(both - negm1);
        negm = both;
        l = l * w0 + l1 * w1;
        z = z * w0 + out[64 * 66] * w1;
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int k = 0; k < 16; ++k)
                acc[d][k] = acc[d][k] * w0 + out[64 * (16 * d + k)] * w1;
    }
    if (row >= a.rows)
        return;
    // (no weight at all where every score of the run is -inf: zeros that the join leaves out, as their lse is -inf)
    const float inv = l == 0.f ? 0.f : 1.f / l;
    // accumulator d, register 4 q + i: row 32 d + 8 q + 4 h + i of V^T, dim 8 (8 (q % 2) + 4 h + i) + 2 d + q / 2
    float *o = part_row(a.parts, head_row, a.splits, sp);
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float4 *to = reinterpret_cast<float4 *>(o + 8 * (8 * q + 4 * h + i));
            const int k = 4 * q + i;
            to[0] = float4{(acc[0][k] + z) * inv, (acc[0][8 + k] + z) * inv, (acc[1][k] + z) * inv, (acc[1][8 + k] + z) * inv};
            to[1] = float4{(acc[2][k] + z) * inv, (acc[2][8 + k] + z) * inv, (acc[3][k] + z) * inv, (acc[3][8 + k] + z) * inv};
        }
    if (h == 0)
        part_lse(a.parts, a.total_rows, head_row, a.splits)[sp] = (__builtin_amdgcn_logf(l) - negm) * kLn2;
}

// One wave per (q-head, sequence): the prefix's part rows, of sequences that have as many tokens, and the
// sequence's own (one row when `whole`, else as many as its step left), joined as merge_parts_kernel
// does; a sink logit (fp32 [Hq], may be null) adds to the sum.  Lane: dims 2 lane, 2 lane + 1.  Latency
// (both kinds of rows, the lengths and the counts are asked for at once): 7 us for 256 rows of 32 parts, 8 for 2048 of 16
// (17 MB, 2.2 TB/s).
template <typename OutT>
__global__ __launch_bounds__(kWave) void join_kernel(const float *__restrict__ shared, int n_shared,
                                                     const float *__restrict__ own, int num_splits, int whole,
                                                     const int32_t *__restrict__ seq_lens, int prefix,
                                                     const float *__restrict__ sinks, OutT *__restrict__ out,
                                                     float *__restrict__ lse, int num_q_heads) {
    constexpr int CHUNK = 16;
    // Own rows asked for ahead: tails have few of the num_splits there are places for (16 ahead: 200 sequences of up to 100
    // tokens behind 4096 82.5 us the whole call, 78.2 with four).
    constexpr int kFewParts = 4;
    const int b = blockIdx.y, lane = threadIdx.x;
    const int64_t row = (int64_t)b * num_q_heads + blockIdx.x;
    const int64_t total_rows = (int64_t)gridDim.y * num_q_heads;
    typedef float float2a __attribute__((ext_vector_type(2), aligned(4)));
    struct Chunk {
        float l;
        float2a v[CHUNK];
    };
    auto load = [&](Chunk &k, const float *rows, int slots, int s0, int n) {
        k.l = part_lse(const_cast<float *>(rows), total_rows, row, slots)[s0 + min(lane, n - 1)];
        const float *r = part_row(const_cast<float *>(rows), row, slots, s0) + 2 * lane;
#pragma unroll
        for (int i = 0; i < CHUNK; ++i)
            k.v[i] = *reinterpret_cast<const float2a *>(r + (int64_t)min(i, n - 1) * kHeadDim);
    };
    // the first rows of both go out before the length and the count arrive (all in bounds)
    Chunk ks, ko;
    load(ks, shared, n_shared, 0, min(CHUNK, n_shared));
    load(ko, own, num_splits, 0, min(kFewParts, num_splits));
    const uint32_t mark = __builtin_bit_cast(uint32_t, part_lse(const_cast<float *>(own), total_rows, row, num_splits)[num_splits - 1]);
    const int len = seq_lens[b];
    const bool has_shared = len >= prefix;
    int n_own = !whole && (mark & kPartMark) == kPartMark ? (int)(mark & ~kPartMark) : num_splits;
    n_own = (has_shared ? len - prefix : len) > 0 ? min(n_own, num_splits) : 0;  // no tokens of its own: nothing written

    float mx = -INFINITY, a0 = 0.f, a1 = 0.f, wsum = 0.f;
    auto add = [&](const Chunk &k, int n) {
        const float l = lane < n ? k.l : -INFINITY;
        const float m_new = fmaxf(mx, wave_max(l));
        // (nothing but weights of zero so far: exp(-inf - -inf) would be NaN)
        const float scale = mx == -INFINITY ? 0.f : expf(mx - m_new);
        const float wt = l == -INFINITY ? 0.f : expf(l - m_new);
        a0 *= scale;
        a1 *= scale;
        wsum = wsum * scale + wave_sum(wt);
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) {
            const float wi = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wt), i));
            a0 = fmaf(wi, i < n ? k.v[i][0] : 0.f, a0);
            a1 = fmaf(wi, i < n ? k.v[i][1] : 0.f, a1);
        }
        mx = m_new;
    };
    if (has_shared)
        for (int s0 = 0; s0 < n_shared; s0 += CHUNK) {
            const int n = min(CHUNK, n_shared - s0);
            if (s0 > 0)
                load(ks, shared, n_shared, s0, n);
            add(ks, n);
        }
    for (int s0 = 0, n; s0 < n_own; s0 += n) {
        n = min(s0 == 0 ? kFewParts : CHUNK, n_own - s0);
        if (s0 > 0)
            load(ko, own, num_splits, s0, n);
        add(ko, n);
    }
    if (sinks && len > 0) {
        const float sink = sinks[blockIdx.x], m_new = fmaxf(mx, sink), scale = expf(mx - m_new);
        a0 *= scale;
        a1 *= scale;
        wsum = wsum * scale + expf(sink - m_new);
        mx = m_new;
    }
    const float inv = 1.f / wsum;  // a sequence without tokens: NaN rows and -inf, as the step
    OutT *o = out + row * kHeadDim;
    o[2 * lane] = from_float<OutT>(a0 * inv);
    o[2 * lane + 1] = from_float<OutT>(a1 * inv);
    if (lane == 0)
        lse[row] = mx + logf(wsum);
}

}  // namespace prefix
}  // namespace tq4
