// Attention of many query rows over one run of tokens of the quantised cache: the prefix that the
// sequences of a batch share.  One decode step reads it once for all of them.
//
// For a kv-head the batch has M = B * group query rows, so the scores are a matrix product Q K^T with
// M rows and so are the outputs P V; K and V are decoded once per workgroup and used by all of its
// rows.  Against the step, whose wave has 4 or 8 rows, a tile's decoding is spread over 128 (64) rows
// and every operand is a plain f16 tile.
//
//   S^T[token][row] = sum_d K[token][d] q[row][d]       v_mfma_f32_32x32x16_f16, A = K, B = q
//   O^T[dim][row]  += sum_t V^T[dim][t] P^T[t][row]     the same, A = V^T, B = P
//
// With the rows in the columns a lane (c, h) = (lane % 32, lane / 32) has one row's scores (tokens 8 (i / 4) +
// 4 h + i % 4 of its 32): the running maximum and the sum are its own values, the accumulators are
// rescaled by its own factor, and P's registers are the B operand as they stand: k-slot (h, j) of a
// 16-token product is token 8 (j / 4) + 4 h + j % 4, and V^T is laid out in LDS in that order.
//
// A workgroup of four waves takes WR * 32 rows (WR = 4: each wave the whole tile of 64 tokens for 32
// rows; WR = 2, for up to 64 rows: half of the tile's tokens each, as rows of their own for the merge).
// Per tile a thread decodes 32 elements of K (a quarter of a token) and 32 of V (8 dims of 4 tokens),
// from registers loaded one tile ahead, into one of two LDS tiles; one barrier per tile.
//
// Roundings: K = f16(f16(c) * f16(norm)), V = f16(code * scale + zero) (one fused rounding) and q scaled
// to f16 by a power of two of its row: each is half a step of f16, 2^-12 on average, where the step's
// hi + lo operands keep 2^-22; scores, the softmax's statistics and the sums are fp32, P is rounded to
// nearest f16.  On outputs in 16 bits (the only ones taken) this is below their own rounding.  V beyond
// f16's range (65504) becomes infinite here.
#pragma once
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

constexpr int kThreads = 256;
constexpr int kTile = 64;                       // tokens per LDS tile
constexpr int kTileBytes = 2 * kTile * kHeadDim * 2;  // K and V^T

struct Args {
    const void *query;       // fp32 rows, already rotated; FP8 keys: q_dtype rows
    const float *centroids;  // [16], 3-bit keys [8], FP8 keys null
    const uint8_t *cache;
    const int32_t *pages;    // the prefix's blocks
    float *parts;            // part rows (stage2.h) of n_parts per (sequence, head)
    int64_t block_stride;
    float score_scale_log2;
    int q_dtype, num_q_heads, num_kv_heads, group, rows;  // rows: batch * group, per kv-head
    int total_rows;          // batch * num_q_heads
    int row_tiles, splits, n_parts;
    int tokens, tiles;       // of the prefix
    int block_size_log2, slot_pos, slot_head;
};

__device__ __forceinline__ floatx16 mfma32(half8 a, half8 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ half2v as_half2(uint32_t x) { return __builtin_bit_cast(half2v, x); }
__device__ __forceinline__ uint32_t as_u32(half2v x) { return __builtin_bit_cast(uint32_t, x); }
__device__ __forceinline__ half2v splat(_Float16 x) { return half2v{x, x}; }

// LDS tiles, in 16-byte chunks.  K: token t's row of 16 chunks (8 dims each), chunk k at k ^ (t & 15).
// V^T: dim d's row of 8 chunks, chunk 2 T + h = tokens 16 T + 8 (j / 4) + 4 h + j % 4, j = 0 .. 7, at
// (2 T + h) ^ vswz(d).  The 16 lanes that read (or write) together then touch all 64 banks: K reads and
// writes, V reads; V's 8-byte writes (16 lanes: dims 8 apart) two lanes a bank.
__device__ __forceinline__ int k_at(int t, int chunk) { return t * 16 + (chunk ^ (t & 15)); }
__device__ __forceinline__ int vswz(int d) { return ((d >> 1) ^ (d >> 3)) & 7; }

// What a thread loads of a tile: K bytes of token tid / 4 (dims 32 (tid % 4) ..), V bytes of tokens
// 4 (tid / 16) .. +3 (dims 8 (tid % 16) ..), and their scalars.
template <int LAYOUT, bool KF8, bool KB3> struct Raw {
    uint4 k, k2;           // (k2: FP8 keys)
    uint32_t v[4];
    uint32_t norm;
    uint32_t sz[4];        // SoA: four scales, four zeros; AoS: scale | zero of each token
};

template <int LAYOUT, bool KF8, bool KB3, bool V3>
__device__ __forceinline__ void load_raw(Raw<LAYOUT, KF8, KB3> &r, const Args &a, int kvh, int kt, int kblk, int vt,
                                         int vblk, int tid) {
    constexpr int rec = xdl::record_bytes<LAYOUT, KF8, KB3, V3>(), kv0 = xdl::v_offset<LAYOUT, KF8, KB3>();
    constexpr int kbytes = KF8 ? kHeadDim : KB3 ? xdl::kK3Bytes : kHalfD, vbytes = V3 ? xdl::kK3Bytes : kHalfD;
    const int mask = (1 << a.block_size_log2) - 1, hk = a.num_kv_heads, bs = mask + 1;
    const int pos = LAYOUT == 0 ? hk * rec : a.slot_pos, head = LAYOUT == 0 ? rec : a.slot_head;
    const uint8_t *kb = a.cache + (int64_t)kblk * a.block_stride, *vb = a.cache + (int64_t)vblk * a.block_stride;
    const int ko = kt & mask, vo = vt & mask, j = tid & 3, dg = tid & 15;
    const uint8_t *kp = kb + (int64_t)ko * pos + (int64_t)kvh * head + j * (kbytes / 4);
    if constexpr (KB3) {
        const u32x3a2 w = *reinterpret_cast<const u32x3a2 *>(kp);
        r.k = uint4{w[0], w[1], w[2], 0u};
    } else {
        const u32x4a2 w = *reinterpret_cast<const u32x4a2 *>(kp);
        r.k = uint4{w[0], w[1], w[2], w[3]};
        if constexpr (KF8) {
            const u32x4a2 w2 = *reinterpret_cast<const u32x4a2 *>(kp + 16);
            r.k2 = uint4{w2[0], w2[1], w2[2], w2[3]};
        }
    }
    const uint8_t *vp = vb + (int64_t)vo * pos + (int64_t)kvh * head + kv0 + (V3 ? 3 : 4) * dg;
#pragma unroll
    for (int t = 0; t < 4; ++t)  // (3-bit values: the fourth byte is the next field's first)
        r.v[t] = *reinterpret_cast<const u32a1 *>(vp + (int64_t)t * pos);
    if constexpr (LAYOUT == 0) {
        constexpr int nf = KF8 ? 2 : 3;
        const uint16_t *km = reinterpret_cast<const uint16_t *>(kb + (int64_t)bs * hk * rec) + kvh * nf * bs + ko;
        const uint16_t *vm = reinterpret_cast<const uint16_t *>(vb + (int64_t)bs * hk * rec) + kvh * nf * bs + vo;
        if constexpr (!KF8)
            r.norm = km[0];
        const uint2 s = *reinterpret_cast<const uint2 *>(vm + (nf - 2) * bs), z = *reinterpret_cast<const uint2 *>(vm + (nf - 1) * bs);
        r.sz[0] = s.x;
        r.sz[1] = s.y;
        r.sz[2] = z.x;
        r.sz[3] = z.y;
    } else {
        if constexpr (!KF8)
            r.norm = *reinterpret_cast<const uint16_t *>(kp - j * (kbytes / 4) + kbytes);
#pragma unroll
        for (int t = 0; t < 4; ++t)
            r.sz[t] = *reinterpret_cast<const u32a2 *>(vp - (V3 ? 3 : 4) * dg + (int64_t)t * pos + vbytes);
    }
}

// The thread's 32 K elements into the LDS tile.  4-bit keys: a byte's pair of centroids from a 256-entry
// table; 3-bit: six bits' from 64.
template <int LAYOUT, bool KF8, bool KB3>
__device__ __forceinline__ void store_k(const Raw<LAYOUT, KF8, KB3> &r, uint4 *ktile, const uint32_t *lut, int tid) {
    const int t = tid >> 2, j = tid & 3;
    uint32_t e[16];
    if constexpr (KF8) {
        const uint32_t w[8] = {r.k.x, r.k.y, r.k.z, r.k.w, r.k2.x, r.k2.y, r.k2.z, r.k2.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false);
            const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
            e[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(lo[0], lo[1]));  // (exact)
            e[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(hi[0], hi[1]));
        }
    } else {
        const uint32_t w[4] = {r.k.x, r.k.y, r.k.z, r.k.w};
#pragma unroll
        for (int b = 0; b < 16; ++b) {
            if constexpr (KB3) {
                const int bit = 6 * b, wi = bit >> 5, sh = bit & 31;
                uint32_t v = w[wi] >> sh;
                if (sh > 26)
                    v |= w[wi + 1] << (32 - sh);
                e[b] = lut[v & 63u];
            } else {
                e[b] = lut[(w[b >> 2] >> (8 * (b & 3))) & 0xFFu];
            }
        }
        float n = half_bits_to_float(r.norm);
        if constexpr (LAYOUT == 1) {  // the raw norm over the norm of the decoded direction
            float csq = 0.f;
#pragma unroll
            for (int b = 0; b < 16; ++b) {
                const auto h = __builtin_bit_cast(__fp16 __attribute__((ext_vector_type(2))), e[b]);
                csq = __builtin_amdgcn_fdot2(h, h, csq, false);
            }
            csq += xdl::dppf<0xB1>(csq);  // quad_perm [1, 0, 3, 2]: the token's four threads
            csq += xdl::dppf<0x4E>(csq);  // quad_perm [2, 3, 0, 1]
            n *= __builtin_amdgcn_rsqf(csq + 1e-16f);
        }
        const half2v n2 = splat((_Float16)n);
#pragma unroll
        for (int b = 0; b < 16; ++b)
            e[b] = as_u32(as_half2(e[b]) * n2);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
        ktile[k_at(t, 4 * j + q)] = uint4{e[4 * q], e[4 * q + 1], e[4 * q + 2], e[4 * q + 3]};
}

// The thread's V elements (8 dims of 4 tokens), transposed into the LDS tile: for dim i the f16 pairs of
// tokens (0, 1) and (2, 3).  A code is put into the significand of 1024 and 1024 taken off again.
template <int LAYOUT, bool KF8, bool KB3, bool V3>
__device__ __forceinline__ void store_v(const Raw<LAYOUT, KF8, KB3> &r, uint4 *vtile, int tid) {
    const int dg = tid & 15, quad = tid >> 4;
    half2v s01, s23, z01, z23;
    if constexpr (LAYOUT == 0) {
        s01 = as_half2(r.sz[0]);
        s23 = as_half2(r.sz[1]);
        z01 = as_half2(r.sz[2]);
        z23 = as_half2(r.sz[3]);
    } else {
        s01 = as_half2(__builtin_amdgcn_perm(r.sz[1], r.sz[0], 0x05040100u));
        z01 = as_half2(__builtin_amdgcn_perm(r.sz[1], r.sz[0], 0x07060302u));
        s23 = as_half2(__builtin_amdgcn_perm(r.sz[3], r.sz[2], 0x05040100u));
        z23 = as_half2(__builtin_amdgcn_perm(r.sz[3], r.sz[2], 0x07060302u));
    }
    const half2v k1024 = splat((_Float16)1024.f);
    auto value = [&](uint32_t codes, half2v s, half2v z) {
        const half2v x = as_half2(codes | 0x64006400u) - k1024;
        return as_u32(__builtin_elementwise_fma(x, s, z));
    };
    const int T = quad >> 2, h = quad & 1, half = (quad >> 1) & 1;
    uint2 *vt = reinterpret_cast<uint2 *>(vtile);
    auto put = [&](int i, uint32_t c01, uint32_t c23) {
        const int d = 8 * dg + i;
        vt[(d * 8 + ((2 * T + h) ^ vswz(d))) * 2 + half] = uint2{value(c01, s01, z01), value(c23, s23, z23)};
    };
    if constexpr (V3) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            auto code = [&](int t) { return (r.v[t] >> (3 * i)) & 7u; };
            put(i, code(0) | (code(1) << 16), code(2) | (code(3) << 16));
        }
    } else {
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const uint32_t sel = (uint32_t)m | 0x0C00u | ((uint32_t)(4 + m) << 16) | 0x0C000000u;
            const uint32_t p01 = __builtin_amdgcn_perm(r.v[1], r.v[0], sel), p23 = __builtin_amdgcn_perm(r.v[3], r.v[2], sel);
            put(2 * m, p01 & 0x000F000Fu, p23 & 0x000F000Fu);
            put(2 * m + 1, (p01 >> 4) & 0x000F000Fu, (p23 >> 4) & 0x000F000Fu);
        }
    }
}

// The row's q as B operands (dims 16 i + 8 h .. +7), scaled by the power of two that puts its largest
// magnitude in [0.5, 1); returns what a product has to be multiplied by for scores in log2 units.
template <bool KF8>
__device__ __forceinline__ float load_q(half8 (&bq)[8], const Args &a, int64_t head_row, int h) {
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
    const int e = (amax > 0.f && amax < __builtin_inff()) ? -__builtin_amdgcn_frexp_expf(amax) : 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j)
            bq[i][j] = (_Float16)__builtin_ldexpf(x[i][j], e);
    return __builtin_ldexpf(a.score_scale_log2, -e);
}

// (no NaN-quieting copies of the operands, as fmaxf makes; a NaN operand is passed over)
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
// Rows of a lane pair (c, c + 32): max and sum over both.
__device__ __forceinline__ float pair_max(float x) { return xdl::max_xor32(x); }
__device__ __forceinline__ float pair_sum(float x) { return xdl::sum_xor32(x); }

template <int LAYOUT, bool KF8, bool KB3, bool V3, int WR>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void prefix_kernel(const Args a) {
    constexpr int WT = 4 / WR;        // waves that share the rows and halve the tokens
    constexpr int NH = 2 / WT;        // 32-token halves of a tile per wave
    __shared__ __align__(16) uint4 tile_mem[2][kTileBytes / 16];
    __shared__ __align__(16) uint32_t lut[KF8 ? 4 : KB3 ? 64 : 256];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 31, h = lane >> 5, wr = w % WR, wt = w / WR;
    // Row tiles of one (kv-head, split) read the same tokens: they come one after the other on one XCD
    // (workgroup i runs on XCD i % 8).
    const int y = blockIdx.x >> 3, rt = y % a.row_tiles, gi = (y / a.row_tiles) * 8 + (blockIdx.x & 7);
    if (gi >= a.num_kv_heads * a.splits)
        return;
    const int kvh = gi % a.num_kv_heads, sp = gi / a.num_kv_heads;
    const int tile0 = (int)((int64_t)a.tiles * sp / a.splits), tile1 = (int)((int64_t)a.tiles * (sp + 1) / a.splits);

    // this thread's tokens of a tile, kept inside the prefix (whole blocks: a multiple of 16 tokens)
    auto k_tok = [&](int i) { return min(kTile * i + (tid >> 2), a.tokens - 1); };
    auto v_tok = [&](int i) { return min(kTile * i + 4 * (tid >> 4), a.tokens - 4); };
    auto page = [&](int t) { return a.pages[t >> a.block_size_log2]; };
    Raw<LAYOUT, KF8, KB3> raw;
    int kblk = page(k_tok(tile0)), vblk = page(v_tok(tile0));
    if constexpr (!KF8) {
        if constexpr (KB3) {
            if (tid < 64)
                lut[tid] = as_u32(half2v{(_Float16)a.centroids[tid & 7], (_Float16)a.centroids[tid >> 3]});
        } else {
            lut[tid] = as_u32(half2v{(_Float16)a.centroids[tid & 15], (_Float16)a.centroids[tid >> 4]});
        }
    }
    load_raw<LAYOUT, KF8, KB3, V3>(raw, a, kvh, k_tok(tile0), kblk, v_tok(tile0), vblk, tid);
    const int next = min(tile0 + 1, tile1 - 1);
    kblk = page(k_tok(next));
    vblk = page(v_tok(next));

    const int row = rt * 32 * WR + 32 * wr + c, row_in = min(row, a.rows - 1);
    const int b = row_in / a.group, hh = row_in - b * a.group;
    const int64_t head_row = (int64_t)b * a.num_q_heads + kvh * a.group + hh;
    half8 bq[8];
    const float f = load_q<KF8>(bq, a, head_row, h);

    floatx16 acc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < 16; ++k)
            acc[i][k] = 0.f;
    float negm = __FLT_MAX__, l = 0.f;  // -max in log2 units (+FLT_MAX: no token yet), this lane's share of the sum

    xdl::lds_barrier();  // the table
    store_k<LAYOUT, KF8, KB3>(raw, tile_mem[0], lut, tid);
    store_v<LAYOUT, KF8, KB3, V3>(raw, tile_mem[0] + kTileBytes / 32, tid);
    load_raw<LAYOUT, KF8, KB3, V3>(raw, a, kvh, k_tok(next), kblk, v_tok(next), vblk, tid);
    xdl::lds_barrier();

    for (int i = tile0; i < tile1; ++i) {
        const int n2 = min(i + 2, tile1 - 1);
        kblk = page(k_tok(n2));
        vblk = page(v_tok(n2));
        const half8 *kt = reinterpret_cast<const half8 *>(tile_mem[(i - tile0) & 1]);
        const half8 *vt = kt + kTileBytes / 32;
        floatx16 s[NH];
#pragma unroll
        for (int q = 0; q < NH; ++q) {
            const int t = 32 * (WT == 1 ? q : wt) + c;
#pragma unroll
            for (int k = 0; k < 16; ++k)
                s[q][k] = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k)
                s[q] = mfma32(kt[k_at(t, 2 * k + h)], bq[k], s[q]);
        }
        if (kTile * (i + 1) > a.tokens) {  // tokens past the prefix (the last tile's)
#pragma unroll
            for (int q = 0; q < NH; ++q)
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    if (kTile * i + 32 * (WT == 1 ? q : wt) + 8 * (k >> 2) + 4 * h + (k & 3) >= a.tokens)
                        s[q][k] = -INFINITY;
        }
        // scores less the running maximum, in log2 units; it moves only when a score passes it by more than
        // kRescaleLogX (p stays below 256).  (The three-way maximum reads the fma's results, never the
        // matrix core's: its wait states are the compiler's to insert, and it does not see into asm.)
        float x[NH][16];
        float mx = -INFINITY;
#pragma unroll
        for (int q = 0; q < NH; ++q)
#pragma unroll
            for (int k = 0; k < 16; k += 2) {
                x[q][k] = fmaf(s[q][k], f, negm);
                x[q][k + 1] = fmaf(s[q][k + 1], f, negm);
                mx = max3(mx, x[q][k], x[q][k + 1]);
            }
        if (__any(mx > xdl::kRescaleLogX)) {
            float m_row = -INFINITY;
#pragma unroll
            for (int q = 0; q < NH; ++q)
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    m_row = fmaxf(m_row, s[q][k] * f);
            m_row = pair_max(m_row);
            const float negm_new = m_row + negm > xdl::kRescaleLogX ? -m_row : negm;
            const float alpha = __builtin_amdgcn_exp2f(negm_new - negm);  // 0 at the first tile
            negm = negm_new;
            l *= alpha;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                acc[j] *= alpha;
#pragma unroll
            for (int q = 0; q < NH; ++q)
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    x[q][k] = fmaf(s[q][k], f, negm);
        }
        half8 p[2 * NH];
#pragma unroll
        for (int q = 0; q < NH; ++q)
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                const float e = __builtin_amdgcn_exp2f(x[q][k]);
                l += e;
                p[2 * q + (k >> 3)][k & 7] = (_Float16)e;
            }
#pragma unroll
        for (int u = 0; u < 2 * NH; ++u)
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const int dim = 32 * d + c, T = (WT == 1 ? 0 : 2 * wt) + u;
                acc[d] = mfma32(vt[dim * 8 + ((2 * T + h) ^ vswz(dim))], p[u], acc[d]);
            }
        if (i + 1 < tile1) {
            uint4 *to = tile_mem[(i + 1 - tile0) & 1];
            store_k<LAYOUT, KF8, KB3>(raw, to, lut, tid);
            store_v<LAYOUT, KF8, KB3, V3>(raw, to + kTileBytes / 32, tid);
            load_raw<LAYOUT, KF8, KB3, V3>(raw, a, kvh, k_tok(n2), kblk, v_tok(n2), vblk, tid);
        }
        xdl::lds_barrier();
    }

    l = pair_sum(l);
    if (row >= a.rows)
        return;
    const int part = sp * WT + wt;
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;  // (a wave whose tokens all lie past the prefix: l = 0)
    float *o = part_row(a.parts, head_row, a.n_parts, part);
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int q = 0; q < 4; ++q)
            *reinterpret_cast<float4 *>(o + 32 * d + 8 * q + 4 * h) =
                float4{acc[d][4 * q] * inv, acc[d][4 * q + 1] * inv, acc[d][4 * q + 2] * inv, acc[d][4 * q + 3] * inv};
    if (h == 0)
        part_lse(a.parts, a.total_rows, head_row, a.n_parts)[part] =
            l == 0.f ? -INFINITY : (__builtin_amdgcn_logf(l) - negm) * kLn2;
}

// One wave per (q-head, sequence): the prefix's part rows, of sequences that have as many tokens, and the
// sequence's own (one row when `whole`, else as many as its step left), joined as merge_parts_kernel
// does; a sink logit (fp32 [Hq], may be null) adds to the sum.  Lane: dims 2 lane, 2 lane + 1.
template <typename OutT>
__global__ __launch_bounds__(kWave) void join_kernel(const float *__restrict__ shared, int n_shared,
                                                     const float *__restrict__ own, int num_splits, int whole,
                                                     const int32_t *__restrict__ seq_lens, int prefix,
                                                     const float *__restrict__ sinks, OutT *__restrict__ out,
                                                     float *__restrict__ lse, int num_q_heads) {
    constexpr int CHUNK = 16;
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
    load(ko, own, num_splits, 0, min(CHUNK, num_splits));
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
    for (int s0 = 0; s0 < n_own; s0 += CHUNK) {
        const int n = min(CHUNK, n_own - s0);
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
