// Appending keys and values to the quantised paged cache with the rotary position applied on the way
// (and to the queries), gfx950.
//
// Of a head's 128 dims the first `rot` are rotated in rot / 2 planes: plane f turns by the angle of
// position p in frequency f, whose cosine and sine are table[p][f] and table[p][rot / 2 + f]:
//   (a, b) -> (a cos - b sin, b cos + a sin),
// (a, b) being dims (f, f + rot / 2), or (2 f, 2 f + 1) when planes are adjacent pairs.  With several axes
// every frequency belongs to one, and p is the token's position on it.  K then goes through the writer of
// store.h (norm, rotation, midpoints, norm correction; FP8 keys: the cast) and V as it is.
//
// Against a rotary launch before the writer, K is neither written nor read again, and is not rounded to
// its type on the way.  The bytes are those of the definition in 64 bits: the writer's fp32-grade path
// (f16 hi + lo products) works out every row, and what lies next to a border is worked out again in fp64
// by the whole wave (Exact): y within kNearY of a midpoint (y is off by less: the split operands by
// 2^-22 sum |x R| <= 2.4e-7, the sums by a few 2^-24), and a K scalar whose fp16 rounding changes within
// 2^-19 of it (its sums of at most 32 squares are off by less than 2^-20).  Gaussian keys: one element in 15000
// and one row in 200 (4-bit keys).  FP8 keys are rotated in fp64 throughout and rounded to fp32,
// then to E4M3.  Rows whose squares underflow fp32 (norms below 1e-19) count as zero.  Queries: fp32, rounded once.
//
// Layout: the writer's lane (n, g) holds 32 dims of row n; which 32 is free for the contraction, so it
// takes the chunks (8 dims) of planes 16 g .. 16 g + 15, both members of each: unit u = 2 g, 2 g + 1 of a row is the two
// chunks whose dims are rotated with each other and 8 frequencies (units past rot / 16: 16 dims that are
// not rotated).  A query thread takes one unit of one row.
//
// What bounds it, and what it measured (32 / 8 heads, bf16, 4-bit keys).  32768 tokens: the queries' rows are
// copied through in 99 to 104 us (537 MB, 5.4 TB/s: the card's copy rate), the writer takes 78 to 87 us for 170 MB: a
// chain per tile (positions, then angles and keys, 96 matrix products, codes, V), four waves of a SIMD in turn,
// 16 tiles per SIMD; without the fp64 rows 61, without the angles too 53.  4097 tokens on three axes 36 us: one tile for all
// but one of the 2048 waves, and at most two workgroups of either role on a CU, for the writer's LDS.  64 tokens
// 14.5 us: one workgroup's chain, the rotation matrix staged and split in LDS (8.6 us in the plain writer), positions and angles before it, and the fp64 rows of the
// slowest wave (4 us).  Registers bind the
// large form (128 at four waves per SIMD): V asked for behind the products instead of ahead of the tile took
// 34 spilled registers to 14, a unit's angles one unit at a time 50 to 12 (139 us to 104), one axis known to
// the compiler 104 to 97; two waves per SIMD without spills 139.  A row in fp64 without a loop over its codes'
// centroids, its sums by register moves: 97 to 89.
#pragma once
#include "store.h"

namespace tq4 {
namespace rope {

using store::Chunk;
using store::half8;

constexpr float kNearY = 1e-6f;
constexpr int kQueryRows = 32;  // rows (token, head) of 128 dims that a wave takes at a time
constexpr int kQueryWaves = 4;  // per workgroup of query_kernel
constexpr int kMostAxes = 4;

struct Args {
    const void *query;            // may be null
    void *query_out;              // [tokens, num_q_heads, 128], contiguous
    const void *key, *value;
    int64_t q_stride, k_stride, v_stride;  // elements from token to token
    const int64_t *positions;     // [axes][tokens], axes axis_stride apart
    int64_t axis_stride;
    const void *table;            // [table_rows][rot]: cosines, sines
    const int32_t *slots;
    const float *pit, *midpoints, *centroids;
    uint8_t *cache;
    int64_t block_stride, num_slots;
    uint64_t axis_bit[2];         // bits 0 and 1 of frequency f's axis at bit f
    int axes, table_rows, table_f32, rot, neox;
    int tokens, num_q_heads, num_kv_heads, block_size, slot_pos, slot_head, norm_correction;
    int store_groups;             // workgroups of the writer; the rest rotate queries
};

// ---- Planes -----------------------------------------------------------------------------
// Chunk (of 8 dims) of member m of unit u.
__device__ __forceinline__ int unit_chunk(const Args &a, int u, int m) {
    const int r = a.rot >> 4;  // rotated units
    return u < r ? (a.neox ? u + (m ? r : 0) : 2 * u + m) : 2 * u + m;
}
// (Rotated units first: u >= r is chunks 2 r + 2 (u - r) + m = 2 u + m.)

// A token's positions as they lie in memory (axes past the last: the last one's again, or 0), and checked:
// ok if all are in the table.
struct RawPositions {
    int64_t at[kMostAxes];
};
struct Positions {
    int at[kMostAxes];
    bool ok;
};
template <bool ONE = false> __device__ __forceinline__ void load_positions(RawPositions &p, const Args &a, int tok) {
    p.at[0] = a.positions[tok];
#pragma unroll
    for (int x = 1; x < kMostAxes; ++x)
        p.at[x] = 0;
    if (!ONE && a.axes > 1)
#pragma unroll
        for (int x = 1; x < kMostAxes; ++x)
            p.at[x] = a.positions[min(x, a.axes - 1) * a.axis_stride + tok];
}
__device__ __forceinline__ Positions checked(const RawPositions &p, const Args &a, bool ok) {
    Positions r{{}, ok};
#pragma unroll
    for (int x = 0; x < kMostAxes; ++x) {
        const bool in = (uint64_t)p.at[x] < (uint64_t)(uint32_t)a.table_rows;
        r.at[x] = in ? (int)p.at[x] : 0;
        r.ok = r.ok && in;
    }
    return r;
}
template <class T> __device__ __forceinline__ float table_at(const Args &a, int row, int col) {
    const int64_t i = (int64_t)row * a.rot + col;
    return a.table_f32 ? static_cast<const float *>(a.table)[i] : (float)static_cast<const T *>(a.table)[i];
}
// Eight consecutive entries (col a multiple of 8).
template <class T> __device__ __forceinline__ void table_row8(const Args &a, int row, int col, float (&v)[8]) {
    const int64_t i = (int64_t)row * a.rot + col;
    if (sizeof(T) == 4 || a.table_f32) {
        const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(a.table) + i);
        const float4 x = p[0], y = p[1];
        v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
    } else {
        typedef T t8 __attribute__((ext_vector_type(8)));
        const t8 x = *reinterpret_cast<const t8 *>(static_cast<const T *>(a.table) + i);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            v[j] = (float)x[j];
    }
}
// Cosines and sines of frequencies 8 u .. 8 u + 7 for a token (u < rot / 16).  pos: its positions.
// ONE: there is one axis.
template <class T, bool ONE = false>
__device__ __forceinline__ void unit_angles(const Args &a, const int (&pos)[kMostAxes], int u, float (&c)[8], float (&s)[8]) {
    if (ONE || a.axes == 1) {
        table_row8<T>(a, pos[0], 8 * u, c);
        table_row8<T>(a, pos[0], a.rot / 2 + 8 * u, s);
        return;
    }
    const uint32_t b0 = (uint32_t)(a.axis_bit[0] >> (8 * u)) & 0xFFu, b1 = (uint32_t)(a.axis_bit[1] >> (8 * u)) & 0xFFu;
#pragma unroll
    for (int x = 0; x < kMostAxes; ++x) {
        const uint32_t mine = (x & 1 ? b0 : ~b0) & (x & 2 ? b1 : ~b1) & 0xFFu;
        if (x >= a.axes || mine == 0)
            continue;
        float cx[8], sx[8];
        table_row8<T>(a, pos[x], 8 * u, cx);
        table_row8<T>(a, pos[x], a.rot / 2 + 8 * u, sx);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            c[j] = (mine >> j) & 1 ? cx[j] : c[j];
            s[j] = (mine >> j) & 1 ? sx[j] : s[j];
        }
    }
}
// A unit's two chunks x0, x1 rotated in place.
template <class F>
__device__ __forceinline__ void turn(float (&x0)[8], float (&x1)[8], const float (&c)[8], const float (&s)[8], bool neox, F plane) {
    if (neox) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            plane(x0[j], x1[j], c[j], s[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            plane(x0[2 * j], x0[2 * j + 1], c[j], s[j]);
            plane(x1[2 * j], x1[2 * j + 1], c[4 + j], s[4 + j]);
        }
    }
}
__device__ __forceinline__ void plane32(float &a, float &b, float c, float s) {
    const float x = fmaf(a, c, -(b * s)), y = fmaf(b, c, a * s);
    a = x;
    b = y;
}
// (a and b cos and sin have at most 48 bits: exact products, one rounding of each sum, one to fp32)
__device__ __forceinline__ void plane64(float &a, float &b, float c, float s) {
    const double x = (double)a * c - (double)b * s, y = (double)b * c + (double)a * s;
    a = (float)x;
    b = (float)y;
}

// 8 elements.
template <class T> struct Eight {
    uint4 u[sizeof(T) / 2];
};
template <class T> __device__ __forceinline__ Eight<T> load8(const T *p) {
    Eight<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i)
        r.u[i] = reinterpret_cast<const uint4 *>(p)[i];
    return r;
}
template <class T> __device__ __forceinline__ void floats8(float (&x)[8], const Eight<T> &r) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
        const uint32_t w[4] = {r.u[i].x, r.u[i].y, r.u[i].z, r.u[i].w};
#pragma unroll
        for (int e = 0; e < 16 / (int)sizeof(T); ++e) {
            if constexpr (sizeof(T) == 4)
                x[4 * i + e] = __builtin_bit_cast(float, w[e]);
            else
                x[e] = (float)__builtin_bit_cast(T, (uint16_t)(w[e / 2] >> (16 * (e % 2))));
        }
    }
}
template <class T> __device__ __forceinline__ void put8(T *p, const float (&x)[8]) {
    typedef T t8 __attribute__((ext_vector_type(8)));
    t8 v;
#pragma unroll
    for (int j = 0; j < 8; ++j)
        v[j] = (T)x[j];
    *reinterpret_cast<t8 *>(p) = v;
}

// ---- Queries ----------------------------------------------------------------------------
// Waves `wave` of `waves` take kQueryRows rows at a time, 8 lanes (one unit each) a row.  A query row
// whose token has a position outside the table becomes NaN.
template <class T> __device__ __forceinline__ void rotate_queries(const Args &a, int wave, int waves, int lane) {
    const int rows = a.tokens * a.num_q_heads, u = lane & 7, r8 = a.rot >> 4;
    const T *query = static_cast<const T *>(a.query);
    T *out = static_cast<T *>(a.query_out);
    const int c0 = 8 * unit_chunk(a, u, 0), c1 = 8 * unit_chunk(a, u, 1);
    constexpr int kSteps = kQueryRows / 8;
    for (int64_t r0 = (int64_t)wave * kQueryRows; r0 < rows; r0 += (int64_t)waves * kQueryRows) {
        Eight<T> x0[kSteps], x1[kSteps];
        RawPositions raw[kSteps];
        int tok[kSteps], row[kSteps];
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            row[i] = (int)min(r0 + 8 * i + (lane >> 3), (int64_t)rows - 1);  // (past the end: the last one again)
            tok[i] = row[i] / a.num_q_heads;
            load_positions(raw[i], a, tok[i]);
            const T *q = query + tok[i] * a.q_stride + (int64_t)(row[i] - tok[i] * a.num_q_heads) * kHeadDim;
            x0[i] = load8(q + c0);
            x1[i] = load8(q + c1);
        }
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const Positions pos = checked(raw[i], a, true);
            float y0[8], y1[8];
            floats8(y0, x0[i]);
            floats8(y1, x1[i]);
            if (u < r8) {
                float c[8], s[8];
                unit_angles<T>(a, pos.at, u, c, s);
                turn(y0, y1, c, s, a.neox != 0, plane32);
            }
            if (!pos.ok)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    y0[j] = y1[j] = __builtin_nanf("");
            // (rows past the end are not written, so that out may be query itself)
            if (r0 + 8 * i + (lane >> 3) < rows) {
                T *o = out + (int64_t)row[i] * kHeadDim;
                put8(o + c0, y0);
                put8(o + c1, y1);
            }
        }
    }
}

// ---- Keys and values --------------------------------------------------------------------
template <class T> struct RawKey {
    Eight<T> c[4];  // member m of unit 2 g + i at c[2 i + m]
};
template <class T> struct Row {
    const T *key, *value;
    int tok, head;
};
template <class T> __device__ __forceinline__ Row<T> row_at(const Args &a, int row, bool in_range) {
    Row<T> r;
    r.tok = in_range ? row / a.num_kv_heads : 0;
    r.head = in_range ? row - r.tok * a.num_kv_heads : 0;
    r.key = static_cast<const T *>(a.key) + r.tok * a.k_stride + r.head * kHeadDim;
    r.value = static_cast<const T *>(a.value) + r.tok * a.v_stride + r.head * kHeadDim;
    return r;
}
// (rows past the end read the first one and are not stored)
template <class T> __device__ __forceinline__ void load_key(RawKey<T> &k, const T *key, const int (&chunk)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        k.c[i] = load8(key + 8 * chunk[i]);
}
// The rotated K of the lane's 32 dims (chunk i at x[8 i ..]).
template <class T, bool ONE, class F>
__device__ __forceinline__ void turned_key(float (&x)[32], const RawKey<T> &k, const Positions &pos, const Args &a, int g, F plane) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float x0[8], x1[8];
        floats8(x0, k.c[2 * i]);
        floats8(x1, k.c[2 * i + 1]);
        if (2 * g + i < a.rot >> 4) {
            float c[8], s[8];
            unit_angles<T, ONE>(a, pos.at, 2 * g + i, c, s);
            turn(x0, x1, c, s, a.neox != 0, plane);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[16 * i + j] = x0[j];
            x[16 * i + 8 + j] = x1[j];
        }
    }
}

// The sum over the wave, in every lane, by register moves (a shuffle goes through LDS and waits for it).
template <int CTRL> __device__ __forceinline__ double dpp64(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, 0xF, 0xF, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, 0xF, 0xF, true);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_sum64(double v) {
    v += dpp64<0xB1>(v);   // quad_perm [1, 0, 3, 2]
    v += dpp64<0x4E>(v);   // quad_perm [2, 3, 0, 1]
    v += dpp64<0x141>(v);  // row_half_mirror
    v += dpp64<0x140>(v);  // row_mirror
    auto pairs = [](double x, auto swap) {  // x of the one half of the lanes plus x of the other
        const uint64_t b = __builtin_bit_cast(uint64_t, x);
        const auto lo = swap((uint32_t)b), hi = swap((uint32_t)(b >> 32));
        const uint32_t l0 = lo[0], l1 = lo[1], h0 = hi[0], h1 = hi[1];
        return __builtin_bit_cast(double, (uint64_t)h0 << 32 | l0) + __builtin_bit_cast(double, (uint64_t)h1 << 32 | l1);
    };
    v = pairs(v, [](uint32_t x) { return __builtin_amdgcn_permlane16_swap(x, x, false, false); });
    return pairs(v, [](uint32_t x) { return __builtin_amdgcn_permlane32_swap(x, x, false, false); });
}
// A row in fp64, worked out by the wave: lane f < rot / 2 has plane f, the others two dims each that are
// not rotated.
template <class T> struct Exact {
    double x0, x1, norm;
    int d0, d1;
    __device__ __forceinline__ Exact(const Args &a, int row, int lane) {
        const Row<T> r = row_at<T>(a, row, true);
        const int half = a.rot / 2;
        const bool turned = lane < half;
        d0 = turned && a.neox ? lane : 2 * lane;  // (not rotated: rot + 2 (lane - half) = 2 lane)
        d1 = turned && a.neox ? lane + half : 2 * lane + 1;
        const double p = (double)(float)r.key[d0], q = (double)(float)r.key[d1];
        x0 = p;
        x1 = q;
        if (turned) {
            const int axis = a.axes == 1 ? 0 : (int)(a.axis_bit[0] >> lane & 1) + 2 * (int)(a.axis_bit[1] >> lane & 1);
            RawPositions raw;
            load_positions(raw, a, r.tok);
            const Positions p4 = checked(raw, a, true);
            const int pos = axis == 0 ? p4.at[0] : axis == 1 ? p4.at[1] : axis == 2 ? p4.at[2] : p4.at[3];
            const double c = table_at<T>(a, pos, lane), s = table_at<T>(a, pos, half + lane);
            x0 = p * c - q * s;
            x1 = q * c + p * s;
        }
        norm = sqrt(wave_sum64(x0 * x0 + x1 * x1));
    }
    __device__ __forceinline__ double y(const float *pit, int dim) const {
        return wave_sum64(x0 * pit[d0 * kHeadDim + dim] + x1 * pit[d1 * kHeadDim + dim]) / (norm + 1e-8);
    }
};

// Code j of packed words.
template <int KB> __device__ __forceinline__ uint32_t code_at(const uint32_t (&w)[KB], int j) {
    uint32_t v = 0;
#pragma unroll
    for (int i = 0; i < KB; ++i) {
        const int sh = KB * j - 32 * i;
        if (sh > -KB && sh < 32)
            v |= sh >= 0 ? w[i] >> sh : w[i] << -sh;
    }
    return v & ((1u << KB) - 1);
}
template <int KB> __device__ __forceinline__ void flip_code(uint32_t (&w)[KB], int j, uint32_t d) {
#pragma unroll
    for (int i = 0; i < KB; ++i) {
        const int sh = KB * j - 32 * i;
        if (sh > -KB && sh < 32)
            w[i] ^= sh >= 0 ? d << sh : d >> -sh;
    }
}

// The writer's tile loop.  W: waves per workgroup (see store_kernel).
template <int LAYOUT, class T, int KB, int VB, int W, bool ONE>
__device__ __forceinline__ void store_rows(const Args &a, int group, int groups) {
    using namespace store;
    __shared__ __align__(16) _Float16 pt_hi[kHeadDim * kHeadDim];
    __shared__ __align__(16) _Float16 pt_lo[kHeadDim * kHeadDim];
    __shared__ float c2tab[16];
    __shared__ __align__(16) float2 btab[kCells];
    constexpr int kMids = (1 << KB) - 1;
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    const int n = lane & 15, g = lane >> 4;
    const int rows = a.tokens * a.num_kv_heads, tiles = (rows + kRows - 1) / kRows, stride = groups * W;
    int tile = group * W + wave;
    Book<KB> book;
    load_book<KB>(book, a.midpoints, a.centroids, a.norm_correction);
    PitLoads<W> pw;
    load_pit<W>(pw, a.pit);
    __builtin_amdgcn_sched_barrier(0);
    int chunk[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        chunk[i] = unit_chunk(a, 2 * g + (i >> 1), i & 1);
    // (a tile's positions and slot are requested with its keys)
    RawKey<T> kr;
    Chunk<T> vr;
    Row<T> at;
    RawPositions raw;
    int slot;
    auto start = [&](int t) {
        at = row_at<T>(a, t * kRows + n, t < tiles && t * kRows + n < rows);
        load_positions<ONE>(raw, a, at.tok);
        slot = a.slots[at.tok];
        load_key<T>(kr, at.key, chunk);
    };
    start(tile);
    __builtin_amdgcn_sched_barrier(0);
    store_pit<W>(pw, pt_hi, pt_lo);
    const Cells cells = build_cells<KB>(book, a.norm_correction, c2tab, btab);

    for (; tile < tiles; tile += stride) {
        const Positions pos = checked(raw, a, tile * kRows + n < rows);
        const bool live = pos.ok && slot >= 0 && slot < a.num_slots;
        float x[32];
        turned_key<T, ONE>(x, kr, pos, a, g, plane32);
        // (four sums: an error of 8 roundings each)
        float s4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 32; ++i)
            s4[i & 3] = fmaf(x[i], x[i], s4[i & 3]);
        const float norm = sqrtf(row_sum((s4[0] + s4[1]) + (s4[2] + s4[3])));
        const float rn = 16.f / (norm + 1e-8f);
        half8 b_hi[4], b_lo[4];
        split_x(x, rn, b_hi, b_lo);
        floatx4 acc[8];
        rotate_tile(acc, b_hi, b_lo, pt_hi, pt_lo, n, [&](int kb) { return chunk[kb]; });
        // (V here: earlier, or 32 registers of it, they spill at four waves per SIMD)
        constexpr bool kEarlyV = sizeof(T) < 4;
        if constexpr (kEarlyV) {
            __builtin_amdgcn_sched_barrier(0);
            load_raw(vr, at.value + 32 * g, true);
        }
        uint32_t kw[KB];
        float csq, nearest = __builtin_inff();
        code_keys<KB, true>(acc, cells, book, btab, c2tab, kw, csq, nearest);
        // elements next to a midpoint (a zero row has y = 0 exactly)
        constexpr float kNear = 256.f * kNearY;
        bool near = live && norm > 0.f && nearest < kNear;
        if (__builtin_expect(__any(near), 0)) {
            uint32_t which = 0;
#pragma unroll
            for (int j = 0; j < 32; ++j) {
                const float v = acc[j / 4][j % 4];
                float d = __builtin_inff();
                if (cells.use)
                    d = fminf(d, fabsf(v - cell_of(v, cells, btab).x));
                else
#pragma unroll
                    for (int i = 0; i < kMids; ++i)
                        d = fminf(d, fabsf(v - 256.f * book.mid[i]));
                which |= d < 2.f * kNear ? 1u << j : 0u;  // (the other path's roundings of the same distance)
            }
            for (uint64_t todo = __ballot(near); todo; todo &= todo - 1) {
                const int l = __builtin_ctzll(todo);
                const Exact<T> r(a, tile * kRows + (l & 15), lane);
                for (uint32_t bits = (uint32_t)__builtin_amdgcn_readlane((int)which, l); bits; bits &= bits - 1) {
                    const int j = __builtin_ctz(bits);
                    const double y = r.y(a.pit, 32 * (l >> 4) + j);
                    uint32_t idx = 0;
#pragma unroll
                    for (int i = 0; i < kMids; ++i)
                        idx += (double)book.mid[i] <= y ? 1u : 0u;
                    const uint32_t old = code_at<KB>(kw, j);
                    if (lane == l && idx != old) {
                        flip_code<KB>(kw, j, idx ^ old);
                        csq += c2tab[idx] - c2tab[old];
                    }
                }
            }
        }
        const float csum = row_sum(csq);
        float kscalar = a.norm_correction ? norm * (1.0f / sqrtf(csum + 1e-16f)) : norm;
        const bool torn = live && half_bits(kscalar * (1.f - 0x1p-19f)) != half_bits(kscalar * (1.f + 0x1p-19f));
        if (__builtin_expect(__any(torn), 0)) {
            const float cent = a.norm_correction ? a.centroids[lane & kMids] : 0.f;
            for (uint32_t todo = (uint32_t)__ballot(torn) & 0xFFFFu; todo; todo &= todo - 1) {
                const int m = __builtin_ctz(todo);
                const Exact<T> r(a, tile * kRows + m, lane);
                double c2 = 0.0;
                if (a.norm_correction) {  // this lane's two of the row's 128 codes
                    uint32_t two = 0;
                    const int bit = 2 * KB * n;
#pragma unroll
                    for (int i = 0; i < KB; ++i) {
                        const uint32_t w = (uint32_t)__shfl((int)kw[i], m + 16 * g, kWave);
                        const int sh = bit - 32 * i;
                        two |= sh >= 0 && sh < 32 ? w >> sh : sh < 0 && sh > -2 * KB ? w << -sh : 0u;
                    }
                    const double c0 = __shfl(cent, (int)(two & kMids), kWave), c1 = __shfl(cent, (int)(two >> KB & kMids), kWave);
                    c2 = wave_sum64(c0 * c0 + c1 * c1);
                }
                const double k = a.norm_correction ? r.norm / sqrt(c2 + 1e-16) : r.norm;
                kscalar = n == m ? (float)k : kscalar;
            }
        }
        if constexpr (!kEarlyV)
            load_raw(vr, at.value + 32 * g, true);
        to_floats(x, vr);
        float scale, vmin;
        uint32_t vw[VB];
        quantize_v<VB>(x, vw, scale, vmin);
        if (live)
            put_record<LAYOUT, KB, VB>(a.cache, slot, at.head, g, kw, vw, kscalar, scale, vmin, a.num_kv_heads, a.block_size,
                                       a.block_stride, a.slot_pos, a.slot_head);
        start(tile + stride);
    }
}

// W = kWaves: large launches, two workgroups per CU, the queries in a launch of their own; kSmallWaves: few
// rows (see store_kernel), the query rows' workgroups behind the writer's in one launch.  ONE: one axis.
template <int LAYOUT, class T, int KB, int VB, int W, bool ONE>
__global__ __launch_bounds__(kWave *W) __attribute__((amdgpu_waves_per_eu(W == store::kWaves ? 4 : 1)))
void append_kernel(const Args a) {
    if (W == store::kWaves || (int)blockIdx.x < a.store_groups)
        store_rows<LAYOUT, T, KB, VB, W, ONE>(a, blockIdx.x, a.store_groups);
    else
        rotate_queries<T>(a, (blockIdx.x - a.store_groups) * W + threadIdx.x / kWave, (gridDim.x - a.store_groups) * W,
                          threadIdx.x % kWave);
}

template <class T> __global__ __launch_bounds__(kWave *kQueryWaves) void query_kernel(const Args a) {
    rotate_queries<T>(a, blockIdx.x * kQueryWaves + threadIdx.x / kWave, gridDim.x * kQueryWaves, threadIdx.x % kWave);
}

// FP8 keys (see store_fp8_kernel).
template <int LAYOUT, class T>
__global__ __launch_bounds__(kWave *store::kFp8Waves) void append_fp8_kernel(const Args a) {
    using namespace store;
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    if ((int)blockIdx.x >= a.store_groups) {
        rotate_queries<T>(a, (blockIdx.x - a.store_groups) * kFp8Waves + wave, (gridDim.x - a.store_groups) * kFp8Waves, lane);
        return;
    }
    const int n = lane & 15, g = lane >> 4;
    const int rows = a.tokens * a.num_kv_heads, tiles = (rows + kRows - 1) / kRows;
    int chunk[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        chunk[i] = unit_chunk(a, 2 * g + (i >> 1), i & 1);
    for (int tile = blockIdx.x * kFp8Waves + wave; tile < tiles; tile += a.store_groups * kFp8Waves) {
        const int row = tile * kRows + n;
        const Row<T> at = row_at<T>(a, row, row < rows);
        RawPositions raw;
        load_positions(raw, a, at.tok);
        const int slot = a.slots[at.tok];
        RawKey<T> kr;
        Chunk<T> vr;
        load_key<T>(kr, at.key, chunk);
        load_raw(vr, at.value + 32 * g, true);
        const Positions pos = checked(raw, a, row < rows);
        float x[32];
        turned_key<T, false>(x, kr, pos, a, g, plane64);
        uint2 kw[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t w[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float *v = x + 8 * i + 4 * h;
                int p = __builtin_amdgcn_cvt_pk_fp8_f32(sat_e4m3(v[0]), sat_e4m3(v[1]), 0, false);
                w[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(sat_e4m3(v[2]), sat_e4m3(v[3]), p, true);
            }
            kw[i] = uint2{w[0], w[1]};
        }
        to_floats(x, vr);
        float scale, vmin;
        uint32_t vw[4];
        quantize_v<4>(x, vw, scale, vmin);
        if (!pos.ok || slot < 0 || slot >= a.num_slots)
            continue;
        const int64_t blk = slot / a.block_size, off = slot % a.block_size;
        uint8_t *base = a.cache + blk * a.block_stride;
        uint32_t *r = reinterpret_cast<uint32_t *>(
            base + (LAYOUT == 0 ? (off * a.num_kv_heads + at.head) * kFp8Record : off * a.slot_pos + (int64_t)at.head * a.slot_head));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            r[2 * chunk[i]] = kw[i].x;
            r[2 * chunk[i] + 1] = kw[i].y;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            r[kHeadDim / 4 + 4 * g + i] = vw[i];
        if (g == 0) {
            uint16_t *f;
            int fstride;
            if constexpr (LAYOUT == 0) {
                f = reinterpret_cast<uint16_t *>(base + (int64_t)a.block_size * a.num_kv_heads * kFp8Record) +
                    (int64_t)at.head * 2 * a.block_size + off;
                fstride = a.block_size;
            } else {
                f = reinterpret_cast<uint16_t *>(reinterpret_cast<uint8_t *>(r) + kFp8Record);
                fstride = 1;
            }
            f[0] = half_bits(scale);
            f[fstride] = half_bits(vmin);
        }
    }
}

}  // namespace rope
}  // namespace tq4
