// Attention of several new tokens per sequence over the paged quantised cache: chunks of prompts, drafted tokens.
//
// For a kv-head a sequence has M = new tokens * group query rows (new tokens first), so scores are a matrix product with
// M rows.  As in the shared prefix (prefix.h) the rows stand in the columns:
//
//   S^T[token][row] = sum_d c[token][d] q[row][d]       v_mfma_f32_32x32x16_f16, A = the keys' codes, B = q
//   O^T[dim][row]  += sum_t V^T[dim][t] P^T[t][row]     the same, A = V, B = the weights
//
// so a lane (c, h) = (lane % 32, lane / 32) has one row's scores (tokens 8 (i / 4) + 4 h + i % 4 of 32): the running
// maximum and sum are its own values, and the weights' registers are the B operand as they stand.
//
// Three launches.  chunk_start_kernel turns the queries into the keys' basis and rounds them to the products' operands;
// its first workgroup cuts the work (chunk_plan.h), the next that of sequences with few rows, which have a product and a join
// of their own (chunk_few.h).  chunk_kernel: a workgroup of WR * WT waves takes its stretch of
// the list of row tiles of 32 WR rows; each wave has 32 rows and 1 / WT of the tokens of a tile of KT, which the
// workgroup decodes once into LDS.  A row tile that one workgroup had whole is written as the result, the parts of one
// that was cut go to the workspace, where chunk_merge_kernel joins them.
//
// Precision.  FINE (fp16 results, or a log-sum-exp): keys' codes and queries are f16 hi + lo, three products, V's codes
// are exact and its scale is part of the weight, one f16.  Otherwise (bf16 results): codes, queries (and the matrix that turns
// them), V and weights are rounded to one f16 each, every one of these an eighth of the result's own rounding.  Weights
// keep that down to 2^-22 of a row's largest one (Headroom).
#pragma once
#include "chunk_plan.h"
#include "prefix.h"

namespace tq4 {
namespace chunk {

using prefix::floatx16;
using prefix::half2v;
using xdl::half8;

struct Args {
    const void *query;       // [tokens, heads, 128] of q_dtype
    const float *rot_t;      // null: FP8 keys
    const float *centroids;
    const uint8_t *cache;
    const int32_t *pages;    // block table [batch, table_width]
    const int32_t *seq_lens, *starts;
    const float *sinks;
    void *out;
    float *lse;              // may be null
    // workspace
    _Float16 *q_hi, *q_lo;   // [tokens * heads, 128]
    float *q_factor;         // [tokens * heads]
    double *work;            // [batch + 1]
    Cut *cuts;               // [groups + 1]
    float *parts;            // [2 groups][rows][128], then [2 groups][rows] log-sum-exps in log2 units
    int64_t block_stride, query_stride;
    float score_scale_log2;
    int q_dtype, out_dtype, num_q_heads, num_kv_heads;
    int tokens, batch, table_width, groups;  // groups: workgroups of the grid
    int block_size_log2, slot_pos, slot_head;
    Shape shape;
    int longest;             // table_width blocks
    int rows_least, rows_most;  // of a kv-head: sequences with fewer or more count as without new tokens
};
__device__ __forceinline__ Seq seq_at(const Args &a, int b) {
    Seq q = seq_of(a.starts, a.seq_lens, b, a.tokens, a.longest);
    const int rows = q.n * a.shape.group;
    if (rows < a.rows_least || rows > a.rows_most)
        q.n = 0;
    return q;
}

// ---- Queries and cuts ------------------------------------------------------------------------

constexpr int kStartWaves = 4, kStartThreads = kWave * kStartWaves, kStartRows = 16 * kStartWaves;

// One workgroup: the work before each sequence, and from it every workgroup's place in the list.  (Batches of up to
// kPlanned sequences are planned in LDS: 64 sequences 8 us in the workspace, 4 so.)
constexpr int kPlanned = 1024;
struct PlanLds {
    double sums[kStartThreads], work[kPlanned + 1];
    Seq seqs[kPlanned];
};
__device__ __forceinline__ void plan_cuts(const Args &a, PlanLds &lds) {
    const int tid = threadIdx.x, per = (a.batch + kStartThreads - 1) / kStartThreads;
    const int b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
    const bool small = a.batch <= kPlanned;
    double *work = small ? lds.work : a.work, *sums = lds.sums;
    double own = 0;
    for (int b = b0; b < b1; ++b) {
        const Seq q = seq_at(a, b);
        if (small)
            lds.seqs[b] = q;
        work[b] = work_of(a.shape, q);
        own += work[b];
    }
    auto seq = [&](int b) { return small ? lds.seqs[b] : seq_at(a, b); };
    // sums over the threads before this one
    double at = own;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const double x = __shfl_up(at, d, kWave);
        at += (tid & (kWave - 1)) >= d ? x : 0.0;
    }
    if ((tid & (kWave - 1)) == kWave - 1)
        sums[tid / kWave] = at;
    __syncthreads();
    double total = 0;
    for (int w = 0; w < kStartWaves; ++w) {
        at += w < tid / kWave ? sums[w] : 0.0;
        total += sums[w];
    }
    at -= own;
    for (int b = b0; b < b1; ++b) {
        const double x = work[b];
        work[b] = at;
        at += x;
    }
    __syncthreads();
    const int used = groups_used(total, a.groups);
    for (int w = tid; w <= a.groups; w += kStartThreads)
        a.cuts[w] = cut_of(a.shape, seq, work, a.batch, total, used, w);
}

// Query rows into operands: y = q @ rot_t (a row scaled by a power of two first; rot_t as f16 hi + lo where LO keeps y as
// pairs too, else rounded to f16, as much of an error as rounding y is), times the score scale, as f16 hi (and lo); rows
// that would pass f16's range, or lie below 2^-8 near its denormals, are scaled to its top and q_factor undoes it.  FP8
// keys: the row itself, scaled by the power of two that puts its largest magnitude in [0.5, 1): exact for dims down to
// 2^-13 of it, below that to 2^-25 of it.
// Bound by each workgroup's own rounding of rot_t: 8192 x 32 rows 39 us (with its low part 53), 134 MB in and out.  A form
// whose workgroups stage rot_t once and take one row tile after the other (32x32x16 products) took 39 with the low part, but
// the whole call was slower by 70 of 710 us: behind its dense matrix phases the device kept a lower clock through
// chunk_kernel (634 : 720 us, the same code).
template <typename InT, bool KF8, bool LO>
__global__ __launch_bounds__(kStartThreads) void chunk_start_kernel(const Args a, const Args few, int plans) {
    constexpr int PT = KF8 ? 8 : kHeadDim * kRotPt;
    __shared__ __align__(16) union {
        _Float16 pt[LO ? 2 : 1][PT];
        PlanLds plan;
    } lds;
    _Float16 *pt_hi = lds.pt[0], *pt_lo = lds.pt[LO];
    if (blockIdx.x == 0) {
        plan_cuts(a, lds.plan);
        return;
    }
    if ((int)blockIdx.x < plans) {
        plan_cuts(few, lds.plan);
        return;
    }
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, n = lane & 15, g = lane >> 4;
    const int64_t rows = (int64_t)a.tokens * a.num_q_heads, r0 = ((int64_t)blockIdx.x - plans) * kStartRows + 16 * wave;
    const int64_t ra = min(r0 + n, rows - 1);
    const int64_t token = ra / a.num_q_heads;
    const InT *from = static_cast<const InT *>(a.query) + token * a.query_stride + (ra - token * a.num_q_heads) * kHeadDim;
    typedef InT in8 __attribute__((ext_vector_type(8)));
    in8 qv[4];
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
        qv[kb] = *reinterpret_cast<const in8 *>(from + 32 * kb + 8 * g);
    float amax = 0.f;
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
        for (int j = 0; j < 8; ++j)
            amax = fmaxf(amax, fabsf(to_float<InT>(qv[kb][j])));
    amax = rot_row_max(amax);
    const bool finite = amax > 0.f && amax < __builtin_inff();
    if constexpr (KF8) {
        const int e = finite ? -__builtin_amdgcn_frexp_expf(amax) : 0;
        if (r0 + n >= rows)
            return;
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
            half8 y;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                y[j] = (_Float16)__builtin_ldexpf(to_float<InT>(qv[kb][j]), e);
            *reinterpret_cast<half8 *>(a.q_hi + ra * kHeadDim + 32 * kb + 8 * g) = y;
        }
        if (g == 0)
            a.q_factor[ra] = __builtin_ldexpf(a.score_scale_log2, -e);
        return;
    } else {
        constexpr int kIters = kHeadDim * (kHeadDim / 8) / kStartThreads;
#pragma unroll
        for (int it = 0; it < kIters; ++it) {
            const int i = threadIdx.x + it * kStartThreads, c = i % kHeadDim, kg = i / kHeadDim;
            half8 h, l;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float w = a.rot_t[(8 * kg + j) * kHeadDim + c];
                h[j] = (_Float16)w;
                if constexpr (LO)
                    l[j] = (_Float16)(w - (float)h[j]);
            }
            *reinterpret_cast<half8 *>(pt_hi + c * kRotPt + 8 * kg) = h;
            if constexpr (LO)
                *reinterpret_cast<half8 *>(pt_lo + c * kRotPt + 8 * kg) = l;
        }
        __syncthreads();
        if (r0 >= rows)
            return;
        const int e = finite ? 15 - __builtin_amdgcn_frexp_expf(amax) : 0;
        half8 q[4];
#pragma unroll
        for (int kb = 0; kb < 4; ++kb)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                q[kb][j] = (_Float16)__builtin_ldexpf(to_float<InT>(qv[kb][j]), e);
        // D: lane (n, g) has dims 16 cb + 4 g .. +3 of row n
        floatx4 y[8];
#pragma unroll
        for (int cb = 0; cb < 8; ++cb) {
            y[cb] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kb = 0; kb < 4; ++kb) {
                const int off = (16 * cb + n) * kRotPt + 32 * kb + 8 * g;
                y[cb] = xdl::mfma(*reinterpret_cast<const half8 *>(pt_hi + off), q[kb], y[cb]);
                if constexpr (LO)
                    y[cb] = xdl::mfma(*reinterpret_cast<const half8 *>(pt_lo + off), q[kb], y[cb]);
            }
        }
        float top = 0.f;
#pragma unroll
        for (int cb = 0; cb < 8; ++cb)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                y[cb][i] = __builtin_ldexpf(y[cb][i], -e) * a.score_scale_log2;
                top = fmaxf(top, fabsf(y[cb][i]));
            }
        top = rot_row_max(top);
        const bool small = top > 0.f && top < 0x1p-8f, large = top >= 32768.f && top < __builtin_inff();
        const int f = small || large ? 15 - __builtin_amdgcn_frexp_expf(top) : 0;
        if (r0 + n >= rows)
            return;
        typedef _Float16 half4 __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int cb = 0; cb < 8; ++cb) {
            half4 hi, lo;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v = __builtin_ldexpf(y[cb][i], f);
                asm("" : "+v"(v));  // (rounded once: hi and lo belong together)
                hi[i] = (_Float16)v;
                lo[i] = (_Float16)(v - (float)hi[i]);
            }
            *reinterpret_cast<half4 *>(a.q_hi + ra * kHeadDim + 16 * cb + 4 * g) = hi;
            if constexpr (LO)
                *reinterpret_cast<half4 *>(a.q_lo + ra * kHeadDim + 16 * cb + 4 * g) = lo;
        }
        if (g == 0)
            a.q_factor[ra] = __builtin_ldexpf(1.f, -f);
    }
}

// ---- Token tiles -----------------------------------------------------------------------------

// LDS tiles as prefix.h's: K (hi, and lo) in rows of a token, V^T in rows of a dim.
constexpr int kKRow = prefix::kKRow;
template <bool V3> constexpr float kMiddle = prefix::kMiddle<V3>;
constexpr float kShrink = 1.f / 32.f;   // 15 codes of the largest f16 scale and the largest zero are below 2^20
constexpr int kAhead = 4;               // operands that are read ahead of their products

template <int WR, int WT, int KT, int BUFS, bool KF8, bool FINE> struct Form {
    static constexpr int threads = 64 * WR * WT;
    static constexpr int vrow = 2 * KT + 16;
    static constexpr int klo = KT * kKRow;  // bytes: K hi at 0, K lo, V^T
    static constexpr int v = klo * (!KF8 && FINE ? 2 : 1);
    static constexpr int tile = v + kHeadDim * vrow;
    static constexpr int join = (WT - 1) * WR * 64 * 67 * 4;
    static constexpr int bytes = BUFS * tile > join ? BUFS * tile : join;
    static constexpr bool halves = threads == 8 * KT;  // threads decode K or V, else both
    static constexpr int units = halves ? 1 : 4 * KT / threads;  // of either that a thread decodes
    static constexpr int sub = KT / (32 * WT);         // products of 32 tokens per wave and tile
    static_assert(halves || (4 * KT) % threads == 0, "whole units");
};
// What the softmax takes of a tile's tokens.  v: V's scale and its value at the middle code (FINE).  special: of each 16
// tokens (those that one wave decodes at a time), whether their `fix` may differ from 1: the weight's factor where V is
// stored smaller, NaN where V is not finite.  top: the bits of their largest finite scale (FINE).
template <int KT, bool KF8, bool FINE> struct alignas(16) Factors {
    float norm[KF8 ? 4 : KT];
    float2 v[FINE ? KT : 2];
    float fix[KT];
    uint32_t special[KT / 16];
    uint32_t top[FINE ? KT / 16 : 4];
};
// The codes' table: pairs of centroids as f16, with their low parts (FINE), or with the sum of their squares (AoS slots,
// which hold the raw norm).  It has LDS address 0, so that a lookup's address is the byte of codes, shifted.
template <bool KF8, bool KB3, bool WIDE> struct Table {
    using Entry = std::conditional_t<WIDE, uint2, uint32_t>;
    static constexpr int entries = KF8 ? 4 : KB3 ? 64 : 256;
};
template <int LAYOUT, bool KF8, bool KB3, bool FINE, class Entry>
__device__ __forceinline__ void fill_table(Entry *table, const float *centroids, int tid, int threads) {
    if constexpr (!KF8)
        for (int e = tid; e < (KB3 ? 64 : 256); e += threads) {
            const float c0 = centroids[KB3 ? e & 7 : e & 15], c1 = centroids[KB3 ? e >> 3 : e >> 4];
            if constexpr (FINE) {
                const uint32_t x = xdl::split_f16(c0), z = xdl::split_f16(c1);
                table[e] = uint2{(x & 0xFFFFu) | (z << 16), (x >> 16) | (z & 0xFFFF0000u)};
            } else {
                const uint32_t both = prefix::as_u32(half2v{(_Float16)c0, (_Float16)c1});
                if constexpr (LAYOUT == 1)
                    table[e] = uint2{both, xdl::fbits(fmaf(c0, c0, c1 * c1))};
                else
                    table[e] = both;
            }
        }
}
// Codes 2 b, 2 b + 1 of a lane's 32.
template <bool KB3> __device__ __forceinline__ uint32_t code_pair(const uint32_t (&w)[4], int b) {
    if constexpr (KB3) {
        const int bit = 6 * b, wi = bit >> 5, sh = bit & 31;
        uint32_t v = w[wi] >> sh;
        if (sh > 26)
            v |= w[wi + 1] << (32 - sh);
        return v & 63u;
    } else {
        return (w[b >> 2] >> (8 * (b & 3))) & 0xFFu;
    }
}

// Unit u of K: token u / 4 of the tile, dims 32 (u % 4) .. +31.  Unit u of V: tokens 16 (u / 64) + 4 q .. +3, dims 8 e .. +7, where
// u % 64 = 16 r + 4 q + j and e = 4 j + r: the lane loads 32 dims of one token (r of the four), and the four lanes with
// the same q and j exchange what they hold.  The 64 units that a wave decodes at a time are those of 16 tokens,
// which lie in one block: where they begin is the wave's, a lane's place in them the same in every tile.
template <int LAYOUT, bool KF8, bool KB3, bool V3> struct Codes {
    static constexpr int rec = xdl::record_bytes<LAYOUT, KF8, KB3, V3>(), v0 = xdl::v_offset<LAYOUT, KF8, KB3>();
    static constexpr int kbytes = KF8 ? kHeadDim : KB3 ? xdl::kK3Bytes : kHalfD, vbytes = V3 ? xdl::kK3Bytes : kHalfD;
    static constexpr int nf = KF8 ? 2 : 3;
};
struct Raw {
    uint4 a, b;  // codes; K: norm (FP8 keys: the codes' second half), V: scales and zeros
};
// The wave's 16 tokens: their records of the kv-head, and (SoA) its scalars, as buffers: a lane's offset in them is the
// same in every tile, so that no address is worked out in vector registers.
struct Place {
    __amdgpu_buffer_rsrc_t data, meta;
};
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_at(const uint8_t *p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(p), 0, 0x7FFFFFFF, 0x00020000);
}
__device__ __forceinline__ uint4 load16(__amdgpu_buffer_rsrc_t b, uint32_t at, int more) {
    return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(b, (int)at, more, 0));
}
__device__ __forceinline__ uint4 load12(__amdgpu_buffer_rsrc_t b, uint32_t at, int more) {
    const auto v = __builtin_amdgcn_raw_buffer_load_b96(b, (int)at, more, 0);
    return uint4{(uint32_t)v[0], (uint32_t)v[1], (uint32_t)v[2], 0u};
}
__device__ __forceinline__ uint2 load8(__amdgpu_buffer_rsrc_t b, uint32_t at, int more) {
    return __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(b, (int)at, more, 0));
}
__device__ __forceinline__ uint32_t load4(__amdgpu_buffer_rsrc_t b, uint32_t at, int more) {
    return (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(b, (int)at, more, 0);
}
__device__ __forceinline__ uint32_t load2(__amdgpu_buffer_rsrc_t b, uint32_t at, int more) {
    return (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(b, (int)at, more, 0);
}
template <int LAYOUT, bool KF8, bool KB3, bool V3>
__device__ __forceinline__ Place place_of(const Args &a, int kvh, int blk, int within) {
    using C = Codes<LAYOUT, KF8, KB3, V3>;
    const uint8_t *b = a.cache + (uint64_t)(uint32_t)blk * (uint32_t)a.block_stride;
    const int bs = 1 << a.block_size_log2;
    const uint8_t *data = b + (uint32_t)(within * a.slot_pos + kvh * a.slot_head);
    const uint8_t *meta = LAYOUT == 0 ? b + (uint32_t)(bs * a.num_kv_heads * C::rec + 2 * (kvh * C::nf * bs + within)) : data;
    return Place{buffer_at(data), buffer_at(meta)};
}
template <int LAYOUT, bool KF8, bool KB3, bool V3>
__device__ __forceinline__ void load_k(Raw &r, const Args &a, const Place &at, int lane) {
    using C = Codes<LAYOUT, KF8, KB3, V3>;
    const uint32_t token = (uint32_t)(lane >> 2) * (uint32_t)a.slot_pos, part = token + (lane & 3) * (C::kbytes / 4);
    r.a = KB3 ? load12(at.data, part, 0) : load16(at.data, part, 0);
    if constexpr (KF8)
        r.b = load16(at.data, part, 16);
    else
        r.b.x = LAYOUT == 0 ? load2(at.meta, 2u * (lane >> 2), 0) : load2(at.data, token, C::kbytes);
}
// (a: the lane's token's codes, 32 dims; b.xy or b.x: scales and zeros, see exchange)
template <int LAYOUT, bool KF8, bool KB3, bool V3>
__device__ __forceinline__ void load_v(Raw &r, const Args &a, const Place &at, int lane) {
    using C = Codes<LAYOUT, KF8, KB3, V3>;
    const int row = lane >> 4, quad = (lane >> 2) & 3, j = lane & 3;
    const uint32_t token = (uint32_t)(4 * quad + row) * (uint32_t)a.slot_pos;
    r.a = V3 ? load12(at.data, token + 12 * j, C::v0) : load16(at.data, token + 16 * j, C::v0);
    if constexpr (LAYOUT == 0) {  // even rows the four tokens' scales, odd rows their zeros
        const uint2 s = load8(at.meta, ((uint32_t)(row & 1) << (a.block_size_log2 + 1)) + 8u * quad, (C::nf - 2) * 2 << a.block_size_log2);
        r.b.x = s.x;
        r.b.y = s.y;
    } else {  // the token's own
        r.b.x = load4(at.data, token, C::v0 + C::vbytes);
    }
}
// Swaps x of the odd rows of 16 lanes with y of the even rows before them; of the upper two rows with the lower two.
__device__ __forceinline__ void swap16(uint32_t &x, uint32_t &y) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, y, false, false);
    const uint32_t a = r[0], b = r[1];
    x = a;
    y = b;
}
__device__ __forceinline__ void swap32(uint32_t &x, uint32_t &y) {
    const auto r = __builtin_amdgcn_permlane32_swap(x, y, false, false);
    const uint32_t a = r[0], b = r[1];
    x = a;
    y = b;
}
// The loaded parts to units: v[t] the eight codes of token t; s, z: scales and zeros of tokens (0, 1) and (2, 3).
template <int LAYOUT, bool V3> __device__ __forceinline__ void exchange(const Raw &r, uint32_t (&v)[4], uint32_t (&s)[2], uint32_t (&z)[2]) {
    v[0] = r.a.x;
    v[1] = r.a.y;
    v[2] = r.a.z;
    v[3] = r.a.w;
    if constexpr (V3) {  // 24 bits each
        const uint32_t w0 = v[0], w1 = v[1], w2 = v[2];
        v[1] = __builtin_amdgcn_alignbit(w1, w0, 24);
        v[2] = __builtin_amdgcn_alignbit(w2, w1, 16);
        v[3] = w2 >> 8;
    }
    // row r has parts 0 .. 3 of token r: to part r of tokens 0 .. 3
    swap32(v[0], v[2]);
    swap32(v[1], v[3]);
    swap16(v[0], v[1]);
    swap16(v[2], v[3]);
    if constexpr (LAYOUT == 0) {
        s[0] = z[0] = r.b.x;
        s[1] = z[1] = r.b.y;
        swap16(s[0], z[0]);
        swap16(s[1], z[1]);
    } else {
        uint32_t t[4] = {r.b.x, r.b.x, r.b.x, r.b.x};
        swap32(t[0], t[2]);
        swap32(t[1], t[3]);
        swap16(t[0], t[1]);
        swap16(t[2], t[3]);
        s[0] = __builtin_amdgcn_perm(t[1], t[0], 0x05040100u);
        s[1] = __builtin_amdgcn_perm(t[3], t[2], 0x05040100u);
        z[0] = __builtin_amdgcn_perm(t[1], t[0], 0x07060302u);
        z[1] = __builtin_amdgcn_perm(t[3], t[2], 0x07060302u);
    }
}

// A unit of K into LDS, in four steps (a quarter of its codes looked up, the quarter before written); the fifth
// writes the last.
template <int LAYOUT, bool KF8, bool KB3, bool FINE> struct KUnit {
    static constexpr bool WIDE = FINE || LAYOUT == 1;
    uint32_t hi[2][4], lo[2][4];
    float sq = 0.f, hl = 0.f;
    __device__ __forceinline__ void look_up(const Raw &r, const typename Table<KF8, KB3, WIDE>::Entry *table, int q) {
        if constexpr (KF8) {
            const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const auto x = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[2 * q + i], false);
                const auto y = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[2 * q + i], true);
                hi[q & 1][2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x[0], x[1]));  // (exact)
                hi[q & 1][2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(y[0], y[1]));
            }
        } else {
            const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t v = code_pair<KB3>(w, 4 * q + i);
                if constexpr (WIDE) {
                    const uint2 c = table[v];
                    hi[q & 1][i] = c.x;
                    lo[q & 1][i] = c.y;
                } else {
                    hi[q & 1][i] = table[v];
                }
            }
        }
    }
    // `at`: the unit's place among K's rows
    __device__ __forceinline__ void write(unsigned char *khi, unsigned char *klo, int at, int q) {
        const uint32_t(&e)[4] = hi[q & 1], (&f)[4] = lo[q & 1];
        *reinterpret_cast<uint4 *>(khi + at + 16 * q) = uint4{e[0], e[1], e[2], e[3]};
        if constexpr (FINE && !KF8)
            *reinterpret_cast<uint4 *>(klo + at + 16 * q) = uint4{f[0], f[1], f[2], f[3]};
        if constexpr (LAYOUT == 1 && !KF8)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (FINE) {  // h.h + 2 h.l
                    const auto h = __builtin_bit_cast(__fp16 __attribute__((ext_vector_type(2))), e[i]);
                    const auto l = __builtin_bit_cast(__fp16 __attribute__((ext_vector_type(2))), f[i]);
                    sq = __builtin_amdgcn_fdot2(h, h, sq, false);
                    hl = __builtin_amdgcn_fdot2(h, l, hl, false);
                } else {
                    sq += xdl::bitsf(f[i]);
                }
            }
    }
    // (every thread of a token writes its norm: the same one)
    template <class F> __device__ __forceinline__ void write_norm(const Raw &r, F &factors, int u) {
        if constexpr (!KF8) {
            float n = half_bits_to_float(r.b.x);
            if constexpr (LAYOUT == 1) {  // the raw norm over the norm of the decoded direction
                sq = fmaf(2.f, hl, sq);
                sq += xdl::dppf<0xB1>(sq);  // quad_perm [1, 0, 3, 2]: the token's four threads
                sq += xdl::dppf<0x4E>(sq);  // quad_perm [2, 3, 0, 1]
                n *= __builtin_amdgcn_rsqf(sq + 1e-16f);
            }
            factors.norm[u >> 2] = n;
        }
    }
};

// Of pairs of f16: the larger magnitudes, as whole numbers (NaN and infinities above all others); of one, the larger.
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t most_of(uint32_t x, uint32_t y) {
    auto mag = [](uint32_t x) { return __builtin_bit_cast(u16x2, x & 0x7FFF7FFFu); };
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(mag(x), mag(y)));
}
__device__ __forceinline__ uint32_t top_of(uint32_t x) {
    const u16x2 v = __builtin_bit_cast(u16x2, x);
    return v[0] > v[1] ? v[0] : v[1];
}

// Dims 2 m and 2 m + 1 of two tokens' eight codes, less `less`, as f16 pairs: the code is put into the significand of 1024, or,
// where it lies four bits up, of 64, whose last place there is a sixteenth; then that is taken off.
template <bool V3>
__device__ __forceinline__ void code_values(uint32_t a, uint32_t b, int m, float less, half2v &even, half2v &odd) {
    if constexpr (V3) {
        auto value = [&](int i) {
            const uint32_t pair = ((a >> (3 * i)) & 7u) | (((b >> (3 * i)) & 7u) << 16);
            return prefix::as_half2(pair | 0x64006400u) - prefix::splat((_Float16)(1024.f + less));
        };
        even = value(2 * m);
        odd = value(2 * m + 1);
    } else {
        uint32_t low = 0x64006400u, high = 0x54005400u;
        asm("" : "+v"(low), "+v"(high));
        const uint32_t p = __builtin_amdgcn_perm(b, a, (uint32_t)m | 0x0C00u | ((uint32_t)(4 + m) << 16) | 0x0C000000u);
        even = prefix::as_half2((p & 0x000F000Fu) | low) - prefix::splat((_Float16)(1024.f + less));
        odd = prefix::as_half2((p & 0x00F000F0u) | high) - prefix::splat((_Float16)(64.f + less));
    }
}

// A unit of V into LDS: begin() takes its scalars, write(m) dims 2 m and 2 m + 1 of it.
template <int LAYOUT, bool V3, bool FINE, int VROW> struct VUnit {
    half2v s01, s23, z01, z23;
    uint32_t v[4];
    // `valid`: tokens of the unit that the sequence has and a row may see (4 or more: all; the others' bytes may hold anything,
    // and count as zeros).  `quad`: of the tile.  (Of a wave, together.)
    template <class F> __device__ __forceinline__ void begin(const Raw &r, F &factors, int quad, bool cut, int valid) {
        uint32_t s[2], z[2];  // scales and zeros of tokens (0, 1) and (2, 3)
        exchange<LAYOUT, V3>(r, v, s, z);
        if (cut) {
            const uint32_t m0 = valid <= 0 ? 0u : valid == 1 ? 0xFFFFu : 0xFFFFFFFFu, m1 = valid <= 2 ? 0u : valid == 3 ? 0xFFFFu : 0xFFFFFFFFu;
            s[0] &= m0;
            s[1] &= m1;
            z[0] &= m0;
            z[1] &= m1;
        }
        // magnitudes as whole numbers: scales of 2048 or zeros of 16384 and more might pass f16's range together; NaN and
        // infinities are above those
        uint32_t top_s = top_of(most_of(s[0], s[1]));
        const uint32_t top_z = top_of(most_of(z[0], z[1]));
        const bool special = __any(top_s >= (FINE ? 0x7C00u : 0x6800u) || top_z >= (FINE ? 0x7C00u : 0x7400u));
        float scale[4], zero[4];
        if (FINE || special)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                scale[i] = half_bits_to_float(s[i >> 1] >> (16 * (i & 1)));
                zero[i] = half_bits_to_float(z[i >> 1] >> (16 * (i & 1)));
            }
        if (special) {
            float fix[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float top = fmaf(15.f, fabsf(scale[i]), fabsf(zero[i]));
                fix[i] = 1.f;
                if (!(top < __builtin_inff())) {
                    fix[i] = __builtin_nanf("");
                    scale[i] = zero[i] = 0.f;
                } else if (!FINE && top > 60000.f) {
                    fix[i] = 1.f / kShrink;
                    scale[i] *= kShrink;
                    zero[i] *= kShrink;
                }
            }
            *reinterpret_cast<float4 *>(factors.fix + 4 * quad) = float4{fix[0], fix[1], fix[2], fix[3]};
            if constexpr (FINE) {
                const float top = fmaxf(fmaxf(fabsf(scale[0]), fabsf(scale[1])), fmaxf(fabsf(scale[2]), fabsf(scale[3])));
                top_s = __builtin_bit_cast(uint16_t, (_Float16)top);
            } else {
                auto pair = [](float x, float y) { return prefix::as_u32(half2v{(_Float16)x, (_Float16)y}); };
                s[0] = pair(scale[0], scale[1]);
                s[1] = pair(scale[2], scale[3]);
                z[0] = pair(zero[0], zero[1]);
                z[1] = pair(zero[2], zero[3]);
            }
        }
        factors.special[quad >> 2] = special;
        if constexpr (FINE) {
            // (the four quads of the wave's tokens: lanes 4 and 8 apart in each 16)
            top_s = max(top_s, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top_s, 0x124, 0xF, 0xF, false));  // row_ror:4
            top_s = max(top_s, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top_s, 0x128, 0xF, 0xF, false));  // row_ror:8
            factors.top[quad >> 2] = top_s;
            float4 *to = reinterpret_cast<float4 *>(factors.v + 4 * quad);
            auto mid = [&](int i) { return fmaf(scale[i], kMiddle<V3>, zero[i]); };
            to[0] = float4{scale[0], mid(0), scale[1], mid(1)};
            to[1] = float4{scale[2], mid(2), scale[3], mid(3)};
        } else {
            s01 = prefix::as_half2(s[0]);
            s23 = prefix::as_half2(s[1]);
            z01 = prefix::as_half2(z[0]);
            z23 = prefix::as_half2(z[1]);
        }
    }
    // codes to f16 (see code_values), FINE: less the middle code
    __device__ __forceinline__ void write(unsigned char *to, int m) {
        auto put = [&](int i, half2v x, half2v y) {
            if constexpr (!FINE) {
                x = __builtin_elementwise_fma(x, s01, z01);
                y = __builtin_elementwise_fma(y, s23, z23);
            }
            *reinterpret_cast<uint2 *>(to + 16 * i * VROW) = uint2{prefix::as_u32(x), prefix::as_u32(y)};
        };
        constexpr float less = FINE ? kMiddle<V3> : 0.f;
        half2v x0, x1, y0, y1;
        code_values<V3>(v[0], v[1], m, less, x0, x1);
        code_values<V3>(v[2], v[3], m, less, y0, y1);
        put(2 * m, x0, y0);
        put(2 * m + 1, x1, y1);
    }
};

// Where the softmax's running maximum lies.  A weight enters the products as one f16, so it is to use that range: with the
// largest one at 1, weights below 2^-14 of it were denormals, and rows that one token dominates (13 nats above 32768 others, its
// value small) off by 1 %.  A move puts the row's largest weight at 2^goal, and the next one waits until the weights of a
// lane's tokens in a tile sum to more than `most`: so weights are at most that, and normal down to 2^(-14 - goal) of the
// largest.  V's values as operands: weights themselves, 2^kGoal and 2^15 (where they may be multiplied by
// 1 / kShrink, 2^10).  V's scale in the weight: products below 2^15, for scales below 2^e (the tile's largest one).
constexpr float kGoal = 8.f, kMost = 0x1p15f, kMostShrunk = 0x1p10f;
constexpr int kGoalBelow = 8;
struct Headroom {
    float goal, most;
};
__device__ __forceinline__ Headroom headroom_of(int e) {
    return Headroom{(float)(15 - kGoalBelow - e), xdl::bitsf((uint32_t)(127 + 15 - e) << 23)};
}

// ---- The product -----------------------------------------------------------------------------

// Bound by what a tile costs beside its products, and by the clock that both leave.  32 heads on 8 kv-heads: 8192 tokens on
// themselves 655 us, 0.85 PFLOP/s of the visible products; 2048 behind 32768 1220 us, 0.93 (a bf16 product of 8192^3 reaches
// 1.24).  A tile of 64 tokens takes a wave of 32 rows about 5060 cycles: its products 2050, softmax and decoding about 2490 of
// vector work, and little of the one beside the other, since the four waves that decode V take longer than those
// that decode K, which wait for them at the barrier.  FINE has three score products for one: 4 sequences of up to 1000 tokens, up to
// 10000 before them, 3 bits, GQA 8: 740 us.
// Tiles of 256 rows (WT = 1, eight waves) have two LDS buffers and decode a tile between the products of the one before it;
// tiles of 64 rows (WT = 2) decode and multiply in turn, two workgroups a CU.  What did not pay: the next tile's
// scores before the softmax of this one (registers spill), and the two halves of the waves a phase apart (the same time).

__device__ __forceinline__ float *part_rows(const Args &a, int slot) { return a.parts + (int64_t)slot * a.shape.rows * kHeadDim; }
__device__ __forceinline__ float *part_sums(const Args &a, int slot) {
    return a.parts + (int64_t)2 * a.groups * a.shape.rows * kHeadDim + (int64_t)slot * a.shape.rows;
}
template <typename T> __device__ __forceinline__ void put8(void *out, int64_t at, const float (&v)[8]) {
    typedef T t8 __attribute__((ext_vector_type(8)));
    t8 x;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        x[i] = (T)v[i];
    *reinterpret_cast<t8 *>(static_cast<T *>(out) + at) = x;
}

template <int LAYOUT, bool KF8, bool KB3, bool V3, int WR, int WT, int KT, int BUFS, bool FINE>
__global__ __launch_bounds__(64 * WR * WT) __attribute__((amdgpu_waves_per_eu(2, 2)))
void chunk_kernel(const Args a) {
    using S = Form<WR, WT, KT, BUFS, KF8, FINE>;
    using F = Factors<KT, KF8, FINE>;
    using K = KUnit<LAYOUT, KF8, KB3, FINE>;
    using V = VUnit<LAYOUT, V3, FINE, S::vrow>;
    using T = Table<KF8, KB3, K::WIDE>;
    __shared__ struct alignas(16) {
        typename T::Entry table[T::entries];
        F factors[BUFS];
        alignas(16) unsigned char mem[S::bytes];
    } lds;
    auto &factors = lds.factors;
    unsigned char *mem = lds.mem;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 31, h = lane >> 5, wr = w % WR, wt = w / WR;
    // neighbours in the list read the same tokens: eight runs of it, one per XCD (workgroup i runs on XCD i % 8)
    const int per = gridDim.x >> 3, group_id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (group_id >= a.groups)
        return;
    Cut at = a.cuts[group_id];
    const Cut end = a.cuts[group_id + 1];
    if (at.b >= a.batch || (same_tile(at, end) && at.at == end.at))
        return;
    fill_table<LAYOUT, KF8, KB3, FINE>(lds.table, a.centroids, tid, S::threads);
    const bool does_k = !S::halves || w < WR * WT / 2, does_v = !S::halves || w >= WR * WT / 2;
    const int group = a.shape.group;
    xdl::lds_barrier();  // the table
    while (at.b < a.batch) {
        const Seq seq = seq_at(a, at.b);
        const int rows = seq.n * group, kvh = at.h;
        const Visits vis = visits_of(a.shape, seq, at.r);
        const Seen seen = seen_of(a.shape, seq, at.r);
        const bool last = same_tile(at, end);
        const int tile0 = at.at, tile1 = last ? end.at : vis.count;
        if (last && tile0 >= tile1)
            break;
        const int n_tiles = tile1 - tile0;
        const int32_t *pages = a.pages + (int64_t)at.b * a.table_width;

        auto first_of = [&](int i) __attribute__((always_inline)) {  // the first token of tile i of this stretch (past its end: of the last one)
            const int p = tile0 + min(i, n_tiles - 1);
            return KT * (p < vis.head ? p : p + vis.skip);
        };
        constexpr int U = S::units;
        auto unit = [&](int k) __attribute__((always_inline)) { return S::halves ? tid & (4 * KT - 1) : tid + k * S::threads; };
        Raw rk[U], rv_own[U];
        Raw(&rv)[U] = S::halves ? rk : rv_own;
        int blk[U];
        // the first of the 16 tokens of the wave's units, in the tile
        auto group_of = [&](int k) __attribute__((always_inline)) { return 16 * (S::halves ? w % (WR * WT / 2) : w + k * WR * WT); };
        // (no block past the sequence's last one is asked for, and none in front of the window; in the others, any token is in
        // bounds.  A vector load, though every lane's is the same: a scalar one in flight makes every wait for LDS a wait
        // for it)
        auto read_pages = [&](int i) __attribute__((always_inline)) {
#pragma unroll
            for (int k = 0; k < U; ++k) {
                uint32_t at = (uint32_t)read_at(seen, seq.len, first_of(i) + group_of(k)) >> a.block_size_log2;
                asm("" : "+v"(at));
                blk[k] = pages[at];
            }
        };
        auto load = [&](int i, bool does_k, bool does_v) __attribute__((always_inline)) {
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const int within = (first_of(i) + group_of(k)) & ((1 << a.block_size_log2) - 1);
                const Place at = place_of<LAYOUT, KF8, KB3, V3>(a, kvh, __builtin_amdgcn_readfirstlane(blk[k]), within);
                if (does_k)
                    load_k<LAYOUT, KF8, KB3, V3>(rk[k], a, at, lane);
                if (does_v)
                    load_v<LAYOUT, KF8, KB3, V3>(rv[k], a, at, lane);
            }
        };
        // A tile's decoding, in steps 0 .. kSteps - 1; `k`, `v`: of which.
        constexpr int kSteps = 5 * U;
        K kdec[U];
        V vdec[U];
        auto decode = [&](int i, int step, auto k_too, auto v_too) __attribute__((always_inline)) {
            unsigned char *m = mem + (i % BUFS) * S::tile;
            const int x = step / 5, q = step % 5, u = unit(x);
            if constexpr (k_too) {
                const int at = (u >> 2) * kKRow + 64 * (u & 3);
                if (q < 4)
                    kdec[x].look_up(rk[x], lds.table, q);
                if (q > 0)
                    kdec[x].write(m, m + S::klo, at, q - 1);
                if (q == 4)
                    kdec[x].write_norm(rk[x], factors[i % BUFS], u);
                if (q == 4)
                    kdec[x].sq = kdec[x].hl = 0.f;
            }
            if constexpr (v_too) {
                const int quad = 4 * (u >> 6) + ((u >> 2) & 3), e = 4 * (u & 3) + ((u >> 4) & 3);
                if (q == 0) {
                    const bool gone = hidden(seen, first_of(i) + group_of(x));
                    vdec[x].begin(rv[x], factors[i % BUFS], quad, gone || first_of(i) + KT > seq.len,
                                  gone ? 0 : seq.len - first_of(i) - 4 * quad);
                } else
                    vdec[x].write(m + S::v + e * S::vrow + 16 * (2 * (quad >> 2) + (quad & 1)) + 8 * ((quad >> 1) & 1), q - 1);
            }
        };
        if (n_tiles > 0) {
            read_pages(0);
            load(0, does_k, does_v);
            read_pages(1);
        }

        // this lane's row and its query
        const int wave_row = at.r * a.shape.rows + 32 * wr, row = wave_row + c, row_in = min(row, rows - 1);
        const int token = row_in / group, head = kvh * group + (row_in - token * group);
        const int64_t q_row = (int64_t)(seq.row0 + token) * a.num_q_heads + head;
        half8 q_hi[8], q_lo[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            q_hi[k] = *reinterpret_cast<const half8 *>(a.q_hi + q_row * kHeadDim + 16 * k + 8 * h);
            if constexpr (FINE && !KF8)
                q_lo[k] = *reinterpret_cast<const half8 *>(a.q_lo + q_row * kHeadDim + 16 * k + 8 * h);
        }
        const float fac = a.q_factor[q_row];
        // (arrived before the loop: a wait inside it would wait for the tiles' loads too)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            q_hi[k] = prefix::pinned(q_hi[k]);
            if constexpr (FINE && !KF8)
                q_lo[k] = prefix::pinned(q_lo[k]);
        }
        const bool scaled = !KF8 && __any(fac != 1.f);
        const int limit = limit_of(a.shape, seq, row_in), from = a.shape.window ? limit - a.shape.window : 0;
        const int limit_lo = __builtin_amdgcn_readfirstlane(limit_of(a.shape, seq, min(wave_row, rows - 1)));
        const int limit_hi = __builtin_amdgcn_readfirstlane(limit_of(a.shape, seq, min(wave_row + 31, rows - 1)));

        floatx16 acc[4];
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int k = 0; k < 16; ++k)
                acc[d][k] = 0.f;
        float negm = __FLT_MAX__, l = 0.f, z = 0.f;  // goal - max in log2 units, this lane's shares of the sum and of V's middle values

        constexpr int kAtOnce = FINE ? 1 : S::sub;  // sub-tiles of 32 tokens at once
        constexpr int kEvery = 4;                   // products between two steps of decoding
        const unsigned char *k_at = mem + (32 * S::sub * wt + c) * kKRow + 16 * h;
        const unsigned char *v_at = mem + S::v + c * S::vrow + 16 * (4 * S::sub * wt + h);
        const int tok0 = 32 * S::sub * wt + 4 * h;  // s[b][k]: token tok0 + 32 b + 8 (k / 4) + k % 4 of the tile
        std::integral_constant<bool, true> yes;
        std::integral_constant<bool, false> no;

        // Scores of sub-tiles b0 .. b0 + kAtOnce - 1 of tile i, and between their products a share of the decoding of
        // tile j (`decodes`), whose codes are here; with the last ones the loads of the tile after it.
        floatx16 s[kAtOnce];
        auto scores = [&](int i, int b0, int j, auto decodes, auto k_too, auto v_too) __attribute__((always_inline)) {
            const unsigned char *k_from = k_at + (i % BUFS) * S::tile + 32 * b0 * kKRow;
            constexpr int N = 8 * kAtOnce, kSlots = 8 * S::sub / kEvery;  // slots for decoding in a whole tile
            constexpr bool LO = FINE && !KF8;
            constexpr int AHEAD = LO ? 2 : kAhead;  // (three products from one pair of reads)
            half8 hi[AHEAD], lo[LO ? AHEAD : 1];
            auto read = [&](int x) __attribute__((always_inline)) {
                const unsigned char *from = k_from + 32 * (x >> 3) * kKRow + 32 * (x & 7);
                hi[x % AHEAD] = *reinterpret_cast<const half8 *>(from);
                if constexpr (LO)
                    lo[x % AHEAD] = *reinterpret_cast<const half8 *>(from + S::klo);
            };
#pragma unroll
            for (int x = 0; x < AHEAD; ++x)
                read(x);
#pragma unroll
            for (int b = 0; b < kAtOnce; ++b)
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    s[b][k] = 0.f;
#pragma unroll
            for (int x = 0; x < N; ++x) {
                if (decodes && x % kEvery == 0) {
                    __builtin_amdgcn_sched_barrier(0);
                    const int slot = (8 * b0 + x) / kEvery;
#pragma unroll
                    for (int y = slot * kSteps / (kSlots + 1); y < (slot + 1) * kSteps / (kSlots + 1); ++y)
                        decode(j, y, k_too, v_too);
                }
                const int b = x >> 3, k = x & 7;
                s[b] = prefix::mfma32(hi[x % AHEAD], q_hi[k], s[b]);
                if constexpr (LO) {
                    s[b] = prefix::mfma32(lo[x % AHEAD], q_hi[k], s[b]);
                    s[b] = prefix::mfma32(hi[x % AHEAD], q_lo[k], s[b]);
                }
                if (x + AHEAD < N)
                    read(x + AHEAD);
            }
            if (decodes && b0 + kAtOnce == S::sub) {
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int y = kSlots * kSteps / (kSlots + 1); y < kSteps; ++y)
                    decode(j, y, k_too, v_too);
                load(j + 1, k_too, v_too);
                read_pages(j + 2);
            }
        };
        auto softmax_outputs = [&](int i, int b0) __attribute__((always_inline)) {
            const F &f = factors[i % BUFS];
            const int t0 = first_of(i) + 32 * (S::sub * wt + b0), tok = tok0 + 32 * b0;  // the first token, this lane's in the tile
            uint32_t special = 0;
#pragma unroll
            for (int k = 0; k < KT / 16; ++k)
                special |= f.special[k];
            special = __builtin_amdgcn_readfirstlane(special);
            const bool masked = t0 + 32 * kAtOnce > limit_lo || (a.shape.window && t0 < limit_hi - a.shape.window);
            Headroom room{kGoal, special ? kMostShrunk : kMost};
            if constexpr (FINE) {  // (f16 with exponent bits x: below 2^(x - 14))
                uint32_t top = f.top[0];
#pragma unroll
                for (int k = 1; k < KT / 16; ++k)
                    top = max(top, f.top[k]);
                room = headroom_of((__builtin_amdgcn_readfirstlane(top) >> 10) - 14);
            }
            // the scores in log2 units, less the running maximum
            const bool fresh = __any(negm == __FLT_MAX__);  // rows that have seen nothing yet
            const float less = fresh ? 0.f : negm;
#pragma unroll
            for (int b = 0; b < kAtOnce; ++b) {
                float n[16];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if constexpr (KF8) {
                        n[4 * k] = n[4 * k + 1] = n[4 * k + 2] = n[4 * k + 3] = fac;
                    } else {
                        const float4 v = *reinterpret_cast<const float4 *>(f.norm + tok + 32 * b + 8 * k);
                        n[4 * k] = v.x;
                        n[4 * k + 1] = v.y;
                        n[4 * k + 2] = v.z;
                        n[4 * k + 3] = v.w;
                    }
                }
                if (masked || scaled) {
                    const int first = t0 + 4 * h;
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const int t = first + 32 * b + 8 * (k >> 2) + (k & 3);
                        const bool out = t >= limit || (t < from && t >= a.shape.first);
                        s[b][k] = out ? -INFINITY : s[b][k];
                        n[k] = out ? 1.f : KF8 ? n[k] : n[k] * fac;
                    }
                }
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    s[b][k] = fmaf(s[b][k], n[k], less);
            }
            // the maximum moved by what the scores are above its goal (first: to the tile's own)
            auto move = [&](bool first) __attribute__((always_inline)) {
                float mx = -INFINITY;
#pragma unroll
                for (int b = 0; b < kAtOnce; ++b)
#pragma unroll
                    for (int k = 0; k < 16; k += 2)
                        mx = prefix::max3(mx, s[b][k], s[b][k + 1]);
                const float top = prefix::pair_max(mx), above = first ? top + negm : top;
                const float negm_new = above > room.goal ? (first ? room.goal - top : negm + (room.goal - top)) : negm;
                const float alpha = __builtin_amdgcn_exp2f(negm_new - negm), add = first ? negm_new : negm_new - negm;
                negm = negm_new;
                l *= alpha;
                z *= alpha;
#pragma unroll
                for (int d = 0; d < 4; ++d)
                    acc[d] *= alpha;
#pragma unroll
                for (int b = 0; b < kAtOnce; ++b)
#pragma unroll
                    for (int k = 0; k < 16; ++k)
                        s[b][k] += add;
            };
            if (fresh)
                move(true);
            half8 p[kAtOnce][2];
            float sum = 0.f, mid = 0.f;
            auto weights = [&]() __attribute__((always_inline)) {
                sum = mid = 0.f;
                if (special) {
#pragma unroll
                    for (int b = 0; b < kAtOnce; ++b)
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            const int t = tok + 32 * b + 8 * (k >> 2) + (k & 3);
                            const float e = __builtin_amdgcn_exp2f(s[b][k]);
                            sum += e;
                            // (a hidden token's V is nothing, whatever it holds)
                            const float fix = s[b][k] == -INFINITY ? 0.f : f.special[t >> 4] ? f.fix[t] : 1.f;
                            float y = e * fix;
                            if constexpr (FINE) {
                                const float2 vv = f.v[t];
                                mid = fmaf(y, vv.y, mid);
                                y *= vv.x;
                            }
                            p[b][k >> 3][k & 7] = (_Float16)y;
                        }
                    return;
                }
#pragma unroll
                for (int b = 0; b < kAtOnce; ++b) {
                    if constexpr (FINE) {
#pragma unroll
                        for (int k = 0; k < 16; k += 2) {
                            const float4 v = *reinterpret_cast<const float4 *>(f.v + tok + 32 * b + 8 * (k >> 2) + (k & 3));
                            const float e0 = __builtin_amdgcn_exp2f(s[b][k]), e1 = __builtin_amdgcn_exp2f(s[b][k + 1]);
                            sum += e0;
                            sum += e1;
                            mid = fmaf(e0, v.y, mid);
                            mid = fmaf(e1, v.w, mid);
                            p[b][k >> 3][k & 7] = (_Float16)(e0 * v.x);
                            p[b][k >> 3][(k & 7) + 1] = (_Float16)(e1 * v.z);
                        }
                    } else {
                        // (the sum is of the rounded weights, so that their roundings' common part cancels)
                        typedef __fp16 fp16x2 __attribute__((ext_vector_type(2)));
                        uint32_t pk[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const fp16x2 two{(__fp16)__builtin_amdgcn_exp2f(s[b][2 * k]), (__fp16)__builtin_amdgcn_exp2f(s[b][2 * k + 1])};
                            sum = __builtin_amdgcn_fdot2(two, fp16x2{(__fp16)1.f, (__fp16)1.f}, sum, false);
                            pk[k] = __builtin_bit_cast(uint32_t, two);
                        }
                        p[b][0] = xdl::as_half8(pk[0], pk[1], pk[2], pk[3]);
                        p[b][1] = xdl::as_half8(pk[4], pk[5], pk[6], pk[7]);
                    }
                }
            };
            weights();
            if (__any(sum > room.most)) {
                move(false);
                weights();
            }
            l += sum;
            z += mid;
            const unsigned char *v_from = v_at + (i % BUFS) * S::tile;
            half8 v[kAhead];
            constexpr int N = 8 * kAtOnce;
            auto read = [&](int x) __attribute__((always_inline)) {
                v[x % kAhead] = *reinterpret_cast<const half8 *>(v_from + 32 * (x & 3) * S::vrow + 32 * (2 * b0 + (x >> 2)));
            };
#pragma unroll
            for (int x = 0; x < kAhead; ++x)
                read(x);
            auto output = [&](int x) __attribute__((always_inline)) {
                acc[x & 3] = prefix::mfma32(v[x % kAhead], p[x >> 3][(x >> 2) & 1], acc[x & 3]);
                if (x + kAhead < N)
                    read(x + kAhead);
            };
#pragma unroll
            for (int x = 0; x < N; ++x)
                output(x);
        };
        // (each kind of wave has a loop of its own: where the two met, the codes in flight would have to arrive)
        auto loop = [&](auto k_too, auto v_too) __attribute__((always_inline)) {
            auto all = [&](int i) __attribute__((always_inline)) {  // all of a tile's decoding at once
#pragma unroll
                for (int y = 0; y < kSteps; ++y)
                    decode(i, y, k_too, v_too);
                load(i + 1, k_too, v_too);
                read_pages(i + 2);
            };
            if constexpr (BUFS == 2) {
                if (n_tiles > 0)
                    all(0);
                xdl::lds_barrier();
                // (the last tile's turn decodes it again, into the other buffer: no branch in the loop)
                for (int i = 0; i < n_tiles; ++i) {
#pragma unroll
                    for (int b = 0; b < S::sub; b += kAtOnce) {
                        scores(i, b, i + 1, yes, k_too, v_too);
                        softmax_outputs(i, b);
                    }
                    xdl::lds_barrier();
                }
            } else {
                for (int i = 0; i < n_tiles; ++i) {
                    all(i);
                    xdl::lds_barrier();
#pragma unroll
                    for (int b = 0; b < S::sub; b += kAtOnce) {
                        scores(i, b, 0, no, no, no);
                        softmax_outputs(i, b);
                    }
                    xdl::lds_barrier();
                }
            }
        };
        if constexpr (S::halves)
            does_k ? loop(yes, no) : loop(no, yes);
        else
            loop(yes, yes);

        l = prefix::pair_sum(l);
        z = prefix::pair_sum(z);
        if constexpr (WT > 1) {
            // waves wt > 0 leave their sums in LDS, waves wt = 0 join them with theirs
            constexpr int kWords = 64 * 67;
            float *mine = reinterpret_cast<float *>(mem) + lane;
            if (wt > 0) {
                float *to = mine + ((wt - 1) * WR + wr) * kWords;
#pragma unroll
                for (int d = 0; d < 4; ++d)
#pragma unroll
                    for (int k = 0; k < 16; ++k)
                        to[64 * (16 * d + k)] = acc[d][k];
                to[64 * 64] = negm;
                to[64 * 65] = l;
                to[64 * 66] = z;
            }
            xdl::lds_barrier();
            if (wt == 0)
                for (int o = 0; o < WT - 1; ++o) {
                    const float *of = mine + (o * WR + wr) * kWords;
                    const float negm1 = of[64 * 64], both = fminf(negm, negm1);
                    const float w0 = __builtin_amdgcn_exp2f(both - negm), w1 = __builtin_amdgcn_exp2f(both - negm1);
                    negm = both;
                    l = l * w0 + of[64 * 65] * w1;
                    z = z * w0 + of[64 * 66] * w1;
#pragma unroll
                    for (int d = 0; d < 4; ++d)
#pragma unroll
                        for (int k = 0; k < 16; ++k)
                            acc[d][k] = acc[d][k] * w0 + of[64 * (16 * d + k)] * w1;
                }
        }
        const bool whole = tile0 == 0 && tile1 == vis.count;
        if (wt == 0 && row < rows) {
            if (whole && a.sinks) {
                const float sink = a.sinks[head] * kLog2e, negm_new = fminf(negm, -sink);
                const float w0 = __builtin_amdgcn_exp2f(negm_new - negm);
                negm = negm_new;
                l = l * w0 + __builtin_amdgcn_exp2f(sink + negm);
                z *= w0;
#pragma unroll
                for (int d = 0; d < 4; ++d)
                    acc[d] *= w0;
            }
            const float inv = l == 0.f ? 0.f : 1.f / l;
            const int slot = 2 * group_id + (tile0 == 0 ? 1 : 0), place = 32 * wr + c;
            float *part = part_rows(a, slot) + (int64_t)place * kHeadDim;
            const int64_t o = q_row * kHeadDim;
            // accumulator d, register 4 q + i: row 32 d + 8 q + 4 h + i of V^T, dim 8 (8 (q % 2) + 4 h + i) + 2 d + q / 2
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int k = 4 * q + i, dim = 8 * (8 * q + 4 * h + i);
                    const float v[8] = {(acc[0][k] + z) * inv, (acc[0][8 + k] + z) * inv, (acc[1][k] + z) * inv, (acc[1][8 + k] + z) * inv,
                                        (acc[2][k] + z) * inv, (acc[2][8 + k] + z) * inv, (acc[3][k] + z) * inv, (acc[3][8 + k] + z) * inv};
                    if (!whole) {
                        *reinterpret_cast<float4 *>(part + dim) = float4{v[0], v[1], v[2], v[3]};
                        *reinterpret_cast<float4 *>(part + dim + 4) = float4{v[4], v[5], v[6], v[7]};
                    } else if (a.out_dtype == kOutBf16) {
                        put8<__bf16>(a.out, o + dim, v);
                    } else {
                        put8<_Float16>(a.out, o + dim, v);
                    }
                }
            const float lse2 = __builtin_amdgcn_logf(l) - negm;
            if (h == 0 && !whole)
                part_sums(a, slot)[place] = lse2;
            else if (h == 0 && a.lse)
                a.lse[q_row] = l == 0.f ? -INFINITY : lse2 * kLn2;
        }
        if (last)
            break;
        if constexpr (WT > 1)
            xdl::lds_barrier();  // the sums are read
        // the next row tile
        at.at = 0;
        if (++at.r == row_tiles(a.shape, seq.n)) {
            at.r = 0;
            if (++at.h == a.num_kv_heads) {
                at.h = 0;
                do
                    ++at.b;
                while (at.b < a.batch && seq_at(a, at.b).n == 0);
            }
        }
    }
}

// Joins the parts of a row tile that was cut: workgroup (i, w) rows of the one that workgroup w of chunk_kernel began and
// did not end, PER of them per half wave, four parts at a time.  Lane: dims 4 x .. +3 of its half's row.  Bound by the parts'
// bytes: 8192 tokens of 32 heads 18.7 us (1, 4 and 8 rows per half wave: 21, 19.2, 23), 84 MB.  Consecutive workgroups
// have the rows of one row tile: with w in their place the few row tiles of a lone sequence fell to one XCD (8 of them, 32 parts each:
// 50 us, now 15).
constexpr int kMergeThreads = 128, kMergeHalves = kMergeThreads / 32, kMergePer = 2;
template <typename OutT> __global__ __launch_bounds__(kMergeThreads) void chunk_merge_kernel(const Args a) {
    constexpr int PER = kMergePer;
    const int w = blockIdx.y, x = threadIdx.x & 31, half = threadIdx.x >> 5;
    const Cut from = a.cuts[w], cut = a.cuts[w + 1];
    if (cut.b >= a.batch || cut.at == 0 || (same_tile(from, cut) && from.at > 0))
        return;
    const Seq seq = seq_at(a, cut.b);
    const int rows = seq.n * a.shape.group, place0 = (blockIdx.x * kMergeHalves + half) * PER;
    if (cut.r * a.shape.rows + (int)blockIdx.x * kMergeHalves * PER >= rows)
        return;
    // part i: of workgroup w + i; the last is of the first whose own stretch ends in another row tile (64 cuts at a time: one
    // after the other 32 parts took 10 us)
    int parts = 2;
    for (;;) {
        const uint64_t same = __ballot(same_tile(a.cuts[min(w + parts + (int)(threadIdx.x & 63), a.groups)], cut));
        if (~same) {
            parts += __builtin_ctzll(~same);
            break;
        }
        parts += 64;
    }
    auto slot = [&](int j) { return 2 * (w + j) + (j == 0 ? 1 : 0); };
    auto wrote = [&](int j) {  // (a workgroup without tiles wrote nothing)
        const Cut p = a.cuts[w + j], q = a.cuts[w + j + 1];
        return j == 0 || !same_tile(p, q) || p.at < q.at;
    };
    float mx[PER], sum[PER];
    float4 acc[PER];
#pragma unroll
    for (int r = 0; r < PER; ++r) {
        mx[r] = -INFINITY;
        sum[r] = 0.f;
        acc[r] = float4{0.f, 0.f, 0.f, 0.f};
    }
    for (int i0 = 0; i0 < parts; i0 += 32) {
        const int i = i0 + x, n = min(32, parts - i0);
        const bool there = i < parts && wrote(i);
        float wt[PER];
#pragma unroll
        for (int r = 0; r < PER; ++r) {
            const float s = there ? part_sums(a, slot(i))[min(place0 + r, a.shape.rows - 1)] : -INFINITY;
            float top = s;
#pragma unroll
            for (int m = 16; m >= 1; m >>= 1)
                top = fmaxf(top, __shfl_xor(top, m, 32));
            const float m_new = fmaxf(mx[r], top), scale = mx[r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mx[r] - m_new);
            wt[r] = s == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s - m_new);
            float all = wt[r];
#pragma unroll
            for (int m = 16; m >= 1; m >>= 1)
                all += __shfl_xor(all, m, 32);
            sum[r] = sum[r] * scale + all;
            acc[r] = float4{acc[r].x * scale, acc[r].y * scale, acc[r].z * scale, acc[r].w * scale};
            mx[r] = m_new;
        }
        constexpr int AT_ONCE = 4;  // parts
        for (int j0 = 0; j0 < n; j0 += AT_ONCE) {
            float4 v[AT_ONCE][PER];
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j)
#pragma unroll
                for (int r = 0; r < PER; ++r)
                    v[j][r] = reinterpret_cast<const float4 *>(part_rows(a, slot(i0 + min(j0 + j, n - 1))) +
                                                               (int64_t)min(place0 + r, a.shape.rows - 1) * kHeadDim)[x];
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j)
#pragma unroll
                for (int r = 0; r < PER; ++r) {
                    const float wj = __shfl(wt[r], j0 + j, 32);
                    if (j0 + j < n && wj != 0.f) {  // (a part without weight may hold anything)
                        acc[r].x = fmaf(wj, v[j][r].x, acc[r].x);
                        acc[r].y = fmaf(wj, v[j][r].y, acc[r].y);
                        acc[r].z = fmaf(wj, v[j][r].z, acc[r].z);
                        acc[r].w = fmaf(wj, v[j][r].w, acc[r].w);
                    }
                }
        }
    }
#pragma unroll
    for (int r = 0; r < PER; ++r) {
        const int row = cut.r * a.shape.rows + place0 + r;
        if (place0 + r >= a.shape.rows || row >= rows)
            break;
        const int token = row / a.shape.group, head = cut.h * a.shape.group + row - token * a.shape.group;
        float scale = 1.f;
        if (a.sinks) {
            const float sink = a.sinks[head] * kLog2e, m_new = fmaxf(mx[r], sink);
            scale = mx[r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mx[r] - m_new);
            sum[r] = sum[r] * scale + (sink == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sink - m_new));
            mx[r] = m_new;
        }
        const float inv = sum[r] == 0.f ? 0.f : scale / sum[r];
        const int64_t q_row = (int64_t)(seq.row0 + token) * a.num_q_heads + head;
        typedef OutT out4 __attribute__((ext_vector_type(4)));
        reinterpret_cast<out4 *>(static_cast<OutT *>(a.out) + q_row * kHeadDim)[x] =
            out4{(OutT)(acc[r].x * inv), (OutT)(acc[r].y * inv), (OutT)(acc[r].z * inv), (OutT)(acc[r].w * inv)};
        if (x == 0 && a.lse)
            a.lse[q_row] = sum[r] == 0.f ? -INFINITY : (mx[r] + __builtin_amdgcn_logf(sum[r])) * kLn2;
    }
}

}  // namespace chunk
}  // namespace tq4
