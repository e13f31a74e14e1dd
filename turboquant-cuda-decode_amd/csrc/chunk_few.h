// chunk_attention for sequences with few query rows (drafted tokens, short chunks): up to 32 rows of a kv-head, on average.
//
// Here the cache's bytes count, and nothing is gained by sharing decoded tiles between waves: each wave takes 32 tokens of
// its own at a time and keeps them in registers, with the rows in the columns of 16x16x32 products,
//
//   S^T[token][row] = sum_d c[token][d] q[row][d]      A = the keys' codes, B = q: lane (n, g) = (lane % 16, lane / 16) has
//                                                      dims 32 g .. +31 of token n as they lie in the cache (one load)
//   O^T[dim][row]  += sum_t V^T[dim][t] P^T[t][row]    A = V's codes less the middle one: lane (n, g) has dims 8 n .. +7 of
//                                                      tokens 4 g .. +3 of both halves of 16 (one dword each)
//
// A lane's scores are those of row n and tokens 4 g .. +3 of both halves: the weights are the second product's operand as
// they stand, in the order of V's tokens.  The four waves of a workgroup take 32 of each 128 tokens and join in LDS.
// Scores are one f16 product, or three of f16 pairs (FINE); V's scale is part of the weight, one f16.
//
// 64 sequences of 1 to 8 drafted tokens behind 512 to 8192 (32 heads on 8 kv-heads, 302 MB): 105 us, 2.9 TB/s of the copy's 5.1:
// vector instructions in 58 % of the cycles, the rest the latency of records and lookups with two waves a SIMD.  The same
// in tiles of 64 rows that a workgroup's waves share (chunk_kernel): 152.
#pragma once
#include "chunk.h"

namespace tq4 {
namespace chunk {

constexpr int kFewWaves = 4, kFewTile = 32 * kFewWaves, kFewBlocks = 2, kFewRows = 16 * kFewBlocks;

// What a lane loads of a wave's 32 tokens: K of token n of each half; V of eight tokens; and scalars: SoA those of its eight
// score tokens (norm, scale, zero: four and four), AoS those of token n of each half (norm; scale | zero << 16).
template <int LAYOUT, bool KF8> struct FewRaw {
    uint4 k[2], k2[KF8 ? 2 : 1];
    uint32_t v[8];
    uint32_t s[LAYOUT == 0 ? 12 : 4];
};
template <int LAYOUT, bool KF8, bool KB3, bool V3>
__device__ __forceinline__ void few_load_k(FewRaw<LAYOUT, KF8> &r, const Args &a, const Place &at, int half, int lane) {
    using C = Codes<LAYOUT, KF8, KB3, V3>;
    const int n = lane & 15, g = lane >> 4;
    const uint32_t token = (uint32_t)n * (uint32_t)a.slot_pos, part = token + g * (C::kbytes / 4);
    r.k[half] = KB3 ? load12(at.data, part, 0) : load16(at.data, part, 0);
    if constexpr (KF8)
        r.k2[half] = load16(at.data, part, 16);
}
template <int LAYOUT, bool KF8, bool KB3, bool V3>
__device__ __forceinline__ void few_load_v(FewRaw<LAYOUT, KF8> &r, const Args &a, const Place &at, int half, int lane) {
    using C = Codes<LAYOUT, KF8, KB3, V3>;
    const int n = lane & 15, g = lane >> 4;
    const uint32_t token = (uint32_t)n * (uint32_t)a.slot_pos;
    const uint32_t quad = (uint32_t)(4 * g) * (uint32_t)a.slot_pos + (V3 ? 3 : 4) * n;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        r.v[4 * half + i] = load4(at.data, quad, i * a.slot_pos + C::v0);
    if constexpr (LAYOUT == 0) {
#pragma unroll
        for (int f = 0; f < C::nf; ++f) {
            const uint2 s = load8(at.meta, 8u * g, (2 * f) << a.block_size_log2);
            const int to = f + 3 - C::nf;
            r.s[4 * to + 2 * half] = s.x;
            r.s[4 * to + 2 * half + 1] = s.y;
        }
    } else {
        if constexpr (!KF8)
            r.s[half] = load2(at.data, token, C::kbytes);
        r.s[2 + half] = load4(at.data, token, C::v0 + C::vbytes);
    }
}

template <int LAYOUT, bool KF8, bool KB3, bool V3, bool FINE>
__global__ __launch_bounds__(kWave *kFewWaves) __attribute__((amdgpu_waves_per_eu(2, 2)))
void chunk_few_kernel(const Args a) {
    constexpr int RB = kFewBlocks;
    constexpr bool WIDE = FINE || LAYOUT == 1;
    using T = Table<KF8, KB3, WIDE>;
    constexpr int kWords = RB * 32 + 3 * RB;  // of a lane's state
    __shared__ struct alignas(16) {
        typename T::Entry table[T::entries];
        float norm[LAYOUT == 1 ? kFewWaves : 1][32];
        float2 v[LAYOUT == 1 ? kFewWaves : 1][32];
        float join[(kFewWaves - 1) * kWords * kWave];
    } lds;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15, g = lane >> 4;
    const int per = gridDim.x >> 3, group_id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (group_id >= a.groups)
        return;
    Cut at = a.cuts[group_id];
    const Cut end = a.cuts[group_id + 1];
    if (at.b >= a.batch || (same_tile(at, end) && at.at == end.at))
        return;
    fill_table<LAYOUT, KF8, KB3, FINE>(lds.table, a.centroids, tid, kWave * kFewWaves);
    __syncthreads();
    const int group = a.shape.group;
    while (at.b < a.batch) {
        const Seq seq = seq_at(a, at.b);
        const int rows = seq.n * group, kvh = at.h, row0 = at.r * a.shape.rows;
        const Visits vis = visits_of(a.shape, seq, at.r);
        const Seen seen = seen_of(a.shape, seq, at.r);
        const bool last = same_tile(at, end);
        const int tile0 = at.at, tile1 = last ? end.at : vis.count;
        if (last && tile0 >= tile1)
            break;
        const int n_tiles = tile1 - tile0;
        const int blocks = rows - row0 > 16 ? 2 : 1;  // of 16 rows that the row tile has
        const int32_t *pages = a.pages + (int64_t)at.b * a.table_width;
        auto first_of = [&](int i) __attribute__((always_inline)) {  // this wave's first token of tile i of the stretch
            const int p = tile0 + min(i, n_tiles - 1);
            return kFewTile * (p < vis.head ? p : p + vis.skip) + 32 * w;
        };
        int blk[2];
        auto read_pages = [&](int i) __attribute__((always_inline)) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                uint32_t p = (uint32_t)read_at(seen, seq.len, first_of(i) + 16 * k) >> a.block_size_log2;
                asm("" : "+v"(p));
                blk[k] = pages[p];
            }
        };
        FewRaw<LAYOUT, KF8> raw;
        auto load = [&](int i, auto k_too, auto v_too) __attribute__((always_inline)) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const Place p = place_of<LAYOUT, KF8, KB3, V3>(a, kvh, __builtin_amdgcn_readfirstlane(blk[k]),
                                                               (first_of(i) + 16 * k) & ((1 << a.block_size_log2) - 1));
                if constexpr (k_too)
                    few_load_k<LAYOUT, KF8, KB3, V3>(raw, a, p, k, lane);
                if constexpr (v_too)
                    few_load_v<LAYOUT, KF8, KB3, V3>(raw, a, p, k, lane);
            }
        };
        const std::integral_constant<bool, true> yes;
        const std::integral_constant<bool, false> no;
        if (n_tiles > 0) {
            read_pages(0);
            load(0, yes, yes);
            read_pages(1);
        }
        // the lane's rows
        half8 q_hi[RB][4], q_lo[FINE && !KF8 ? RB : 1][4];
        float fac[RB], negm[RB], l[RB], z[RB];
        int limit[RB], from[RB];
        bool any_scaled = false;
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            const int row = min(row0 + 16 * b + n, rows - 1), token = row / group, head = kvh * group + row - token * group;
            const int64_t q_row = (int64_t)(seq.row0 + token) * a.num_q_heads + head;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                q_hi[b][k] = *reinterpret_cast<const half8 *>(a.q_hi + q_row * kHeadDim + 32 * g + 8 * k);
                if constexpr (FINE && !KF8)
                    q_lo[b][k] = *reinterpret_cast<const half8 *>(a.q_lo + q_row * kHeadDim + 32 * g + 8 * k);
            }
            fac[b] = a.q_factor[q_row];
            limit[b] = limit_of(a.shape, seq, row);
            from[b] = a.shape.window ? limit[b] - a.shape.window : 0;
            negm[b] = __FLT_MAX__;
            l[b] = z[b] = 0.f;
        }
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            any_scaled |= fac[b] != 1.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                q_hi[b][k] = prefix::pinned(q_hi[b][k]);
                if constexpr (FINE && !KF8)
                    q_lo[b][k] = prefix::pinned(q_lo[b][k]);
            }
        }
        const bool scaled = !KF8 && __any(any_scaled);
        const int limit_lo = __builtin_amdgcn_readfirstlane(limit_of(a.shape, seq, min(row0, rows - 1)));
        const int limit_hi = __builtin_amdgcn_readfirstlane(limit_of(a.shape, seq, min(row0 + a.shape.rows - 1, rows - 1)));
        floatx4 acc[RB][8];
#pragma unroll
        for (int b = 0; b < RB; ++b)
#pragma unroll
            for (int d = 0; d < 8; ++d)
                acc[b][d] = floatx4{0.f, 0.f, 0.f, 0.f};

        auto tile = [&](int i) __attribute__((always_inline)) {
            const int t0 = first_of(i);
            // scores of half k: s[b][4 k + i]
            float s[RB][8], norm[8], scale[8], mid[8];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                half8 c_hi[4], c_lo[WIDE ? 4 : 1];
                float sq = 0.f, hl = 0.f;
                const uint32_t wd[4] = {raw.k[k].x, raw.k[k].y, raw.k[k].z, raw.k[k].w};
#pragma unroll
                for (int kb = 0; kb < 4; ++kb) {
                    uint32_t e[4], f[4];
                    if constexpr (KF8) {
                        const uint32_t w8[8] = {wd[0], wd[1], wd[2], wd[3], raw.k2[k].x, raw.k2[k].y, raw.k2[k].z, raw.k2[k].w};
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const auto p = __builtin_amdgcn_cvt_pk_f32_fp8((int)w8[2 * kb + x], false);
                            const auto q = __builtin_amdgcn_cvt_pk_f32_fp8((int)w8[2 * kb + x], true);
                            e[2 * x] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(p[0], p[1]));  // (exact)
                            e[2 * x + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(q[0], q[1]));
                        }
                    } else {
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const uint32_t v = code_pair<KB3>(wd, 4 * kb + x);
                            if constexpr (WIDE) {
                                const uint2 c = lds.table[v];
                                e[x] = c.x;
                                f[x] = c.y;
                                if constexpr (LAYOUT == 1 && FINE) {
                                    const auto h = __builtin_bit_cast(__fp16 __attribute__((ext_vector_type(2))), c.x);
                                    const auto lo = __builtin_bit_cast(__fp16 __attribute__((ext_vector_type(2))), c.y);
                                    sq = __builtin_amdgcn_fdot2(h, h, sq, false);
                                    hl = __builtin_amdgcn_fdot2(h, lo, hl, false);
                                } else if constexpr (LAYOUT == 1) {
                                    sq += xdl::bitsf(c.y);
                                }
                            } else {
                                e[x] = lds.table[v];
                            }
                        }
                    }
                    c_hi[kb] = xdl::as_half8(e[0], e[1], e[2], e[3]);
                    if constexpr (FINE && !KF8)
                        c_lo[kb] = xdl::as_half8(f[0], f[1], f[2], f[3]);
                }
                if constexpr (LAYOUT == 1) {
                    // the token's scalars to the lanes that have its scores, through the wave's own LDS
                    if constexpr (!KF8) {
                        sq = xdl::sum_xor32(xdl::sum_xor16(fmaf(2.f, hl, sq)));
                        lds.norm[w][16 * k + n] = half_bits_to_float(raw.s[k]) * __builtin_amdgcn_rsqf(sq + 1e-16f);
                    }
                    const float sc = half_bits_to_float(raw.s[2 + k]);
                    lds.v[w][16 * k + n] = float2{sc, fmaf(sc, kMiddle<V3>, half_bits_to_float(raw.s[2 + k] >> 16))};
                }
#pragma unroll
                for (int b = 0; b < RB; ++b) {
                    if (b >= blocks)
                        break;
                    floatx4 y{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int kb = 0; kb < 4; ++kb) {
                        y = xdl::mfma(c_hi[kb], q_hi[b][kb], y);
                        if constexpr (FINE && !KF8) {
                            y = xdl::mfma(c_lo[kb], q_hi[b][kb], y);
                            y = xdl::mfma(c_hi[kb], q_lo[b][kb], y);
                        }
                    }
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        s[b][4 * k + x] = y[x];
                }
            }
            load(i + 1, yes, no);  // (its codes are used up: as early as may be)
            if constexpr (LAYOUT == 0) {
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    auto field = [&](int f) { return half_bits_to_float(raw.s[4 * f + (x >> 1)] >> (16 * (x & 1))); };
                    norm[x] = KF8 ? 1.f : field(0);
                    scale[x] = field(1);
                    mid[x] = fmaf(scale[x], kMiddle<V3>, field(2));
                }
            } else {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    if constexpr (!KF8) {
                        const float4 x = *reinterpret_cast<const float4 *>(&lds.norm[w][16 * k + 4 * g]);
                        norm[4 * k] = x.x;
                        norm[4 * k + 1] = x.y;
                        norm[4 * k + 2] = x.z;
                        norm[4 * k + 3] = x.w;
                    }
#pragma unroll
                    for (int x = 0; x < 4; x += 2) {
                        const float4 y = *reinterpret_cast<const float4 *>(&lds.v[w][16 * k + 4 * g + x]);
                        scale[4 * k + x] = y.x;
                        mid[4 * k + x] = y.y;
                        scale[4 * k + x + 1] = y.z;
                        mid[4 * k + x + 1] = y.w;
                    }
                }
            }
            // V's codes less the middle one: dim 8 n + d, the lane's eight tokens
            half8 v[8];
            {
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    half2v even[4], odd[4];
#pragma unroll
                    for (int t = 0; t < 4; ++t)
                        code_values<V3>(raw.v[2 * t], raw.v[2 * t + 1], m, kMiddle<V3>, even[t], odd[t]);
                    auto pack = [](const half2v(&x)[4]) {
                        return xdl::as_half8(prefix::as_u32(x[0]), prefix::as_u32(x[1]), prefix::as_u32(x[2]), prefix::as_u32(x[3]));
                    };
                    v[2 * m] = pack(even);
                    v[2 * m + 1] = pack(odd);
                }
            }
            // what is not finite (of tokens past the sequence too, which then costs time only)
            uint32_t top_v;
            if constexpr (LAYOUT == 0)
                top_v = top_of(most_of(most_of(most_of(raw.s[4], raw.s[5]), most_of(raw.s[6], raw.s[7])),
                                       most_of(most_of(raw.s[8], raw.s[9]), most_of(raw.s[10], raw.s[11]))));
            else
                top_v = top_of(most_of(raw.s[2], raw.s[3]));
            const bool special = __any(top_v >= 0x7C00u);
            load(i + 1, no, yes);
            read_pages(i + 2);
            const bool masked = t0 + 32 > limit_lo || (a.shape.window && t0 < limit_hi - a.shape.window);
            // tokens past the sequence, and those whose block is not read: their bytes may hold anything
            const bool gone[2] = {hidden(seen, t0), hidden(seen, t0 + 16)};
            if (t0 + 32 > seq.len || gone[0] || gone[1])
#pragma unroll
                for (int x = 0; x < 8; ++x)
                    if (gone[x >> 2] || t0 + 16 * (x >> 2) + 4 * g + (x & 3) >= seq.len)
                        scale[x] = mid[x] = 0.f;
            // the largest scale of the wave's 32 tokens
            float top_s = 0.f;
            if (special) {
#pragma unroll
                for (int x = 0; x < 8; ++x)
                    top_s = fmaxf(top_s, fabsf(scale[x]) < __builtin_inff() ? fabsf(scale[x]) : 0.f);
            } else {
#pragma unroll
                for (int x = 0; x < 8; ++x)
                    top_s = fmaxf(top_s, fabsf(scale[x]));
            }
            top_s = xdl::max_xor16(xdl::max_xor32(top_s));
            const Headroom room = headroom_of(__builtin_amdgcn_readfirstlane(__builtin_amdgcn_frexp_expf(top_s)));
#pragma unroll
            for (int b = 0; b < RB; ++b) {
                if (b >= blocks)
                    break;
                const bool fresh = __any(negm[b] == __FLT_MAX__);
                const float less = fresh ? 0.f : negm[b];
                if (masked || scaled) {
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        const int t = t0 + 16 * (x >> 2) + 4 * g + (x & 3);
                        const bool out = t >= limit[b] || (t < from[b] && t >= a.shape.first);
                        const float y = fmaf(s[b][x], KF8 ? fac[b] : norm[x] * fac[b], less);
                        s[b][x] = out ? -INFINITY : y;
                    }
                } else {
#pragma unroll
                    for (int x = 0; x < 8; ++x)
                        s[b][x] = fmaf(s[b][x], KF8 ? fac[b] : norm[x], less);
                }
                auto move = [&](bool first) __attribute__((always_inline)) {
                    float mx = -INFINITY;
#pragma unroll
                    for (int x = 0; x < 8; x += 2)
                        mx = prefix::max3(mx, s[b][x], s[b][x + 1]);
                    const float top = xdl::max_xor16(xdl::max_xor32(mx)), above = first ? top + negm[b] : top;
                    const float negm_new = above > room.goal ? (first ? room.goal - top : negm[b] + (room.goal - top)) : negm[b];
                    const float alpha = __builtin_amdgcn_exp2f(negm_new - negm[b]), add = first ? negm_new : negm_new - negm[b];
                    negm[b] = negm_new;
                    l[b] *= alpha;
                    z[b] *= alpha;
#pragma unroll
                    for (int d = 0; d < 8; ++d)
                        acc[b][d] *= alpha;
#pragma unroll
                    for (int x = 0; x < 8; ++x)
                        s[b][x] += add;
                };
                if (fresh)
                    move(true);
                half8 p;
                float sum, mids;
                auto weights = [&]() __attribute__((always_inline)) {
                    sum = mids = 0.f;
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        const float e = __builtin_amdgcn_exp2f(s[b][x]);
                        sum += e;
                        float y = e * scale[x], m = mid[x];
                        if (special) {  // a hidden token's V is nothing, whatever it holds
                            const bool out = s[b][x] == -INFINITY;
                            y = out ? 0.f : y;
                            m = out ? 0.f : m;
                        }
                        mids = fmaf(e, m, mids);
                        p[x] = (_Float16)y;
                    }
                };
                weights();
                if (__any(sum > room.most)) {
                    move(false);
                    weights();
                }
                l[b] += sum;
                z[b] += mids;
#pragma unroll
                for (int d = 0; d < 8; ++d)
                    acc[b][d] = xdl::mfma(v[d], p, acc[b][d]);
            }
        };
        for (int i = 0; i < n_tiles; ++i) {
            const int t0 = first_of(i);
            // (no row of the tile sees a token of the wave's)
            if (t0 >= limit_hi || (a.shape.window && t0 >= a.shape.first && t0 + 32 <= limit_lo - a.shape.window)) {
                load(i + 1, yes, yes);
                read_pages(i + 2);
            } else {
                tile(i);
            }
        }
        // the waves' sums joined by the first wave
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            l[b] = xdl::sum_xor16(xdl::sum_xor32(l[b]));
            z[b] = xdl::sum_xor16(xdl::sum_xor32(z[b]));
        }
        __syncthreads();  // (the last row tile's sums are read)
        if (w > 0) {
            float *to = lds.join + (w - 1) * kWords * kWave + lane;
#pragma unroll
            for (int b = 0; b < RB; ++b) {
#pragma unroll
                for (int d = 0; d < 8; ++d)
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        to[kWave * (35 * b + 4 * d + x)] = acc[b][d][x];
                to[kWave * (35 * b + 32)] = negm[b];
                to[kWave * (35 * b + 33)] = l[b];
                to[kWave * (35 * b + 34)] = z[b];
            }
        }
        __syncthreads();
        const bool whole = tile0 == 0 && tile1 == vis.count;
        if (w == 0)
#pragma unroll
            for (int b = 0; b < RB; ++b) {
                for (int o = 0; o < kFewWaves - 1; ++o) {
                    const float *of = lds.join + o * kWords * kWave + lane + kWave * 35 * b;
                    const float negm1 = of[kWave * 32], both = fminf(negm[b], negm1);
                    const float w0 = __builtin_amdgcn_exp2f(both - negm[b]), w1 = __builtin_amdgcn_exp2f(both - negm1);
                    negm[b] = both;
                    l[b] = l[b] * w0 + of[kWave * 33] * w1;
                    z[b] = z[b] * w0 + of[kWave * 34] * w1;
#pragma unroll
                    for (int d = 0; d < 8; ++d)
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                            acc[b][d][x] = acc[b][d][x] * w0 + of[kWave * (4 * d + x)] * w1;
                }
                const int place = 16 * b + n, row = row0 + place;
                if (row >= rows)
                    continue;
                const int token = row / group, head = kvh * group + row - token * group;
                const int64_t q_row = (int64_t)(seq.row0 + token) * a.num_q_heads + head;
                float w0 = 1.f;
                if (whole && a.sinks) {
                    const float sink = a.sinks[head] * kLog2e, negm_new = fminf(negm[b], -sink);
                    w0 = __builtin_amdgcn_exp2f(negm_new - negm[b]);
                    negm[b] = negm_new;
                    l[b] = l[b] * w0 + __builtin_amdgcn_exp2f(sink + negm[b]);
                }
                const float inv = l[b] == 0.f ? 0.f : w0 / l[b];
                const int slot = 2 * group_id + (tile0 == 0 ? 1 : 0);
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int dim = 8 * (4 * g + x);
                    float y[8];
#pragma unroll
                    for (int d = 0; d < 8; ++d)
                        y[d] = (acc[b][d][x] + z[b]) * inv;
                    if (!whole) {
                        float4 *to = reinterpret_cast<float4 *>(part_rows(a, slot) + (int64_t)place * kHeadDim + dim);
                        to[0] = float4{y[0], y[1], y[2], y[3]};
                        to[1] = float4{y[4], y[5], y[6], y[7]};
                    } else if (a.out_dtype == kOutBf16) {
                        put8<__bf16>(a.out, q_row * kHeadDim + dim, y);
                    } else {
                        put8<_Float16>(a.out, q_row * kHeadDim + dim, y);
                    }
                }
                const float lse2 = __builtin_amdgcn_logf(l[b]) - negm[b];
                if (g == 0 && !whole)
                    part_sums(a, slot)[place] = lse2;
                else if (g == 0 && a.lse)
                    a.lse[q_row] = l[b] == 0.f ? -INFINITY : lse2 * kLn2;
            }
        if (last)
            break;
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

}  // namespace chunk
}  // namespace tq4
