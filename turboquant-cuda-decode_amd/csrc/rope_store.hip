// The cache writer with rotary positions (tq4_rope_store, include/tq4_decode.h).
#include <algorithm>

#include "abi.h"
#include "rope.h"

using namespace tq4::abi;

namespace {

// Workgroups of `waves` waves for the query rows: enough that a wave takes one run of rows, at most 2048 (eight per
// CU; behind the writer's in one launch they hold its LDS too, 67 KB, and two run on a CU at a time).
int query_groups(const tq4::rope::Args &a, int waves) {
    if (!a.query)
        return 0;
    const int64_t runs = ((int64_t)a.tokens * a.num_q_heads + tq4::rope::kQueryRows - 1) / tq4::rope::kQueryRows;
    return (int)std::min<int64_t>((runs + waves - 1) / waves, 2048);
}

// One launch for both roles has to hold the larger one's registers and LDS for both, two launches cost a
// second start.  Small workgroups with both: 38.7 us at 2049 tiles (4097 tokens, 8 kv-heads) against 24.7 + 19.9
// for two launches of large ones and 43.8 for one; at 16384 tiles 215 against 97 + 103 and 243.  Without queries
// the plain writer's limit holds.
template <int LAYOUT, class T, int KB, int VB> void launch_append(tq4::rope::Args &a, hipStream_t st) {
    using namespace tq4::store;
    const int64_t tiles = ((int64_t)a.tokens * a.num_kv_heads + kRows - 1) / kRows;
    const bool small = tiles <= (a.query ? 4 * kSmallTiles : kSmallTiles);
    const int waves = small ? kSmallWaves : kWaves;
    a.store_groups = (int)std::min<int64_t>((tiles + waves - 1) / waves, kMaxGroups);
    if (small) {
        const dim3 grid(a.store_groups + query_groups(a, waves)), block(tq4::kWave * waves);
        launch(&tq4::rope::append_kernel<LAYOUT, T, KB, VB, kSmallWaves, false>, grid, block, st, a);
        return;
    }
    const dim3 grid(a.store_groups), block(tq4::kWave * waves);
    if (a.axes == 1)
        launch(&tq4::rope::append_kernel<LAYOUT, T, KB, VB, kWaves, true>, grid, block, st, a);
    else
        launch(&tq4::rope::append_kernel<LAYOUT, T, KB, VB, kWaves, false>, grid, block, st, a);
    if (a.query)
        launch(&tq4::rope::query_kernel<T>, dim3(query_groups(a, tq4::rope::kQueryWaves)), dim3(tq4::kWave * tq4::rope::kQueryWaves),
               st, a);
}
template <int LAYOUT, class T> void launch_append(tq4::rope::Args &a, int key_bits, int value_bits, hipStream_t st) {
    if (key_bits == 8) {
        constexpr int waves = tq4::store::kFp8Waves, rows = tq4::store::kRows * waves;
        const int64_t n = (int64_t)a.tokens * a.num_kv_heads;
        a.store_groups = (int)std::min<int64_t>((n + rows - 1) / rows, 2048);
        launch(&tq4::rope::append_fp8_kernel<LAYOUT, T>, dim3(a.store_groups + query_groups(a, waves)),
               dim3(tq4::kWave * waves), st, a);
    } else if (key_bits == 4) {
        launch_append<LAYOUT, T, 4, 4>(a, st);
    } else if (value_bits == 4) {
        launch_append<LAYOUT, T, 3, 4>(a, st);
    } else {
        launch_append<LAYOUT, T, 3, 3>(a, st);
    }
}

}  // namespace

extern "C" int tq4_rope_store(const void *query, void *query_out, const void *key, const void *value, int dtype,
                              int64_t query_stride, int64_t key_stride, int64_t value_stride, const int64_t *positions,
                              int64_t axis_stride, int axes, const int32_t *axis_of, const void *cos_sin,
                              int cos_sin_dtype, int table_rows, int rot_dim, int neox, const int32_t *slot_mapping,
                              const float *rot_t, const float *midpoints, const float *centroids, uint8_t *kv_cache,
                              int num_blocks, int N, int Hq, int Hk, int D, int block_size, int64_t cache_block_stride,
                              int layout, int norm_correction, int key_bits, int value_bits, tq4_stream_t stream) {
    constexpr char what[] = "tq4_rope_store";
    const bool fp8 = key_bits == 8 && value_bits == 4;
    if (!fp8 && !preset_supported(key_bits, value_bits))
        return fail(TQ4_E_UNSUPPORTED, "%s: key_bits / value_bits %d / %d unsupported (4/4, 8/4, 3/4, 3/3)", what,
                    key_bits, value_bits);
    if (!key || !value || !positions || !cos_sin || !slot_mapping || !kv_cache || (!query != !query_out) ||
        (!fp8 && (!rot_t || !midpoints)))
        return fail(TQ4_E_INVALID, "%s: null pointer argument", what);
    if (!fp8 && norm_correction && !centroids)
        return fail(TQ4_E_INVALID, "%s: norm_correction requires centroids", what);
    if (dtype != TQ4_F32 && dtype != TQ4_BF16 && dtype != TQ4_F16)
        return fail(TQ4_E_INVALID, "%s: dtype must be 0 (f32), 1 (bf16) or 2 (f16)", what);
    if (cos_sin_dtype != TQ4_F32 && cos_sin_dtype != dtype)
        return fail(TQ4_E_INVALID, "%s: cos_sin_dtype must be 0 (f32) or the keys' type", what);
    if (N < 0 || Hk <= 0 || block_size <= 0 || num_blocks < 0 || table_rows <= 0 || (query && Hq <= 0))
        return fail(TQ4_E_INVALID, "%s: N and num_blocks must be >= 0, head counts, block_size and table_rows positive", what);
    if (D != tq4::kHeadDim)
        return fail(TQ4_E_UNSUPPORTED, "%s: head_dim %d unsupported (128)", what, D);
    if (rot_dim <= 0 || rot_dim > D || rot_dim % 16)
        return fail(TQ4_E_UNSUPPORTED, "%s: rot_dim %d must be a multiple of 16 up to %d", what, rot_dim, D);
    if (axes < 1 || axes > tq4::rope::kMostAxes || (axes > 1 && !axis_of))
        return fail(TQ4_E_INVALID, "%s: axes %d must be 1 to %d, several with axis_of", what, axes, tq4::rope::kMostAxes);
    if (!layout_valid(layout))
        return fail(TQ4_E_INVALID, "%s: " TQ4_LAYOUT_MSG, what);
    const int slot = fp8 ? tq4::store::kFp8Record + 4 : preset_slot_bytes(key_bits, value_bits);
    const int align = fp8 ? 4 : key_bits == 4 ? 16 : 2;
    const int64_t min_stride = (int64_t)block_size * Hk * slot;
    if (cache_block_stride < min_stride || cache_block_stride % align)
        return fail(TQ4_E_INVALID, "%s: requires cache [blocks,%d,%d,%d]: block stride %lld", what, block_size, Hk, slot,
                    (long long)cache_block_stride);
    const int per16 = dtype == TQ4_F32 ? 4 : 8;
    if (!aligned(key, 16) || !aligned(value, 16) || !aligned(query, 16) || !aligned(query_out, 16) ||
        !aligned(cos_sin, 16) || !aligned(kv_cache, align))
        return fail(TQ4_E_INVALID, "%s: query, key, value and cos_sin must be 16-byte aligned, kv_cache %d-byte", what, align);
    if (key_stride % per16 || value_stride % per16 || (query && query_stride % per16) || key_stride < 0 ||
        value_stride < 0 || query_stride < 0)
        return fail(TQ4_E_INVALID, "%s: token strides must be whole 16-byte pieces", what);
    if ((int64_t)N * std::max(Hk, query ? Hq : 0) > INT32_MAX - 4096)
        return fail(TQ4_E_INVALID, "%s: N * heads = %lld rows exceeds the 32-bit row index", what,
                    (long long)N * std::max(Hk, query ? Hq : 0));
    if (N == 0)
        return ok();
    tq4::rope::Args a{};
    a.query = query;
    a.query_out = query_out;
    a.key = key;
    a.value = value;
    a.q_stride = query_stride;
    a.k_stride = key_stride;
    a.v_stride = value_stride;
    a.positions = positions;
    a.axis_stride = axis_stride;
    a.table = cos_sin;
    a.slots = slot_mapping;
    a.pit = rot_t;
    a.midpoints = midpoints;
    a.centroids = centroids;
    a.cache = kv_cache;
    a.block_stride = cache_block_stride;
    a.num_slots = (int64_t)num_blocks * block_size;
    for (int f = 0; axes > 1 && f < rot_dim / 2; ++f) {
        const int x = axis_of[f];
        if (x < 0 || x >= axes)
            return fail(TQ4_E_INVALID, "%s: axis_of[%d] = %d, must be 0 to %d", what, f, x, axes - 1);
        a.axis_bit[0] |= (uint64_t)(x & 1) << f;
        a.axis_bit[1] |= (uint64_t)(x >> 1) << f;
    }
    a.axes = axes;
    a.table_rows = table_rows;
    a.table_f32 = cos_sin_dtype == TQ4_F32;
    a.rot = rot_dim;
    a.neox = neox != 0;
    a.tokens = N;
    a.num_q_heads = query ? Hq : 1;
    a.num_kv_heads = Hk;
    a.block_size = block_size;
    const CacheGeom geom = cache_geom(layout, block_size, Hk, slot);
    a.slot_pos = geom.pos;
    a.slot_head = geom.head;
    a.norm_correction = !fp8 && norm_correction;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    switch (dtype * 2 + geom.kl) {
    case TQ4_F32 * 2 + 0: launch_append<0, float>(a, key_bits, value_bits, st); break;
    case TQ4_F32 * 2 + 1: launch_append<1, float>(a, key_bits, value_bits, st); break;
    case TQ4_BF16 * 2 + 0: launch_append<0, __bf16>(a, key_bits, value_bits, st); break;
    case TQ4_BF16 * 2 + 1: launch_append<1, __bf16>(a, key_bits, value_bits, st); break;
    case TQ4_F16 * 2 + 0: launch_append<0, _Float16>(a, key_bits, value_bits, st); break;
    default: launch_append<1, _Float16>(a, key_bits, value_bits, st); break;
    }
    return launch_status(what);
}
