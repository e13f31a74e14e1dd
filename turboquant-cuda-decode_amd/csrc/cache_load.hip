// Keys and values out of the cache (tq4_cache_load) and attention results joined (tq4_merge_states), include/tq4_decode.h.
#include <algorithm>

#include "abi.h"
#include "load.h"

using namespace tq4::abi;

namespace {

template <int LAYOUT, bool KF8, bool KB3, bool V3, typename T>
void launch_load(const tq4::load::Args &p, dim3 grid, hipStream_t st) {
    const dim3 block(tq4::load::kThreads);
    if constexpr (!KF8)
        if (p.rot_t) {
            launch(&tq4::load::load_kernel<LAYOUT, KF8, KB3, V3, T, true>, grid, block, st, p);
            return;
        }
    launch(&tq4::load::load_kernel<LAYOUT, KF8, KB3, V3, T, false>, grid, block, st, p);
}
template <int LAYOUT, typename T>
void launch_load(int key_bits, int value_bits, const tq4::load::Args &p, dim3 grid, hipStream_t st) {
    if (key_bits == 8)
        launch_load<LAYOUT, true, false, false, T>(p, grid, st);
    else if (key_bits == 4)
        launch_load<LAYOUT, false, false, false, T>(p, grid, st);
    else if (value_bits == 4)
        launch_load<LAYOUT, false, true, false, T>(p, grid, st);
    else
        launch_load<LAYOUT, false, true, true, T>(p, grid, st);
}
template <typename T>
void launch_load(int kl, int key_bits, int value_bits, const tq4::load::Args &p, dim3 grid, hipStream_t st) {
    kl == 0 ? launch_load<0, T>(key_bits, value_bits, p, grid, st) : launch_load<1, T>(key_bits, value_bits, p, grid, st);
}
// Whether [p, p + n) and [q, q + m) share bytes.
bool overlap(const void *p, int64_t n, const void *q, int64_t m) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q);
    return a < b + (uintptr_t)m && b < a + (uintptr_t)n;
}

}  // namespace

extern "C" {

int tq4_cache_load(const uint8_t *kv_cache, const int32_t *slot_mapping, const float *rot_t, const float *centroids,
                   void *key, void *value, int dtype, int num_blocks, int N, int Hk, int D, int block_size,
                   int64_t cache_block_stride, int layout, int key_bits, int value_bits, tq4_stream_t stream) {
    constexpr char what[] = "tq4_cache_load";
    const bool fp8 = key_bits == 8 && value_bits == 4;
    if (!fp8 && !preset_supported(key_bits, value_bits))
        return fail(TQ4_E_UNSUPPORTED, "%s: key_bits / value_bits %d / %d unsupported (4/4, 8/4, 3/4, 3/3)", what, key_bits,
                    value_bits);
    if (!kv_cache || !slot_mapping || !key || !value || (!fp8 && !centroids))
        return fail(TQ4_E_INVALID, "%s: null pointer argument", what);
    if (dtype != TQ4_F32 && dtype != TQ4_BF16 && dtype != TQ4_F16)
        return fail(TQ4_E_INVALID, "%s: dtype must be 0 (f32), 1 (bf16) or 2 (f16)", what);
    if (N <= 0 || Hk <= 0 || block_size <= 0 || num_blocks <= 0)
        return fail(TQ4_E_INVALID, "%s: N, Hk, block_size and num_blocks must be positive", what);
    if (D != tq4::kHeadDim)
        return fail(TQ4_E_UNSUPPORTED, "%s: head_dim %d unsupported (kernels are built for 128)", what, D);
    if (!layout_valid(layout))
        return fail(TQ4_E_INVALID, "%s: " TQ4_LAYOUT_MSG, what);
    const int slot = fp8 ? tq4::store::kFp8Record + 4 : preset_slot_bytes(key_bits, value_bits);
    const int64_t least = (int64_t)block_size * Hk * slot;
    if (cache_block_stride < least || cache_block_stride % 2)
        return fail(TQ4_E_INVALID, "%s: requires cache [blocks,%d,%d,%d]: block stride %lld < %lld, or odd", what, block_size,
                    Hk, slot, (long long)cache_block_stride, (long long)least);
    if ((int64_t)N * Hk > 1 << 30 || least > 1 << 30)
        return fail(TQ4_E_UNSUPPORTED, "%s: N * Hk and a block's bytes may be 2^30 at most", what);
    if (!aligned(kv_cache, 2) || !aligned(key, 16) || !aligned(value, 16))
        return fail(TQ4_E_INVALID, "%s: kv_cache must be 2-byte aligned, key and value 16-byte aligned", what);
    const int64_t out_bytes = (int64_t)N * Hk * D * (dtype == TQ4_F32 ? 4 : 2);
    const int64_t cache_bytes = (num_blocks - 1) * cache_block_stride + least;
    if (overlap(key, out_bytes, value, out_bytes) || overlap(key, out_bytes, kv_cache, cache_bytes) ||
        overlap(value, out_bytes, kv_cache, cache_bytes))
        return fail(TQ4_E_INVALID, "%s: key, value and kv_cache must not overlap", what);
    const CacheGeom geom = cache_geom(layout, block_size, Hk, slot);
    tq4::load::Args p{};
    p.cache = kv_cache;
    p.slots = slot_mapping;
    p.rot_t = fp8 ? nullptr : rot_t;
    p.centroids = centroids;
    p.key = key;
    p.value = value;
    p.block_stride = cache_block_stride;
    p.num_slots = (int64_t)num_blocks * block_size;
    p.rows = N * Hk;
    p.num_kv_heads = Hk;
    p.block_size = block_size;
    p.slot_pos = geom.pos;
    p.slot_head = geom.head;
    const int cus = step_waves_held() / tq4::xdl::kStepWaves;
    const int64_t tiles = (p.rows + tq4::load::kRows - 1) / tq4::load::kRows;
    const int per_cu = p.rot_t ? (dtype == TQ4_BF16 ? 4 : 2) : 8;
    const dim3 grid((unsigned)std::min<int64_t>((tiles + tq4::load::kWaves - 1) / tq4::load::kWaves, (int64_t)cus * per_cu));
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (dtype == TQ4_F32)
        launch_load<float>(geom.kl, key_bits, value_bits, p, grid, st);
    else if (dtype == TQ4_BF16)
        launch_load<__bf16>(geom.kl, key_bits, value_bits, p, grid, st);
    else
        launch_load<_Float16>(geom.kl, key_bits, value_bits, p, grid, st);
    return launch_status("cache_load");
}

int tq4_merge_states(const void *out_a, const float *lse_a, const void *out_b, const float *lse_b, void *out, int dtype,
                     float *lse, int64_t rows, int D, tq4_stream_t stream) {
    constexpr char what[] = "tq4_merge_states";
    if (!out_a || !lse_a || !out_b || !lse_b || !out || !lse)
        return fail(TQ4_E_INVALID, "%s: null pointer argument", what);
    if (dtype != TQ4_F32 && dtype != TQ4_BF16 && dtype != TQ4_F16)
        return fail(TQ4_E_INVALID, "%s: dtype must be 0 (f32), 1 (bf16) or 2 (f16)", what);
    if (rows <= 0)
        return fail(TQ4_E_INVALID, "%s: rows must be positive", what);
    if (D != tq4::kHeadDim)
        return fail(TQ4_E_UNSUPPORTED, "%s: head_dim %d unsupported (128)", what, D);
    if (!aligned(out_a, 16) || !aligned(out_b, 16) || !aligned(out, 16))
        return fail(TQ4_E_INVALID, "%s: out_a, out_b and out must be 16-byte aligned", what);
    constexpr int64_t per = tq4::load::kThreads / 16 * tq4::load::kJoinRows;  // rows of a workgroup
    if (rows > per * 0x7FFFFFFF)
        return fail(TQ4_E_UNSUPPORTED, "%s: %lld rows are too many", what, (long long)rows);
    const int64_t bytes = rows * D * (dtype == TQ4_F32 ? 4 : 2);
    // in place is fine, partly is not
    const bool shifted = (out != out_a && overlap(out, bytes, out_a, bytes)) || (out != out_b && overlap(out, bytes, out_b, bytes)) ||
                         (lse != lse_a && overlap(lse, 4 * rows, lse_a, 4 * rows)) ||
                         (lse != lse_b && overlap(lse, 4 * rows, lse_b, 4 * rows));
    const bool mixed = overlap(out, bytes, lse, 4 * rows) || overlap(out, bytes, lse_a, 4 * rows) ||
                       overlap(out, bytes, lse_b, 4 * rows) || overlap(lse, 4 * rows, out_a, bytes) ||
                       overlap(lse, 4 * rows, out_b, bytes);
    if (shifted || mixed)
        return fail(TQ4_E_INVALID, "%s: outputs may be one of the inputs, but not overlap them otherwise", what);
    const dim3 grid((unsigned)((rows + per - 1) / per)), block(tq4::load::kThreads);
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    auto go = [&](auto zero) {
        using T = decltype(zero);
        launch(&tq4::load::join_states_kernel<T>, grid, block, st, static_cast<const T *>(out_a), lse_a,
               static_cast<const T *>(out_b), lse_b, static_cast<T *>(out), lse, rows);
    };
    if (dtype == TQ4_F32)
        go(0.f);
    else if (dtype == TQ4_BF16)
        go((__bf16)0.f);
    else
        go((_Float16)0.f);
    return launch_status("merge_states");
}

}  // extern "C"
