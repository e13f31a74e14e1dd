// What the translation units of the C ABI share: error text, launches, argument checks of the
// attention entries, and the step's launch plan.
#pragma once
#include <hip/hip_runtime.h>
#include <hip/hip_ext.h>
#include <atomic>
#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "../../include/tq4_decode.h"
#include "step.h"
#include "store.h"

namespace tq4 {
namespace abi {

inline thread_local char g_err[512] = "";

// Events the next kernel launch of this thread stamps with its own start and end
// (tq4_time_next_launch); cleared by that launch.
inline thread_local hipEvent_t g_time_start = nullptr, g_time_stop = nullptr;

// Every kernel launch goes through here: arguments are converted to the kernel's
// parameter types (the event-stamping launch passes them by address).
template <typename... KArgs, typename... Args>
void launch_lds(void (*kernel)(KArgs...), dim3 grid, dim3 block, int lds_bytes, hipStream_t st, Args... args) {
    static_assert(sizeof...(KArgs) == sizeof...(Args), "argument count");
    if (g_time_start || g_time_stop) {
        const hipEvent_t a = g_time_start, b = g_time_stop;
        g_time_start = g_time_stop = nullptr;
        hipExtLaunchKernelGGL(kernel, grid, block, lds_bytes, st, a, b, 0, static_cast<KArgs>(args)...);
    } else {
        hipLaunchKernelGGL(kernel, grid, block, lds_bytes, st, static_cast<KArgs>(args)...);
    }
}
template <typename... KArgs, typename... Args>
void launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, hipStream_t st, Args... args) {
    launch_lds(kernel, grid, block, 0, st, args...);
}

inline int fail(int code, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof g_err, fmt, ap);
    va_end(ap);
    return code;
}

inline int ok() {
    g_err[0] = '\0';
    return TQ4_OK;
}

inline int launch_status(const char *what) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess)
        return fail((int)e, "%s launch failed: %s", what, hipGetErrorString(e));
    return ok();
}

inline bool aligned(const void *p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

inline int log2_int(int x) {
    int r = 0;
    while ((1 << r) < x)
        ++r;
    return r;
}

struct Stage1Args {
    const float *q_rot;
    const uint8_t *cache;
    const int32_t *bt;
    const int32_t *seq_lens;
    const float *lut;
    float *mid_o;
    int B, Hq, Hk, D, bs, max_blocks;
    int64_t stride;
    int S, layout;  // TQ4_LAYOUT_*
    float scale;
    const float *sinks = nullptr;  // [Hq] sink logits of split 0, or null
    bool key_fp8 = false;  // the FP8-key preset (VALU kernel; pair LUT unused)
    // > 0: the key_bits / value_bits preset on the VALU kernel; lut holds the 2^key_bits
    // centroids (not the pair LUT)
    int key_bits = 0, value_bits = 4;
    // filled by check_stage1: kernel layout (0 SoA, 1 AoS) and the AoS slot strides
    int kl = 0, slot_pos = 0, slot_head = 0;
};

// Kernel layout (0 SoA, 1 AoS) of an ABI layout id and the byte offsets of AoS slot (t, h)
// inside a block, t * pos + h * head: position-major blocks [bs][Hk][slot] (TQ4_LAYOUT_AOS)
// or head-major blocks [Hk][bs][slot] (TQ4_LAYOUT_AOS_HEAD_MAJOR, the layout the vLLM
// backend's [blocks, Hk, bs, slot] cache presents through transpose(1, 2),
// reference/turboquant_attn.py:536, :565).  SoA blocks are addressed by their own layout.
struct CacheGeom {
    int kl, pos, head;
};
inline bool layout_valid(int layout) {
    return layout == TQ4_LAYOUT_SOA || layout == TQ4_LAYOUT_AOS || layout == TQ4_LAYOUT_AOS_HEAD_MAJOR;
}
inline CacheGeom cache_geom(int layout, int bs, int hk, int slot) {
    if (layout == TQ4_LAYOUT_AOS_HEAD_MAJOR)
        return {1, slot, bs * slot};
    return {layout == TQ4_LAYOUT_AOS ? 1 : 0, hk * slot, slot};
}
#define TQ4_LAYOUT_MSG "layout must be 0 (SoA), 1 (AoS) or 2 (AoS, head-major blocks)"

// Bytes of one AoS slot (= SoA bytes per (token, kv-head)) of a key_bits / value_bits preset.
inline int preset_slot_bytes(int key_bits, int value_bits) {
    const int raw = 16 * key_bits + 2 + 16 * value_bits + 4;
    return raw + raw % 2;
}

inline bool preset_supported(int key_bits, int value_bits) {
    return (key_bits == 4 && value_bits == 4) || (key_bits == 3 && (value_bits == 3 || value_bits == 4));
}
static_assert(tq4::kOutF32 == TQ4_F32 && tq4::kOutBf16 == TQ4_BF16 && tq4::kOutF16 == TQ4_F16,
              "output type ids");

inline int check_stage1(Stage1Args &a) {
    if (!a.q_rot || !a.cache || !a.bt || !a.seq_lens || (!a.lut && !a.key_fp8) || !a.mid_o)
        return fail(TQ4_E_INVALID, "tq4_stage1: null pointer argument");
    if (a.B <= 0 || a.Hq <= 0 || a.Hk <= 0 || a.S <= 0 || a.bs <= 0 || a.max_blocks <= 0)
        return fail(TQ4_E_INVALID, "tq4_stage1: B, Hq, Hk, num_kv_splits, block_size and "
                                   "max_blocks_per_seq must be positive");
    if (a.Hq % a.Hk)
        return fail(TQ4_E_INVALID, "tq4_stage1: Hq (%d) must be a multiple of Hk (%d)", a.Hq, a.Hk);
    if (a.S > 65536)
        return fail(TQ4_E_UNSUPPORTED, "tq4_stage1: num_kv_splits %d above 65536", a.S);
    if (a.B > 65535)  // a grid dimension
        return fail(TQ4_E_UNSUPPORTED, "tq4_stage1: batch %d above 65535", a.B);
    if (a.D != tq4::kHeadDim)
        return fail(TQ4_E_UNSUPPORTED, "tq4_stage1: head_dim %d unsupported (kernels are built for 128)", a.D);
    if (!layout_valid(a.layout))
        return fail(TQ4_E_INVALID, "tq4_stage1: " TQ4_LAYOUT_MSG);
    const int slot = a.key_fp8 ? tq4::store::kFp8Record + 4
                               : (a.key_bits > 0 ? preset_slot_bytes(a.key_bits, a.value_bits) : tq4::kAosSlot);
    const int64_t min_stride = (int64_t)a.bs * a.Hk * slot;
    if (a.stride < min_stride || a.stride % 2)
        return fail(TQ4_E_INVALID, "tq4_stage1: requires cache [blocks,%d,%d,%d]: block stride %lld < %lld",
                    a.bs, a.Hk, slot, (long long)a.stride, (long long)min_stride);
    if (!aligned(a.cache, 16) || !aligned(a.q_rot, 16) || !aligned(a.mid_o, 4))
        return fail(TQ4_E_INVALID, "tq4_stage1: kv_cache and q_rot must be 16-byte aligned");
    if (!(a.scale > 0.f) || a.scale != a.scale)
        return fail(TQ4_E_INVALID, "tq4_stage1: attn_scale must be positive");
    const CacheGeom geom = cache_geom(a.layout, a.bs, a.Hk, slot);
    a.kl = geom.kl;
    a.slot_pos = geom.pos;
    a.slot_head = geom.head;
    return TQ4_OK;
}

// q-heads per wave of the 16x16x32 kernel (4 for GQA groups up to 4, else 8) and the waves
// (parts) each kv-head's group takes.
inline int xdl_heads(const Stage1Args &a) { return a.Hq / a.Hk <= 4 ? 4 : 8; }
inline int xdl_parts(const Stage1Args &a) {
    const int g = a.Hq / a.Hk, h = xdl_heads(a);
    return (g + h - 1) / h;
}

// Every GQA group: groups up to 4 on 4-head waves (1, 2 and 3 with padding heads: each KV
// tile is still read and looked up once per wave, so MHA and GQA-2 take about the headline's
// time, 1.4-1.5x faster than the VALU kernel), larger ones in parts of 8 heads (6: one part
// with two padding heads; 16: two parts).
inline bool mfma_applies(const Stage1Args &a) {
    const bool pow2 = a.bs >= 16 && (a.bs & (a.bs - 1)) == 0;
    return pow2 && a.stride % 16 == 0;
}

// ---- The full decode step on the 16x16x32 kernel (decode_step_kernel, step.h) ------------
struct StepIo {
    const void *query;
    int query_dtype;
    const float *rot_t;    // null with FP8 keys
    float *q_rot_ws;
    const float *centroids;
    void *out;
    int out_dtype;
    float *lse;
    bool rotated = false;  // q_rot_ws holds the rotated query rows already
};

// Waves the device holds at once: every kernel of the step is built for two per SIMD.
inline int step_waves_held() {
    static std::atomic<int> held{0};
    int h = held.load(std::memory_order_relaxed);
    if (!h) {
        int dev = 0, cus = 0;
        if (hipGetDevice(&dev) != hipSuccess ||
            hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0)
            cus = 256;
        h = cus * tq4::xdl::kStepWaves;
        held.store(h, std::memory_order_relaxed);
    }
    return h;
}

using tq4::xdl::StepPlan;
// max_blocks: the blocks of the longest sequence that the step may have to read.
inline StepPlan step_plan(const Stage1Args &a, int max_blocks, bool have_parts) {
    const bool whole_lines = a.kl == 0 && !a.key_fp8 && a.key_bits == 0;
    return tq4::xdl::step_plan(
        {step_waves_held(), a.Hk * xdl_parts(a), a.B, max_blocks, a.bs, a.S, whole_lines}, have_parts);
}

// Checks of a full step's own arguments (the rest is check_stage1's).
inline int check_step(const char *what, const void *query, int query_dtype, int out_dtype) {
    if (query_dtype != TQ4_F32 && query_dtype != TQ4_BF16 && query_dtype != TQ4_F16)
        return fail(TQ4_E_INVALID, "%s: query_dtype must be 0, 1 or 2", what);
    if (out_dtype != TQ4_F32 && out_dtype != TQ4_BF16 && out_dtype != TQ4_F16)
        return fail(TQ4_E_INVALID, "%s: out_dtype must be 0 (f32), 1 (bf16) or 2 (f16)", what);
    if (!aligned(query, 16))
        return fail(TQ4_E_INVALID, "%s: query must be 16-byte aligned", what);
    return TQ4_OK;
}

// Arguments of the decode entries that run on the 16x16x32 kernel alone (hidden tokens): `a` filled and
// checked.  key_bits / value_bits 4/4, 3/4, 3/3, or 8/4 for FP8 keys, whose query is used unrotated.
inline int span_args(Stage1Args &a, const char *what, const void *query, int query_dtype, const float *rot_t,
                     const float *centroids, const uint8_t *kv_cache, const int32_t *block_table,
                     const int32_t *seq_lens, float *q_rot_ws, float *mid_o, void *out, int out_dtype, float *lse,
                     int B, int Hq, int Hk, int D, int block_size, int max_blocks, int64_t stride, int num_kv_splits,
                     int layout, float attn_scale, const float *sinks, int key_bits, int value_bits) {
    const bool fp8 = key_bits == 8 && value_bits == 4;
    if (!fp8 && !preset_supported(key_bits, value_bits))
        return fail(TQ4_E_UNSUPPORTED, "%s: key_bits / value_bits %d / %d unsupported (4/4, 8/4, 3/4, 3/3)", what,
                    key_bits, value_bits);
    if (!query || !out || !lse || !q_rot_ws || (!fp8 && (!rot_t || !centroids)))
        return fail(TQ4_E_INVALID, "%s: null pointer argument", what);
    a = Stage1Args{q_rot_ws, kv_cache, block_table, seq_lens, centroids, mid_o, B, Hq, Hk, D, block_size, max_blocks,
                   stride, num_kv_splits, layout, attn_scale, sinks};
    a.key_fp8 = fp8;
    a.key_bits = key_bits == 3 ? 3 : 0;
    a.value_bits = value_bits;
    int rc = check_step(what, query, query_dtype, out_dtype);
    if (rc == TQ4_OK)
        rc = check_stage1(a);
    if (rc)
        return rc;
    if (!mfma_applies(a))
        return fail(TQ4_E_UNSUPPORTED, "%s: needs a power-of-two block_size >= 16 and a 16-byte block stride", what);
    return TQ4_OK;
}

// Entries of tq4_decode.hip that the other units launch through.
int rotate_query(const void *query, int query_dtype, const float *rot_t, float *q_rot, int rows, int D,
                 const float *centroids, float *pair_lut, hipStream_t st);
int merge_parts(const float *parts, const int32_t *seq_lens, void *out, int out_dtype, float *lse, int B, int Hq,
                int num_splits, int64_t expected_parts, hipStream_t st);
int run_step(const Stage1Args &a, const StepIo &io, bool have_parts, hipStream_t st);
// And of span_decode.hip: launch_step_by (step_launch.h) with hidden tokens.
int launch_hidden_step(const Stage1Args &a, const StepIo &io, const StepPlan &plan, const tq4::xdl::Hidden &hidden,
                       hipStream_t st);

}  // namespace abi
}  // namespace tq4
