// Decode steps whose sequences have hidden tokens (include/tq4_decode.h): the sliding window with first
// tokens that stay visible, and the launch that prefix_decode.hip runs the sequences' own tails with.
#include <algorithm>

#include "step_launch.h"

using namespace tq4::abi;

int tq4::abi::launch_hidden_step(const Stage1Args &a, const StepIo &io, const StepPlan &plan,
                                 const tq4::xdl::Hidden &hidden, hipStream_t st) {
    return launch_step_by<true>(a, io, plan, hidden, st);
}

extern "C" int tq4_window_decode(const void *query, int query_dtype, const float *rot_t, const float *centroids,
                                 const uint8_t *kv_cache, const int32_t *block_table, const int32_t *seq_lens,
                                 float *q_rot_ws, float *mid_o, void *out, int out_dtype, float *lse, int B, int Hq,
                                 int Hk, int D, int block_size, int max_blocks_per_seq, int64_t cache_block_stride,
                                 int num_kv_splits, int layout, float attn_scale, const float *sinks, int key_bits,
                                 int value_bits, int window, int first_tokens, tq4_stream_t stream) {
    constexpr char what[] = "tq4_window_decode";
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    Stage1Args a{};
    int rc = span_args(a, what, query, query_dtype, rot_t, centroids, kv_cache, block_table, seq_lens, q_rot_ws, mid_o,
                       out, out_dtype, lse, B, Hq, Hk, D, block_size, max_blocks_per_seq, cache_block_stride,
                       num_kv_splits, layout, attn_scale, sinks, key_bits, value_bits);
    if (rc)
        return rc;
    if (window < 1 || first_tokens < 0)
        return fail(TQ4_E_INVALID, "%s: window (%d) must be at least 1, first_tokens (%d) at least 0", what, window,
                    first_tokens);
    // no sequence has more visible tiles than the two runs of tokens can touch
    const int64_t most = (int64_t)first_tokens + window + 30;
    const int blocks = (int)std::min<int64_t>(max_blocks_per_seq, (most + block_size - 1) / block_size);
    const StepPlan plan = step_plan(a, blocks, num_kv_splits > 1);
    rc = launch_step_by<true>(a, StepIo{query, query_dtype, rot_t, q_rot_ws, centroids, out, out_dtype, lse}, plan,
                              tq4::xdl::Hidden{first_tokens, window, 0}, st);
    if (rc || plan.whole)
        return rc;
    return merge_parts(mid_o, seq_lens, out, out_dtype, lse, B, Hq, num_kv_splits, (plan.nx + B - 1) / B, st);
}
