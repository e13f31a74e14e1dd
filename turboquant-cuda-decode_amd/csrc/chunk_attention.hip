// Attention of several new tokens per sequence (tq4_chunk_attention, include/tq4_decode.h).
#include <algorithm>
#include <cmath>

#include "abi.h"
#include "chunk_few.h"

using namespace tq4::abi;

namespace {

// How a call is spread over the device: workgroups on row tiles of `rows` rows and token tiles of `tile`, `groups` of
// them at once.
enum class Form { kMany, kSome, kFew };
struct ChunkPlan {
    Form form;
    int rows, tile, groups;
    int few;  // sequences with up to this many query rows take kFew in a product of their own (0: none do)
};
int cus() { return step_waves_held() / tq4::xdl::kStepWaves; }
// By a sequence's query rows per kv-head (on average).  Every row tile reads and decodes the sequence again: one of 32, 64
// and 256 rows takes 4 : 7 : 16 parts of a time (64 sequences of 4096 tokens, 8 kv-heads, per row tile 77, 135 and 310 us
// in all), and the least sum is taken: 32, 48, 64, 96, 128 and 256 rows 102, 153, 172, 249, 328, 638 us in tiles of 32, 149, 142,
// 144, 267, 273, 527 in tiles of 64, 304, 295, 298, 303, 310, 349 in tiles of 256.  Up to 16 (sequence, kv-head) pairs,
// whose row tiles are all cut into many parts, those of 32 rows are ahead up to 128 rows (one sequence of 32768
// tokens, 2 kv-heads, 48 and 128 rows: 48 and 55 us, 63 and 72, 64 and 72).
// Batches whose average takes larger tiles may still have sequences with few rows (decoding beside a prompt's chunk), whose
// every tile would cost as much as a full one: they have a product of their own (63 sequences of one token and one of
// 2048, behind 4096: 455 us together, 256 so; a batch without such sequences pays 8 us for it).  The average alone decides: where
// it is small, a long chunk goes through kFew with the rest (256 single tokens and one of 1792, behind 4096: 583 us;
// in two calls 279 and 156).
ChunkPlan chunk_plan(int tokens, int batch, int Hq, int Hk) {
    const int64_t rows = std::max<int64_t>((int64_t)tokens * (Hq / Hk) / batch, 1);
    const int64_t few = 4 * ((rows + 31) / 32), some = 7 * ((rows + 63) / 64), many = 16 * ((rows + 255) / 256);
    if ((few < some && few < many) || ((int64_t)batch * Hk <= 16 && rows <= 128))
        return {Form::kFew, tq4::chunk::kFewRows, tq4::chunk::kFewTile, 2 * cus(), 0};
    if (some < many)
        return {Form::kSome, 64, 64, 2 * cus(), batch > 1 ? 32 : 0};
    return {Form::kMany, 256, 64, cus(), batch > 1 ? 96 : 0};
}

struct Workspace {
    int64_t q_lo, factor, work, cuts, few_work, few_cuts, parts, total;  // offsets in floats
};
Workspace workspace_of(int tokens, int batch, int Hq, int Hk) {
    const int64_t rows = (int64_t)tokens * Hq;
    const ChunkPlan p = chunk_plan(tokens, batch, Hq, Hk);
    auto up = [](int64_t x) { return (x + 63) / 64 * 64; };
    Workspace w{};
    w.q_lo = up(rows * tq4::kHeadDim / 2);
    w.factor = w.q_lo + up(rows * tq4::kHeadDim / 2);
    w.work = w.factor + up(rows);
    w.cuts = w.work + up(2 * ((int64_t)batch + 1));
    w.few_work = w.cuts + up(4 * ((int64_t)p.groups + 1));
    w.few_cuts = w.few_work + (p.few ? up(2 * ((int64_t)batch + 1)) : 0);
    w.parts = w.few_cuts + (p.few ? up(4 * ((int64_t)2 * cus() + 1)) : 0);  // (no less than kFew's; one product after the other)
    w.total = w.parts + up((int64_t)2 * p.groups * p.rows * (tq4::kHeadDim + 1));
    return w;
}
const char *shape_error(int tokens, int B, int Hq, int Hk) {
    if (tokens <= 0 || B <= 0 || Hq <= 0 || Hk <= 0 || Hq % Hk)
        return "tokens, B, Hq and Hk must be positive, Hq a multiple of Hk";
    if ((int64_t)tokens * Hq > 1 << 30)
        return "more than 2^30 query rows";
    return nullptr;
}

template <int LAYOUT, int WR, int WT, int KT, int BUFS, bool FINE>
void launch_chunk(const Stage1Args &a, const tq4::chunk::Args &p, hipStream_t st) {
    const dim3 block(64 * WR * WT), grid((p.groups + 7) / 8 * 8);
    using namespace tq4::chunk;
    if (a.key_fp8)
        launch(&chunk_kernel<LAYOUT, true, false, false, WR, WT, KT, BUFS, FINE>, grid, block, st, p);
    else if (a.key_bits == 3 && a.value_bits == 3)
        launch(&chunk_kernel<LAYOUT, false, true, true, WR, WT, KT, BUFS, FINE>, grid, block, st, p);
    else if (a.key_bits == 3)
        launch(&chunk_kernel<LAYOUT, false, true, false, WR, WT, KT, BUFS, FINE>, grid, block, st, p);
    else
        launch(&chunk_kernel<LAYOUT, false, false, false, WR, WT, KT, BUFS, FINE>, grid, block, st, p);
}
template <int LAYOUT, bool FINE> void launch_few(const Stage1Args &a, const tq4::chunk::Args &p, hipStream_t st) {
    using namespace tq4::chunk;
    const dim3 block(tq4::kWave * kFewWaves), grid((p.groups + 7) / 8 * 8);
    if (a.key_fp8)
        launch(&chunk_few_kernel<LAYOUT, true, false, false, FINE>, grid, block, st, p);
    else if (a.key_bits == 3 && a.value_bits == 3)
        launch(&chunk_few_kernel<LAYOUT, false, true, true, FINE>, grid, block, st, p);
    else if (a.key_bits == 3)
        launch(&chunk_few_kernel<LAYOUT, false, true, false, FINE>, grid, block, st, p);
    else
        launch(&chunk_few_kernel<LAYOUT, false, false, false, FINE>, grid, block, st, p);
}
template <int LAYOUT, bool FINE> void launch_chunk(const Stage1Args &a, const tq4::chunk::Args &p, Form form, hipStream_t st) {
    if (form == Form::kMany)
        launch_chunk<LAYOUT, 8, 1, 64, 2, FINE>(a, p, st);
    else if (form == Form::kSome)
        launch_chunk<LAYOUT, 2, 2, 64, 1, FINE>(a, p, st);
    else
        launch_few<LAYOUT, FINE>(a, p, st);
}
template <bool KF8, bool LO> void launch_start(const tq4::chunk::Args &p, const tq4::chunk::Args &few, int plans, hipStream_t st) {
    using namespace tq4::chunk;
    const int64_t rows = (int64_t)p.tokens * p.num_q_heads;
    const dim3 grid((unsigned)((rows + kStartRows - 1) / kStartRows + plans)), block(kStartThreads);
    if (p.q_dtype == TQ4_BF16)
        launch(&chunk_start_kernel<__bf16, KF8, LO>, grid, block, st, p, few, plans);
    else
        launch(&chunk_start_kernel<_Float16, KF8, LO>, grid, block, st, p, few, plans);
}
template <typename OutT> void launch_merge(const tq4::chunk::Args &p, hipStream_t st) {
    using namespace tq4::chunk;
    constexpr int rows = kMergeHalves * kMergePer;
    launch(&chunk_merge_kernel<OutT>, dim3((p.shape.rows + rows - 1) / rows, p.groups), dim3(kMergeThreads), st, p);
}

}  // namespace

extern "C" {

int64_t tq4_chunk_workspace_floats(int tokens, int B, int Hq, int Hk) {
    if (const char *why = shape_error(tokens, B, Hq, Hk)) {
        fail(TQ4_E_INVALID, "tq4_chunk_workspace_floats: %s", why);
        return -1;
    }
    return workspace_of(tokens, B, Hq, Hk).total;
}

int tq4_chunk_attention(const void *query, int query_dtype, int64_t query_stride, const float *rot_t,
                        const float *centroids, const uint8_t *kv_cache, const int32_t *block_table,
                        const int32_t *seq_lens, const int32_t *query_starts, float *workspace, int64_t workspace_floats,
                        void *out, int out_dtype, float *lse, int tokens, int B, int Hq, int Hk, int D, int block_size,
                        int max_blocks_per_seq, int64_t cache_block_stride, int layout, float attn_scale,
                        const float *sinks, int key_bits, int value_bits, int causal, int window, int first_tokens,
                        tq4_stream_t stream) {
    constexpr char what[] = "tq4_chunk_attention";
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    Stage1Args a{};
    // (the log-sum-exp may be left out: another pointer stands in for it in the common checks)
    int rc = span_args(a, what, query, query_dtype, rot_t, centroids, kv_cache, block_table, seq_lens, workspace, workspace,
                       out, out_dtype, workspace, B, Hq, Hk, D, block_size, max_blocks_per_seq, cache_block_stride, 1,
                       layout, attn_scale, sinks, key_bits, value_bits);
    if (rc)
        return rc;
    if (const char *why = shape_error(tokens, B, Hq, Hk))
        return fail(TQ4_E_INVALID, "%s: %s", what, why);
    if (!query_starts)
        return fail(TQ4_E_INVALID, "%s: null pointer argument", what);
    if (query_dtype == TQ4_F32 || out_dtype == TQ4_F32)
        return fail(TQ4_E_UNSUPPORTED, "%s: 16-bit queries and outputs only (the products have f16 operands)", what);
    if (query_stride < (int64_t)Hq * D || query_stride % 8)
        return fail(TQ4_E_INVALID, "%s: query_stride %lld must be whole 16-byte pieces, at least Hq * D", what,
                    (long long)query_stride);
    if (cache_block_stride > 0x7FFFFFFF)
        return fail(TQ4_E_UNSUPPORTED, "%s: block stride %lld above 2^31 - 1", what, (long long)cache_block_stride);
    if (!aligned(out, 16))
        return fail(TQ4_E_INVALID, "%s: out must be 16-byte aligned", what);
    if (!(attn_scale < INFINITY))
        return fail(TQ4_E_INVALID, "%s: attn_scale must be finite", what);
    if (window < 0 || first_tokens < 0 || (window > 0 && !causal))
        return fail(TQ4_E_INVALID, "%s: window (%d) and first_tokens (%d) must be at least 0, a window only with causal", what,
                    window, first_tokens);
    const Workspace ws = workspace_of(tokens, B, Hq, Hk);
    if (workspace_floats < ws.total || !aligned(workspace, 16))
        return fail(TQ4_E_INVALID, "%s: workspace of %lld floats, needs %lld, 16-byte aligned", what,
                    (long long)workspace_floats, (long long)ws.total);
    const ChunkPlan plan = chunk_plan(tokens, B, Hq, Hk);
    tq4::chunk::Args p{};
    p.query = query;
    p.rot_t = rot_t;
    p.centroids = centroids;
    p.cache = kv_cache;
    p.pages = block_table;
    p.seq_lens = seq_lens;
    p.starts = query_starts;
    p.sinks = sinks;
    p.out = out;
    p.lse = lse;
    p.q_hi = reinterpret_cast<_Float16 *>(workspace);
    p.q_lo = reinterpret_cast<_Float16 *>(workspace + ws.q_lo);
    p.q_factor = workspace + ws.factor;
    p.work = reinterpret_cast<double *>(workspace + ws.work);
    p.cuts = reinterpret_cast<tq4::chunk::Cut *>(workspace + ws.cuts);
    p.parts = workspace + ws.parts;
    p.block_stride = cache_block_stride;
    p.query_stride = query_stride;
    p.score_scale_log2 = attn_scale * tq4::kLog2e;
    p.q_dtype = query_dtype;
    p.out_dtype = out_dtype;
    p.num_q_heads = Hq;
    p.num_kv_heads = Hk;
    p.tokens = tokens;
    p.batch = B;
    p.table_width = max_blocks_per_seq;
    p.groups = plan.groups;
    p.block_size_log2 = log2_int(block_size);
    const int record = 16 * (key_bits + value_bits);  // SoA: bytes of codes
    p.slot_pos = a.kl == 0 ? Hk * record : a.slot_pos;
    p.slot_head = a.kl == 0 ? record : a.slot_head;
    p.shape = tq4::chunk::Shape{plan.rows, plan.tile, Hq / Hk, Hk, causal != 0, std::min(window, 1 << 30), std::min(first_tokens, 1 << 30)};
    p.longest = (int)std::min<int64_t>((int64_t)max_blocks_per_seq * block_size, (1 << 30));
    p.rows_most = 0x7FFFFFFF;
    tq4::chunk::Args few = p;
    if (plan.few) {
        p.rows_least = plan.few + 1;
        few.rows_most = plan.few;
        few.shape.rows = tq4::chunk::kFewRows;
        few.shape.tile = tq4::chunk::kFewTile;
        few.groups = 2 * cus();
        few.work = reinterpret_cast<double *>(workspace + ws.few_work);
        few.cuts = reinterpret_cast<tq4::chunk::Cut *>(workspace + ws.few_cuts);
    }
    const bool fine = lse || out_dtype == TQ4_F16;
    const int plans = plan.few ? 2 : 1;
    if (a.key_fp8)
        launch_start<true, false>(p, few, plans, st);
    else
        fine ? launch_start<false, true>(p, few, plans, st) : launch_start<false, false>(p, few, plans, st);
    rc = launch_status("chunk start");
    auto product = [&](const tq4::chunk::Args &p, Form form) {
        if (a.kl == 0)
            fine ? launch_chunk<0, true>(a, p, form, st) : launch_chunk<0, false>(a, p, form, st);
        else
            fine ? launch_chunk<1, true>(a, p, form, st) : launch_chunk<1, false>(a, p, form, st);
        if (const int rc = launch_status("chunk"))
            return rc;
        out_dtype == TQ4_BF16 ? launch_merge<__bf16>(p, st) : launch_merge<_Float16>(p, st);
        return launch_status("chunk merge");
    };
    if (!rc && plan.few)
        rc = product(few, Form::kFew);
    return rc ? rc : product(p, plan.form);
}

}  // extern "C"
