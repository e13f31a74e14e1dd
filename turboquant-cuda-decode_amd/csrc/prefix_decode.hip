// The decode step of a batch that shares its first tokens (tq4_prefix_decode, include/tq4_decode.h).
#include <algorithm>

#include "abi.h"
#include "prefix.h"

using namespace tq4::abi;

namespace {

// How the prefix is spread over the device: `wr` waves of 32 rows per workgroup (4 with two waves each, or
// 2 up to 64 rows, which four would leave half empty), row tiles of 32 wr rows, `splits` runs of tiles.
struct PrefixPlan {
    int wr, row_tiles, tiles, splits;
    int64_t in_turn;  // tiles that the busiest place works through
};
constexpr int kMaxSplits = 64;  // part rows of the prefix per (sequence, head)

int rows_waves(int64_t rows) { return rows > 64 ? 4 : 2; }
int tile_tokens(int wr) { return wr == 4 ? 64 : 32; }
// workgroups the device holds at once: one of eight waves or four of two per CU
int groups_held(int wr) { return step_waves_held() / tq4::xdl::kStepWaves * (wr == 4 ? 1 : 4); }
int most_splits(int wr, int64_t groups) {
    return (int)std::max<int64_t>(1, std::min<int64_t>(kMaxSplits, 2 * groups_held(wr) / std::max<int64_t>(groups, 1)));
}
// rows: query rows per kv-head.  Of the split counts the one whose rounds of workgroups end first, a
// workgroup's start and end counted as kStart tiles.
PrefixPlan prefix_plan(int rows, int Hk, int tokens) {
    constexpr int kStart = 3;
    PrefixPlan p{};
    p.wr = rows_waves(rows);
    p.row_tiles = (rows + 32 * p.wr - 1) / (32 * p.wr);
    p.tiles = (tokens + tile_tokens(p.wr) - 1) / tile_tokens(p.wr);
    const int64_t groups = (int64_t)p.row_tiles * Hk, held = groups_held(p.wr);
    int64_t best = INT64_MAX;
    for (int s = 1; s <= std::min(most_splits(p.wr, groups), p.tiles); ++s) {
        const int64_t cost = ((groups * s + held - 1) / held) * ((p.tiles + s - 1) / s + kStart);
        if (cost < best) {
            best = cost;
            p.splits = s;
            p.in_turn = ((groups * s + held - 1) / held) * ((p.tiles + s - 1) / s);
        }
    }
    return p;
}

// Whether reading the prefix once is worth its launches.  In microseconds: the step on its own decodes a
// million (token, kv-head) pairs in 19 (waves of four query heads) or 23 (of eight), 3-bit keys in a fifth more, and
// starts in 15; the shared way takes 30 for its four launches, 2.3 per tile in turn, and writes and reads a
// part row of 516 bytes per query row and split.
// Measured (32 / 8 heads, 4-bit keys, tails of 100): batch 8, prefix 2048 36.8 against 17.8 for the step alone,
// 16 x 8192 49 : 36, 64 x 2048 48 : 37, 8 x 32768 66 : 54; 64 x 4096 52 : 56, 32 x 8192 51 : 55,
// 16 x 32768 69 : 94, 64 x 8192 59 : 94.  16 / 2 heads 64 x 8192 49 : 43; 8 / 8 heads 64 x 4096 45 : 56,
// 16 x 8192 39 : 35; 32 / 32 heads 64 x 2048 60 : 97; 32 / 4 heads, 3-bit, 100 x 4000 56 : 58.
// (40 / 8 heads, FP8 keys, 12 x 16384 46 : 49, where it takes the steps.)
bool sharing_pays(const Stage1Args &a, const PrefixPlan &p, int prefix_len) {
    const double each = (xdl_heads(a) == 4 ? 19e-6 : 23e-6) * (a.key_bits == 3 ? 1.2 : 1.0);
    const double alone = 15 + each * a.B * (double)prefix_len * a.Hk * xdl_parts(a);
    const double shared = 30 + 2.3 * p.in_turn + 2.06e-4 * a.B * (double)a.Hq * p.splits;
    return shared < alone;
}

int64_t part_floats(int64_t rows, int parts) { return rows * parts * (tq4::kHeadDim + 1); }

struct Workspace {
    int64_t q_rot, own, shared, total;  // offsets in floats
};
Workspace workspace_of(int B, int Hq, int Hk, int num_kv_splits) {
    const int64_t rows = (int64_t)B * Hq;
    const int wr = rows_waves(rows / Hk);
    const int parts = most_splits(wr, (rows / Hk + 32 * wr - 1) / (32 * wr) * Hk);
    auto up = [](int64_t x) { return (x + 63) / 64 * 64; };
    Workspace w{};
    w.own = up(rows * tq4::kHeadDim);
    w.shared = w.own + up(part_floats(rows, num_kv_splits));
    w.total = w.shared + up(part_floats(rows, parts));
    return w;
}

template <int LAYOUT, int WR, int WT, bool PLO>
void launch_prefix(const Stage1Args &a, const tq4::prefix::Args &p, dim3 grid, hipStream_t st) {
    const dim3 block(64 * WR * WT);
    if (a.key_fp8)
        launch(&tq4::prefix::prefix_kernel<LAYOUT, true, false, false, WR, WT, PLO>, grid, block, st, p);
    else if (a.key_bits == 3 && a.value_bits == 3)
        launch(&tq4::prefix::prefix_kernel<LAYOUT, false, true, true, WR, WT, PLO>, grid, block, st, p);
    else if (a.key_bits == 3)
        launch(&tq4::prefix::prefix_kernel<LAYOUT, false, true, false, WR, WT, PLO>, grid, block, st, p);
    else
        launch(&tq4::prefix::prefix_kernel<LAYOUT, false, false, false, WR, WT, PLO>, grid, block, st, p);
}
template <int LAYOUT>
void launch_prefix(const Stage1Args &a, const tq4::prefix::Args &p, int wr, bool plo, dim3 grid, hipStream_t st) {
    if (wr == 4)
        plo ? launch_prefix<LAYOUT, 4, 2, true>(a, p, grid, st) : launch_prefix<LAYOUT, 4, 2, false>(a, p, grid, st);
    else
        plo ? launch_prefix<LAYOUT, 2, 1, true>(a, p, grid, st) : launch_prefix<LAYOUT, 2, 1, false>(a, p, grid, st);
}

}  // namespace

extern "C" {

int64_t tq4_prefix_workspace_floats(int B, int Hq, int Hk, int num_kv_splits) {
    if (B <= 0 || Hq <= 0 || Hk <= 0 || Hq % Hk || num_kv_splits <= 0) {
        fail(TQ4_E_INVALID, "tq4_prefix_workspace_floats: B, Hq, Hk and num_kv_splits must be positive, Hq a multiple of Hk");
        return -1;
    }
    return workspace_of(B, Hq, Hk, num_kv_splits).total;
}

int tq4_prefix_decode(const void *query, int query_dtype, const float *rot_t, const float *centroids,
                      const uint8_t *kv_cache, const int32_t *block_table, const int32_t *seq_lens, float *workspace,
                      int64_t workspace_floats, void *out, int out_dtype, float *lse, int B, int Hq, int Hk, int D,
                      int block_size, int max_blocks_per_seq, int64_t cache_block_stride, int num_kv_splits, int layout,
                      float attn_scale, const float *sinks, int key_bits, int value_bits, int prefix_len, int kernel,
                      tq4_stream_t stream) {
    constexpr char what[] = "tq4_prefix_decode";
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    Stage1Args a{};
    int rc = span_args(a, what, query, query_dtype, rot_t, centroids, kv_cache, block_table, seq_lens, workspace,
                       workspace, out, out_dtype, lse, B, Hq, Hk, D, block_size, max_blocks_per_seq, cache_block_stride,
                       num_kv_splits, layout, attn_scale, sinks, key_bits, value_bits);
    if (rc)
        return rc;
    if (prefix_len < 0 || prefix_len % block_size || prefix_len / block_size > max_blocks_per_seq)
        return fail(TQ4_E_INVALID, "%s: prefix_len %d must be whole blocks of %d, at most the table's %d", what, prefix_len,
                    block_size, max_blocks_per_seq);
    if (query_dtype == TQ4_F32 || out_dtype == TQ4_F32)
        return fail(TQ4_E_UNSUPPORTED, "%s: 16-bit queries and outputs only (the shared product has f16 operands)", what);
    if (kernel != TQ4_KERNEL_AUTO && kernel != TQ4_KERNEL_SHARED)
        return fail(TQ4_E_INVALID, "%s: kernel must be %d (auto) or %d (shared)", what, TQ4_KERNEL_AUTO, TQ4_KERNEL_SHARED);
    const Workspace ws = workspace_of(B, Hq, Hk, num_kv_splits);
    if (workspace_floats < ws.total || !aligned(workspace, 16))
        return fail(TQ4_E_INVALID, "%s: workspace of %lld floats, needs %lld, 16-byte aligned", what,
                    (long long)workspace_floats, (long long)ws.total);
    float *q_rot = workspace, *own = workspace + ws.own, *shared = workspace + ws.shared;
    a.q_rot = q_rot;
    a.mid_o = own;
    StepIo io{query, query_dtype, rot_t, q_rot, centroids, out, out_dtype, lse};
    const PrefixPlan plan = prefix_plan(B * (Hq / Hk), Hk, prefix_len);
    if (prefix_len == 0 || (kernel == TQ4_KERNEL_AUTO && !sharing_pays(a, plan, prefix_len)))
        return run_step(a, io, true, st);
    if (!a.key_fp8) {
        rc = rotate_query(query, query_dtype, rot_t, q_rot, B * Hq, D, nullptr, nullptr, st);
        if (rc)
            return rc;
        io.rotated = true;
    }
    // the shared tokens
    tq4::prefix::Args p{};
    p.query = a.key_fp8 ? query : q_rot;
    p.q_dtype = query_dtype;
    p.centroids = centroids;
    p.cache = kv_cache;
    p.pages = block_table;
    p.seq_lens = seq_lens;
    p.batch = B;
    p.table_width = max_blocks_per_seq;
    p.parts = shared;
    p.block_stride = cache_block_stride;
    p.score_scale_log2 = attn_scale * tq4::kLog2e;
    p.num_q_heads = Hq;
    p.num_kv_heads = Hk;
    p.group = Hq / Hk;
    p.rows = B * p.group;
    p.total_rows = B * Hq;
    p.tokens = prefix_len;
    p.tiles = plan.tiles;
    p.row_tiles = plan.row_tiles;
    p.splits = plan.splits;
    p.block_size_log2 = log2_int(block_size);
    p.slot_pos = a.slot_pos;
    p.slot_head = a.slot_head;
    const dim3 grid((unsigned)(((int64_t)Hk * plan.splits * plan.row_tiles + 7) / 8 * 8));
    const bool plo = out_dtype == TQ4_F16;
    a.kl == 0 ? launch_prefix<0>(a, p, plan.wr, plo, grid, st) : launch_prefix<1>(a, p, plan.wr, plo, grid, st);
    rc = launch_status("prefix");
    if (rc)
        return rc;
    // the sequences' own tokens; whole: the rows in the place of one part
    const StepPlan step = step_plan(a, tq4::xdl::own_blocks(max_blocks_per_seq, prefix_len / block_size), num_kv_splits > 1);
    const int slots = step.whole ? 1 : num_kv_splits;
    a.sinks = nullptr;  // (the join's)
    io.out = own;
    io.out_dtype = TQ4_F32;
    io.lse = own + (int64_t)B * Hq * tq4::kHeadDim;
    rc = launch_hidden_step(a, io, step, tq4::xdl::Hidden{0, 0, prefix_len}, st);
    if (rc)
        return rc;
    const dim3 rows(Hq, B), wave(tq4::kWave);
    if (out_dtype == TQ4_BF16)
        launch(&tq4::prefix::join_kernel<__bf16>, rows, wave, st, shared, plan.splits, own, slots, (int)step.whole, seq_lens,
               prefix_len, sinks, static_cast<__bf16 *>(out), lse, Hq);
    else
        launch(&tq4::prefix::join_kernel<_Float16>, rows, wave, st, shared, plan.splits, own, slots, (int)step.whole, seq_lens,
               prefix_len, sinks, static_cast<_Float16 *>(out), lse, Hq);
    return launch_status("prefix join");
}

}  // extern "C"
