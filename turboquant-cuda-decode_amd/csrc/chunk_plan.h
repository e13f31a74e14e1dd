// How the work of a chunk_attention call is cut over the workgroups of its grid.  Compiled into the kernels
// (chunk.h), and for the host by the tests.
//
// A sequence's query rows (new token, head of the kv-head's group; new tokens first) are taken in row tiles of
// `rows` rows, a row tile's visible tokens in token tiles of `tile`.  The list of all row tiles (sequence, kv-head,
// row tile) is cut where the work up to there is a whole share of all of it, so a workgroup has the end of one row tile,
// whole ones, and the start of another.
#pragma once
#include <cstdint>

namespace tq4 {
namespace chunk {

struct Shape {
    int rows, tile, group, kv_heads;
    int causal, window, first;  // window 0: none
};
// A sequence: its query rows' first token, how many new tokens, and its length.
struct Seq {
    int row0, n, len;
};
// (whatever starts and lens hold, the tokens stay inside the query and the length inside the table)
__device__ __forceinline__ Seq seq_of(const int32_t *starts, const int32_t *lens, int b, int tokens, int longest) {
    const int s = starts[b], e = starts[b + 1], n = lens[b];
    const int s0 = s < 0 ? 0 : s > tokens ? tokens : s, e0 = e < s0 ? s0 : e > tokens ? tokens : e;
    return Seq{s0, e0 - s0, n < 0 ? 0 : n > longest ? longest : n};
}
__device__ __forceinline__ int row_tiles(const Shape &s, int n) { return (n * s.group + s.rows - 1) / s.rows; }
// Tokens before this many are visible to row `row` (window and first tokens apart).
__device__ __forceinline__ int limit_of(const Shape &s, const Seq &q, int row) {
    if (!s.causal)
        return q.len;
    const int end = q.len - q.n + row / s.group + 1;
    return end < 0 ? 0 : end;
}
// The token tiles of a row tile, [0, head) and [head + skip, count + skip): place i is tile i, or i + skip from
// `head` on.
struct Visits {
    int head, skip, count;
};
__device__ __forceinline__ Visits visits_of(const Shape &s, const Seq &q, int r) {
    const int rows = q.n * s.group, first_row = r * s.rows;
    const int last_row = first_row + s.rows < rows ? first_row + s.rows - 1 : rows - 1;
    const int end = limit_of(s, q, last_row), tiles = (end + s.tile - 1) / s.tile;
    if (!s.window)
        return Visits{0, 0, tiles};
    const int from = limit_of(s, q, first_row) - s.window;
    const int seen = s.first < end ? s.first : end;
    const int head = (seen + s.tile - 1) / s.tile, next = from > 0 ? from / s.tile : 0;
    if (next <= head)
        return Visits{0, 0, tiles};
    return Visits{head, next - head, head + (tiles > next ? tiles - next : 0)};
}
// What a row tile sees: tokens before `first` and from `from` on, all before `end`.  Its token tiles may hold others in front of
// the window, whose blocks may be anybody's by now: 16 tokens (they lie in one block) that no row sees are not read.
struct Seen {
    int first, from, end;
};
__device__ __forceinline__ Seen seen_of(const Shape &s, const Seq &q, int r) {
    const int rows = q.n * s.group, first_row = r * s.rows;
    const int last_row = first_row + s.rows < rows ? first_row + s.rows - 1 : rows - 1;
    return Seen{s.first, s.window ? limit_of(s, q, first_row) - s.window : 0, limit_of(s, q, last_row)};
}
// Whether no row sees any of the 16 tokens from t on.
__device__ __forceinline__ bool hidden(const Seen &s, int t) { return t >= s.first && t + 16 <= s.from; }
// The token whose block is read for them: their own, the sequence's last one behind its end (whose block later rows see),
// the row tile's last one for hidden ones.
__device__ __forceinline__ int read_at(const Seen &s, int len, int t) {
    return hidden(s, t) ? s.end - 1 : t < len - 1 ? t : len - 1;
}
// The work of a row tile in token tiles: about those it visits (a straight line through their number, so that sums
// have a closed form) and kStart for the queries, the first loads and the results.
constexpr double kStart = 3.0;
// Of the row tiles before tile r of a sequence.
__device__ __forceinline__ double work_before(const Shape &s, const Seq &q, int r) {
    const double step = (double)s.rows / s.group;
    if (!s.causal)
        return r * (kStart + (double)q.len / s.tile);
    // the tokens of tile i: base + (i + 1) step, at least 0 and at most `most`
    const double base = (double)q.len - q.n, most = s.window ? (double)s.window + s.first + step : 1e18;
    int lo = base < 0 ? (int)(-base / step) : 0;
    lo = lo < r ? lo : r;
    const double until = (most - base) / step;
    int hi = until < r ? (int)until : r;
    hi = hi < lo ? lo : hi;
    const double n = hi - lo, sum = n * base + step * (n * lo + 0.5 * n * (n + 1));
    return r * kStart + ((sum > 0 ? sum : 0.0) + (r - hi) * (s.window ? most : 0.0)) / s.tile;
}
__device__ __forceinline__ double work_of(const Shape &s, const Seq &q) {
    return s.kv_heads * work_before(s, q, row_tiles(s, q.n));
}
// A place in the list: token tile `at` (its place among the visits) of row tile r of (sequence b, kv-head h);
// b = batch: the end.
struct alignas(16) Cut {
    int b, h, r, at;
};
__device__ __forceinline__ bool same_tile(const Cut &x, const Cut &y) { return x.b == y.b && x.h == y.h && x.r == y.r; }
// The place with work `at` before it inside sequence b (n > 0).  A cut within `snap` tiles of a row tile's
// start or end goes there: parts of a row tile cost a write and a read of all its rows.
__device__ __forceinline__ Cut cut_in(const Shape &s, const Seq &q, int b, double at, int snap) {
    const int tiles = row_tiles(s, q.n);
    const double each = work_before(s, q, tiles);
    int h = (int)(at / each);
    h = h < 0 ? 0 : h >= s.kv_heads ? s.kv_heads - 1 : h;
    const double in = at - h * each;
    int lo = 0, hi = tiles - 1;  // the last row tile with work_before <= in
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (work_before(s, q, mid) <= in)
            lo = mid;
        else
            hi = mid - 1;
    }
    const double w0 = work_before(s, q, lo), w1 = work_before(s, q, lo + 1);
    const int count = visits_of(s, q, lo).count;
    int place = (int)((in - w0) / (w1 - w0) * count + 0.5);
    place = place <= snap ? 0 : place >= count - snap ? count : place;
    Cut c{b, h, lo, place};
    if (place >= count && !(place == 0 && (in - w0) * 2 < w1 - w0)) {  // the next row tile's start
        c.at = 0;
        if (++c.r == tiles) {
            c.r = 0;
            if (++c.h == s.kv_heads) {
                c.h = 0;
                ++c.b;  // (the caller passes over sequences without new tokens)
            }
        }
    }
    return c;
}

// The least work that a workgroup is given, in token tiles: fewer workgroups than the grid's share a small call.
constexpr double kLeast = 4.0;
constexpr int kSnap = 2;
__device__ __forceinline__ int groups_used(double total, int groups) {
    const double n = total / kLeast;
    return n < 1 ? 1 : n < groups ? (int)n : groups;
}
// Where workgroup w of `used` begins (w >= used: the end).  `seq(b)`: the sequences; work[b]: that of those before b.
template <class SeqOf>
__device__ __forceinline__ Cut cut_of(const Shape &s, SeqOf seq, const double *work, int batch, double total, int used, int w) {
    if (w >= used || total <= 0)
        return Cut{batch, 0, 0, 0};
    const double target = total * w / used;
    int lo = 0, hi = batch - 1;  // the last sequence with as little before it
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (work[mid] <= target)
            lo = mid;
        else
            hi = mid - 1;
    }
    const Seq q = seq(lo);
    Cut c{lo, 0, 0, 0};
    if (q.n > 0 && w > 0)
        c = cut_in(s, q, lo, target - work[lo], kSnap);
    if (c.at == 0 && c.r == 0 && c.h == 0)
        while (c.b < batch && seq(c.b).n == 0)
            ++c.b;
    return c;
}

}  // namespace chunk
}  // namespace tq4
