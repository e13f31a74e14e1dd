// chunk_plan.h compiled for the host: a call's cuts, and the tiles that each row tile visits.
#include <cstdint>
#include <vector>

#define __device__
#define __forceinline__ inline
#include "../turboquant-cuda-decode_amd/csrc/chunk_plan.h"

using namespace tq4::chunk;

// shape: rows, tile, group, kv_heads, causal, window, first.  cuts: groups + 1 times (b, h, r, at).
extern "C" void host_cuts(const int *shape, const int32_t *starts, const int32_t *lens, int batch, int tokens, int longest,
                          int groups, int *cuts) {
    const Shape s{shape[0], shape[1], shape[2], shape[3], shape[4], shape[5], shape[6]};
    auto seq = [&](int b) { return seq_of(starts, lens, b, tokens, longest); };
    std::vector<double> work(batch);
    double total = 0;
    for (int b = 0; b < batch; ++b) {
        work[b] = total;
        total += work_of(s, seq(b));
    }
    const int used = groups_used(total, groups);
    for (int w = 0; w <= groups; ++w) {
        const Cut c = cut_of(s, seq, work.data(), batch, total, used, w);
        const int to[4] = {c.b, c.h, c.r, c.at};
        for (int i = 0; i < 4; ++i)
            cuts[4 * w + i] = to[i];
    }
}
// seq: row0, n, len.  visits: head, skip, count of each row tile; returns how many.
extern "C" int host_visits(const int *shape, const int32_t *starts, const int32_t *lens, int b, int tokens, int longest, int *seq,
                           int *visits, int room) {
    const Shape s{shape[0], shape[1], shape[2], shape[3], shape[4], shape[5], shape[6]};
    const Seq q = seq_of(starts, lens, b, tokens, longest);
    seq[0] = q.row0;
    seq[1] = q.n;
    seq[2] = q.len;
    const int tiles = row_tiles(s, q.n);
    for (int r = 0; r < tiles && r < room; ++r) {
        const Visits v = visits_of(s, q, r);
        visits[3 * r] = v.head;
        visits[3 * r + 1] = v.skip;
        visits[3 * r + 2] = v.count;
    }
    return tiles;
}
extern "C" double host_work(const int *shape, int n, int len, int r) {
    const Shape s{shape[0], shape[1], shape[2], shape[3], shape[4], shape[5], shape[6]};
    return work_before(s, Seq{0, n, len}, r);
}
