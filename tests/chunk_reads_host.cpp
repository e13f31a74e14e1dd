// chunk_plan.h compiled for the host: the tokens whose blocks the row tiles of a sequence read.
#include <cstdint>

#define __device__
#define __forceinline__ inline
#include "../turboquant-cuda-decode_amd/csrc/chunk_plan.h"

using namespace tq4::chunk;

// shape: rows, tile, group, kv_heads, causal, window, first.  reads: (row tile, first of 16 tokens, the token whose block is
// read for them, whether they count as hidden) of every 16 tokens that a row tile visits; returns how many.
extern "C" int host_reads(const int *shape, int n, int len, int *reads, int room) {
    const Shape s{shape[0], shape[1], shape[2], shape[3], shape[4], shape[5], shape[6]};
    const Seq q{0, n, len};
    int count = 0;
    for (int r = 0; r < row_tiles(s, n); ++r) {
        const Visits v = visits_of(s, q, r);
        const Seen seen = seen_of(s, q, r);
        for (int i = 0; i < v.count; ++i)
            for (int t = s.tile * (i < v.head ? i : i + v.skip), end = t + s.tile; t < end; t += 16, ++count)
                if (count < room) {
                    const int to[4] = {r, t, read_at(seen, len, t), hidden(seen, t)};
                    for (int k = 0; k < 4; ++k)
                        reads[4 * count + k] = to[k];
                }
    }
    return count;
}
