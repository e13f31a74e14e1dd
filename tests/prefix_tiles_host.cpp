// prefix_tiles.h compiled for the host: what every wave of a workgroup does with the LDS buffers, and between
// which barriers.
#include <cstddef>

#define __device__
#define __forceinline__ inline
#include "../turboquant-cuda-decode_amd/csrc/prefix_tiles.h"

using namespace tq4::prefix;

namespace {

// K, factors, V
enum Place { kKeys, kFactors, kValues };

template <int WT> int run(int n, int late, int does_k, int does_v, int *out, int room, int *barriers) {
    using B = Buffers<WT>;
    int phase = 0, count = 0;
    auto add = [&](int place, int buffer, int tile, int write) {
        if (count < room) {
            int *r = out + 5 * count;
            r[0] = phase;
            r[1] = place;
            r[2] = buffer;
            r[3] = tile;
            r[4] = write;
        }
        ++count;
    };
    run_tiles<WT>(
        n, late != 0, [&] { ++phase; }, [&] { ++phase; },
        [&](int i) {
            if (does_k) {
                add(kKeys, B::tile(i), i, 1);
                add(kFactors, B::factor(i), i, 1);
            }
            if (does_v)
                add(kValues, B::tile(i), i - B::behind, 1);
        },
        [&](int i) { add(kKeys, B::tile(i), i, 0); }, [&](int i) { add(kFactors, B::factor(i), i, 0); },
        [&](int i) { add(kValues, B::tile(i), i, 0); }, [](bool) {});
    *barriers = phase;
    return count <= room ? count : -1;
}

}  // namespace

// One wave's accesses over n tiles, rows of (barriers passed, place, buffer, tile, write).
extern "C" int host_accesses(int wt, int n, int late, int does_k, int does_v, int *out, int room, int *barriers) {
    return wt == 2 ? run<2>(n, late, does_k, does_v, out, room, barriers) : run<1>(n, late, does_k, does_v, out, room, barriers);
}
