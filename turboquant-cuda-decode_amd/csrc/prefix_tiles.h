// The order in which the waves of a prefix_kernel workgroup (prefix.h) work through their tiles, and the
// LDS buffers that they hand each other tiles in.  Compiled into the kernel, and for the host by the tests,
// which check that between two barriers no wave writes what another reads.
#pragma once

namespace tq4 {
namespace prefix {

// WT waves side by side in a tile.  K, V^T: one buffer with WT = 1, where tile j + 1's K takes the place
// of tile j's, whose scores are done, and tile j's V that of tile j - 1's: it is decoded a tile behind K.
// The tokens' factors belong to the softmax, which comes a phase behind the scores: they always alternate (with one
// buffer a wave would write tile j + 1's while the other still reads tile j's).
template <int WT> struct Buffers {
    static constexpr int tiles = WT == 2 ? 2 : 1;
    static constexpr int factors = 2;
    static constexpr int behind = 2 - tiles;  // V of tile i - behind is decoded with K of tile i
    static constexpr int tile(int i) { return i & (tiles - 1); }
    static constexpr int factor(int i) { return i & (factors - 1); }
};

// One wave's way through tiles [0, n), n > 0.  fill(i) decodes tile i (K and the factors of tile i, V of tile
// i - behind), scores(i) reads its K, softmax(i) its factors, outputs(i) its V.  Tile j + 1's scores are worked out
// while tile j's weights go into the accumulators (matrix phase), then its softmax and the decoding of the
// next tile (vector phase).  The two waves of a SIMD are a phase apart (WT = 2; `late`: the second one): one
// uses the matrix core while the other uses the vector unit.  A phase ends at a barrier.
template <int WT, class Barrier, class PhaseEnd, class Fill, class Scores, class Softmax, class Outputs, class Prio>
__device__ __forceinline__ void run_tiles(int n, bool late, Barrier barrier, PhaseEnd phase_end, Fill fill, Scores scores,
                                          Softmax softmax, Outputs outputs, Prio prio) {
    fill(0);
    barrier();
    if (late)
        phase_end();
    scores(0);
    phase_end();
    for (int j = 0; j < n; ++j) {
        softmax(j);
        if (j + 1 < n || Buffers<WT>::behind)
            fill(j + 1);
        phase_end();
        prio(true);
        if (j + 1 < n)
            scores(j + 1);
        outputs(j);
        prio(false);
        phase_end();
    }
    if (WT == 2 && !late)
        phase_end();
}

}  // namespace prefix
}  // namespace tq4
