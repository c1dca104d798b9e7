// Grids of a product's tiles, and the rule by which a head's logits are cut into tiles. Free of device code: a host program that
// gives __host__ and __device__ no meaning may include it.
#pragma once

#include <stdint.h>

namespace twd {

namespace {

struct TileGrid {
    uint32_t na, nb, parts;  // tiles along A and B, and parts of the sum
    __host__ __device__ uint32_t tiles() const { return na * nb * parts; }
};

// Tiles of logits are of 256 vocabulary rows by 256, 192 or 128 hidden rows, whichever takes the least time: rounds of the
// units times a tile's, which goes by its width and some 100 rows more (65,536 x 2,880: 105, 86 and 65 us a round). 518 rows
// of 32,003 x 2,048 take 139, 113 and 124 us, 1,023 of 65,537 x 2,880 take 427, 476 and 476. The few tiles past whole rounds
// are cut into stripes of 64 hidden rows and follow in a launch of their own, which costs some 80 rows of a round.
constexpr uint32_t kVocabTile = 256, kRound = 256, kMostCut = 64;
struct LogitTiles {
    TileGrid grid;
    uint32_t width;  // hidden rows of a tile
    uint32_t cut;    // of the last tiles
};
__host__ __device__ inline LogitTiles logit_tiles(uint32_t count, uint32_t na) {
    LogitTiles best{};
    uint32_t least = ~0u;
#pragma unroll
    for (uint32_t width = 256; width >= 128; width -= 64) {
        const TileGrid g{na, (count + width - 1) / width, 1};
        const uint32_t left = g.tiles() % kRound, cut = left <= kMostCut ? left : 0;
        const uint32_t time = g.tiles() / kRound * (width + 100) + (cut > 0 ? 80 : left > 0 ? width + 100 : 0);
        if (time < least) least = time, best = LogitTiles{g, width, cut};
    }
    return best;
}

}  // namespace

}  // namespace twd
