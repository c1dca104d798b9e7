// Prints the tiles that a head's logits are cut into: for each pair of arguments, rows that count and vocabulary rows, the width
// of a tile, the number of tiles and how many of them are cut into stripes.
#define __host__
#define __device__
#include "tiles.h"

#include <cstdio>
#include <cstdlib>

int main(int argc, char** argv) {
    for (int i = 1; i + 1 < argc; i += 2) {
        const uint32_t rows = std::strtoul(argv[i], nullptr, 10), vocab = std::strtoul(argv[i + 1], nullptr, 10);
        const twd::LogitTiles t = twd::logit_tiles(rows, (vocab + twd::kVocabTile - 1) / twd::kVocabTile);
        std::printf("%u %u %u\n", t.width, t.grid.tiles(), t.cut);
    }
}
