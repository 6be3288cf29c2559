// Walks the stores of a warp over tiles of a matrix of N columns, N = 1 .. 1100, and checks that no block of shared memory is written
// while a store of it may still be reading: store_blocks_check <columns of a store>. (The tensor of tiles is one row of them, walked by
// `stride` pairs: the kernel's order only changes which widths follow one another.)
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "store_blocks.h"

int main(int argc, char** argv) {
  const int cols_block = atoi(argv[1]);
  for (int n = 1; n <= 1100; ++n)
    for (int half = 0; half < 2; ++half)
      for (int stride = 1; stride <= 3; ++stride) {
        std::vector<int> reading;  // blocks of the stores that may not have read them, oldest first
        const int tiles = (n + 255) / 256;
        for (int tile = 0, turn = 0; turn < 12; tile = (tile + stride) % tiles, ++turn) {
          const int col0 = tile * 256 + half * 128;
          for (int b = 0; b < 128 / cols_block; ++b) {
            if (col0 + b * cols_block >= n) break;
            while (static_cast<int>(reading.size()) > kcg::stores_reading(b)) reading.erase(reading.begin());
            for (int other : reading)
              if (other == kcg::store_block(b)) {
                printf("N = %d, half %d, tile %d: store %d overwrites a block that is being read\n", n, half, tile, b);
                return 1;
              }
            reading.push_back(kcg::store_block(b));
          }
        }
      }
  printf("OK\n");
}
