// The two blocks of shared memory through which a warp's 32 rows of a tile leave by TMA stores, one store a block of columns, one after
// another. A tile ends where the matrix does, after any number of stores, and the next begins with the first block again: it is free only
// when no store at all reads on. Within a tile the store before the last has to have read its block.
// Plain C++ for the host as well: a test walks tiles of every width through it.
#pragma once

#ifdef __CUDACC__
#define KCG_STORE_BLOCKS_FN __host__ __device__ constexpr
#else
#define KCG_STORE_BLOCKS_FN constexpr
#endif

namespace kcg {

// The block of a tile's store b = 0, 1, ...
KCG_STORE_BLOCKS_FN int store_block(int b) { return b & 1; }
// How many of the warp's last stores may still read shared memory when that block is written.
KCG_STORE_BLOCKS_FN int stores_reading(int b) { return b == 0 ? 0 : 1; }

}  // namespace kcg

#undef KCG_STORE_BLOCKS_FN
