// How the launches for few tokens deal their items out over the blocks, and where parts of a strip meet.  Plain arithmetic, for the
// kernels and for host code.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define DM_FEW_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define DM_FEW_HOST_DEVICE inline
#endif

namespace dm {

// `strips` strips of `length` items each, in a row, over at most `grid` blocks of at least one item each.
struct FewSplit {
  int64_t items;
  int length, blocks;
  DM_FEW_HOST_DEVICE FewSplit(int64_t strips, int length_, int grid)
      : items(strips * length_), length(length_), blocks(static_cast<int>(strips * length_ < grid ? strips * length_ : grid)) {}
  DM_FEW_HOST_DEVICE int64_t begin(int block) const { return block < blocks ? items * block / blocks : items; }
  DM_FEW_HOST_DEVICE int64_t end(int block) const { return block < blocks ? items * (block + 1) / blocks : items; }
  DM_FEW_HOST_DEVICE int block_of(int64_t item) const { return static_cast<int>(((item + 1) * blocks - 1) / items); }
  // The blocks that have a part of strip q.
  DM_FEW_HOST_DEVICE int first_block(int64_t q) const { return block_of(q * length); }
  DM_FEW_HOST_DEVICE int last_block(int64_t q) const { return block_of((q + 1) * length - 1); }
  // A block has parts of two strips at most: the one that it begins in, and the one that it ends in.
  DM_FEW_HOST_DEVICE int64_t place(int block, int64_t q) const { return 2 * static_cast<int64_t>(block) + (begin(block) / length == q ? 0 : 1); }
};

}  // namespace dm
