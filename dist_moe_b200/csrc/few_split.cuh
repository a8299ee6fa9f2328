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

// `strips` strips of `length` items each, in a row, over at most `grid` blocks of at least one item each: the first `longer` of them
// have one item more than the others.  In 32 bits (the host refuses more items): the divisions of 64-bit numbers took a microsecond.
struct FewSplit {
  uint32_t items, length, blocks, share, longer;
  DM_FEW_HOST_DEVICE FewSplit(uint32_t strips, uint32_t length_, uint32_t grid)
      : items(strips * length_), length(length_), blocks(items < grid ? items : grid), share(blocks ? items / blocks : 0), longer(items - share * blocks) {}
  DM_FEW_HOST_DEVICE uint32_t begin(uint32_t block) const {
    return block < blocks ? share * block + (block < longer ? block : longer) : items;
  }
  DM_FEW_HOST_DEVICE uint32_t end(uint32_t block) const { return block < blocks ? begin(block) + share + (block < longer ? 1 : 0) : items; }
  DM_FEW_HOST_DEVICE uint32_t block_of(uint32_t item) const {
    const uint32_t in_longer = longer * (share + 1);
    return item < in_longer ? item / (share + 1) : longer + (item - in_longer) / share;
  }
  // The blocks that have a part of strip q.
  DM_FEW_HOST_DEVICE uint32_t first_block(uint32_t q) const { return block_of(q * length); }
  DM_FEW_HOST_DEVICE uint32_t last_block(uint32_t q) const { return block_of((q + 1) * length - 1); }
  // A block has parts of two strips at most: the one that it begins in, and the one that it ends in.
  DM_FEW_HOST_DEVICE uint32_t place(uint32_t block, uint32_t q) const { return 2 * block + (begin(block) / length == q ? 0 : 1); }
};

}  // namespace dm
