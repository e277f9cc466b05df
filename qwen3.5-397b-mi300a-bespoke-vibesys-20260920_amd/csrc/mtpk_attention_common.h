// What the attention kernels over the paged cache share: the cache's block, the strides of query and
// output rows, and the places of a tile's keys in LDS for products on 32 x 32 x 16.
#pragma once

#include "mtpk_device.h"

namespace mtpk {

constexpr int kAttnBlock = 16;  // KV cache block size

// Where the query rows come from and the output rows go: element d of (lane b, q head h, step s)
// is at b * sb + h * sh + s * st + d of each tensor (unit stride over d).
struct AttnRows {
  int64_t sb, sh, st;
  __device__ inline int64_t at(int b, int h, int s) const { return b * sb + h * sh + s * st; }
};

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

// Bits 2 and 3 of a tile's key or row index swapped.
__device__ inline int prompt_swap(int i) { return (i & ~12) | ((i & 4) << 1) | ((i & 8) >> 1); }

// The change of place of a K row's pieces: the rows 0..3 and 0..7 that one LDS cycle reads, of either
// half of the wave, then lie in different bank groups.
__device__ inline int prompt_flip(int row) { return ((row & 3) << 1) | (row >> 2 & 1); }

}  // namespace mtpk
