// Trees of drafted tokens, as every kernel that verifies one reads them: `parents` [batch, t], t at most 64,
// where node s of a lane hangs below an earlier node, or, at -1, below the committed context. Any other value
// marks an absent node (the end of a smaller tree), and what hangs below an absent node is absent too.
#pragma once

#include "mtpk_device.h"

namespace mtpk {

constexpr int kTreeNodes = 64;  // a lane of the wave for each

struct TreeParents {
  const void* p;
  int dt;
  int64_t sb, ss;  // element strides of a lane and of a node
  // The parent of node `s` of `t`, or -2 where the node cannot be present.
  __device__ inline int at(int b, int s, int t) const {
    if (s >= t) return -2;
    const int64_t v = load_index(p, dt, b * sb + s * ss);
    return v < -1 || v >= s ? -2 : (int)v;
  }
};

// Node `lane`'s ancestors and itself as bits, 0 where it is absent, from its parent (every lane of the wave takes
// part): each round doubles how far up a node has looked. Parents come before their children, so the set bits
// from the highest down are the way up.
__device__ inline uint64_t tree_ancestors(int parent, int lane) {
  uint64_t m = parent >= -1 ? 1ull << lane : 0ull;
  int up = parent;
  while (__ballot(up >= 0) != 0ull) {
    const int at = up < 0 ? lane : up;
    const uint32_t lo = __shfl((uint32_t)m, at, kWave), hi = __shfl((uint32_t)(m >> 32), at, kWave);
    const int next = __shfl(up, at, kWave);
    if (up >= 0) {
      m |= (uint64_t)hi << 32 | lo;
      up = next;
    }
  }
  return up == -1 ? m : 0ull;
}

// A lane's 64 bits, for a uniform lane index.
__device__ inline uint64_t lane_bits(uint64_t m, int lane) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(m >> 32), lane) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)m, lane);
}

// A path of accepted nodes [t] of a lane, held a node to a lane of the wave: the steps before the first entry that is
// no node, at most `length`.
struct TreePath {
  int node, steps;
  __device__ inline TreePath(const int64_t* path, int64_t length, int t, int lane) {
    const int64_t v = lane < t ? path[lane] : -1;
    node = (int)v;
    const uint64_t no = __ballot(v < 0 || v >= t);
    steps = (int)min(max(length, (int64_t)0), (int64_t)(no ? __builtin_ctzll(no) : kTreeNodes));
  }
  __device__ inline int at(int i) const { return __builtin_amdgcn_readlane(node, i); }
};

}  // namespace mtpk
