// What a round does with a verified tree of drafts: the greedy acceptance of one path of it, and the move of
// that path's cache rows to where a chain would have left them.

#include "mtpk_host.h"
#include "mtpk_tree.h"

namespace mtpk {

// Greedy acceptance. From node 0, the lane's own token, on to the first child whose token is the model's next token
// after the node, as long as there is one, the node's next token is no stop and the budget lasts. One wave a lane of the
// round, a node to each of its lanes: a step is one ballot. All latency: the loads of the tree's three rows, the
// stop ids and the lane's numbers are on their way together (3.1 us alone, 48 lanes of 61 nodes 4.7).
struct TreeAcceptArgs {
  const int64_t* best;  // [B, t]: the model's next token after each node
  int64_t best_stride;
  const int64_t* tokens;
  int64_t tokens_stride;
  TreeParents parents;
  const uint8_t* active;
  const int64_t* pos;
  const int64_t* budget;
  const int64_t* stops;
  int n_stops, t;
  int64_t *path, *accept_len, *lengths;
  uint8_t* keep;
  int64_t *bonus, *next_pos, *budget_left;
  uint8_t* live;
  int64_t* hidden_src;
};

__device__ inline int64_t lane_value(int64_t v, int lane) { return (int64_t)lane_bits((uint64_t)v, lane); }

__global__ __launch_bounds__(kWave) void k_tree_accept(TreeAcceptArgs a) {
  const int b = blockIdx.x, lane = threadIdx.x;
  const bool node = lane < a.t;
  const int64_t best = node ? a.best[b * a.best_stride + lane] : -1;
  const int64_t token = node ? a.tokens[b * a.tokens_stride + lane] : -1;
  const int parent = a.parents.at(b, lane, a.t);
  const int64_t budget = a.budget[b], pos = a.pos[b];
  const bool active = a.active[b] != 0;
  bool stop = false;
  for (int i = 0; i < a.n_stops; ++i) stop |= node && a.stops[(int64_t)b * a.n_stops + i] == best;
  const uint64_t stops = __ballot(stop);
  const bool rooted = __builtin_amdgcn_readlane(parent, 0) == -1;  // else node 0, and so all that hangs below it, is absent
  int at = 0, n = 0, mine = 0;
  while (rooted && n + 1 < budget && !(stops >> at & 1ull)) {
    const uint64_t fits = __ballot(parent == at && token == lane_value(best, at));  // a parent comes before its children
    if (fits == 0ull) break;
    at = __builtin_ctzll(fits);
    ++n;
    if (lane == n) mine = at;
  }
  const int64_t bonus = lane_value(best, at);
  if (node) {
    a.path[(int64_t)b * a.t + lane] = lane <= n ? mine : at;
    a.keep[(int64_t)b * a.t + lane] = active && lane <= n;
  }
  if (lane == 0) {
    const int64_t left = budget - n - 1;
    a.accept_len[b] = n;
    a.lengths[b] = active ? n + 1 : 1;
    a.bonus[b] = bonus;
    a.next_pos[b] = pos + n + 1;
    a.budget_left[b] = left;
    a.live[b] = !(stops >> at & 1ull) && left > 0;
    a.hidden_src[b] = (int64_t)b * a.t + at;
  }
}

// The accepted rows together: cache row base + path[i] to base + i for i below the lane's length, in the K and V pools
// of all layers at once. A path rises, so a row is read before a later one takes its place, and never written before it
// is read, if each thread moves its share of the rows in order. Of K that is 16 bytes of every row; of V, which lies
// transposed in its block, one channel's line of the block's positions. A chain of latencies, base and path, table, rows, store:
// 30 pools of one lane 3.9 us. Of 48 lanes with up to 8 rows 10.6: V goes two bytes at a time, out of a line of 32 for each row.
constexpr int kKeepPools = 64;  // pools a launch takes
constexpr int kKeepAhead = 8;   // rows on their way at once
constexpr int kKeepBlock = 16;  // rows of a cache block

struct KeepPool {
  uint8_t* p;
  int units;  // threads' shares: 16-byte pieces of a K row, channels of a V block
  int size;   // bytes of a V element, 0: a K pool
};

struct KeepArgs {
  KeepPool pool[kKeepPools];
  const int32_t* table;
  int64_t table_stride;
  const int64_t* base;
  const int64_t* path;
  const int64_t* lengths;
  int64_t n_blocks;
  int t, pieces;  // pieces: 256 units each, of the largest pool
};

// All of the wave's lanes come here, with their moves; `on`: whether this one has a share.
template <typename T>
__device__ inline void keep_rows(T* unit, bool on, int64_t block_stride, int row_stride, uint64_t moves, int from_block, int from_row,
                                 int to_block, int to_row) {
  while (moves != 0ull) {
    uint64_t m = moves;
    T v[kKeepAhead];
#pragma unroll
    for (int j = 0; j < kKeepAhead; ++j) {
      if (m == 0ull) continue;  // uniform
      const int i = __builtin_ctzll(m);
      m &= m - 1ull;
      const int64_t at = __builtin_amdgcn_readlane(from_block, i) * block_stride + __builtin_amdgcn_readlane(from_row, i) * row_stride;
      if (on) v[j] = unit[at];
    }
#pragma unroll
    for (int j = 0; j < kKeepAhead; ++j) {
      if (moves == 0ull) continue;
      const int i = __builtin_ctzll(moves);
      moves &= moves - 1ull;
      const int64_t at = __builtin_amdgcn_readlane(to_block, i) * block_stride + __builtin_amdgcn_readlane(to_row, i) * row_stride;
      if (on) unit[at] = v[j];
    }
  }
}

__global__ __launch_bounds__(256) void k_keep_path(KeepArgs a) {
  const int b = blockIdx.z, lane = threadIdx.x & (kWave - 1);
  const KeepPool pool = a.pool[blockIdx.y];
  const int u = blockIdx.x * 256 + threadIdx.x;
  if ((int)(blockIdx.x * 256) + uniform(threadIdx.x / kWave) * kWave >= pool.units) return;  // uniform over the wave
  const int64_t base = a.base[b];
  const TreePath path(a.path + (int64_t)b * a.t, a.lengths[b], a.t, lane);
  // lane i moves row base + node i to base + i
  int from = -1, to = -1;
  const int64_t src = base + path.node, dst = base + lane, held = a.table_stride * kKeepBlock;
  const bool moved = lane < path.steps && path.node != lane && dst >= 0 && src < held && dst < held && src >= 0;
  if (moved) {
    const int32_t* const row = a.table + (int64_t)b * a.table_stride;
    from = row[src / kKeepBlock];
    to = row[dst / kKeepBlock];
  }
  const uint64_t moves = __ballot(moved && from >= 0 && from < a.n_blocks && to >= 0 && to < a.n_blocks);
  const bool on = u < pool.units;
  const int fr = (int)(src % kKeepBlock), tr = (int)(dst % kKeepBlock);
  if (pool.size == 0)
    keep_rows(reinterpret_cast<u32x4_t*>(pool.p) + u, on, (int64_t)kKeepBlock * pool.units, pool.units, moves, from, fr, to, tr);
  else if (pool.size == 2)
    keep_rows(reinterpret_cast<uint16_t*>(pool.p) + (int64_t)u * kKeepBlock, on, (int64_t)kKeepBlock * pool.units, 1, moves, from, fr, to, tr);
  else
    keep_rows(reinterpret_cast<uint32_t*>(pool.p) + (int64_t)u * kKeepBlock, on, (int64_t)kKeepBlock * pool.units, 1, moves, from, fr, to, tr);
}

}  // namespace mtpk

using namespace mtpk;

extern "C" {

int mtpk_tree_accept(const int64_t* step_argmax, int64_t sa_stride, const int64_t* tokens, int64_t tokens_stride,
                     const void* parents, int parents_dtype, const int64_t* parents_strides, const uint8_t* active,
                     const int64_t* pos, const int64_t* budget, const int64_t* stops, int64_t n_stops, int64_t batch, int64_t t,
                     int64_t* path, int64_t* accept_len, int64_t* lengths, uint8_t* keep, int64_t* bonus, int64_t* next_pos,
                     int64_t* budget_left, uint8_t* live, int64_t* hidden_src, void* stream) {
  if (batch < 0 || batch > kMaxGroups || t < 1 || t > kTreeNodes || n_stops < 0 || n_stops > INT32_MAX) return MTPK_EINVAL;
  if (parents_dtype != MTPK_I32 && parents_dtype != MTPK_I64) return MTPK_EINVAL;
  if (batch == 0) return 0;
  if (!step_argmax || !tokens || !parents || !parents_strides || !active || !pos || !budget || (n_stops > 0 && !stops) || !path ||
      !accept_len || !lengths || !keep || !bonus || !next_pos || !budget_left || !live || !hidden_src)
    return MTPK_EINVAL;
  const TreeAcceptArgs a{step_argmax, sa_stride, tokens, tokens_stride, {parents, parents_dtype, parents_strides[0], parents_strides[1]},
                         active, pos, budget, stops, (int)n_stops, (int)t, path, accept_len, lengths, keep, bonus, next_pos,
                         budget_left, live, hidden_src};
  hipLaunchKernelGGL(k_tree_accept, dim3((unsigned)batch), dim3(kWave), 0, (hipStream_t)stream, a);
  return status_of(hipGetLastError());
}

int mtpk_keep_path(void* const* pools, const int64_t* channels, const int* element_bytes, const int* transposed, int n_pools,
                   int64_t n_blocks, const int32_t* block_table, int64_t table_stride, const int64_t* base_pos,
                   const int64_t* path, const int64_t* lengths, int64_t batch, int64_t t, void* stream) {
  if (!pools || !channels || !element_bytes || !transposed || n_pools < 1 || n_blocks < 1 || n_blocks > INT32_MAX) return MTPK_EINVAL;
  if (batch < 0 || batch > INT32_MAX || t < 1 || t > kTreeNodes || table_stride < 1 || table_stride > (1 << 26)) return MTPK_EINVAL;
  for (int i = 0; i < n_pools; ++i) {
    if (!pools[i] || !aligned16(pools[i]) || channels[i] < 1 || channels[i] > (1 << 20)) return MTPK_EINVAL;
    if (element_bytes[i] != 2 && element_bytes[i] != 4) return MTPK_EINVAL;
    if (!transposed[i] && channels[i] * element_bytes[i] % 16) return MTPK_EINVAL;
    // no two may share memory: each moves its rows in an order of its own
    const uintptr_t at = reinterpret_cast<uintptr_t>(pools[i]), bytes = (uintptr_t)(n_blocks * kKeepBlock * channels[i] * element_bytes[i]);
    for (int j = 0; j < i; ++j) {
      const uintptr_t other = reinterpret_cast<uintptr_t>(pools[j]);
      if (at < other + (uintptr_t)(n_blocks * kKeepBlock * channels[j] * element_bytes[j]) && other < at + bytes) return MTPK_EINVAL;
    }
  }
  if (batch == 0 || t == 1) return 0;  // a path of one node is where it belongs
  if (!block_table || !base_pos || !path || !lengths) return MTPK_EINVAL;
  for (int first = 0; first < n_pools; first += kKeepPools) {
    KeepArgs a{};
    const int n = n_pools - first < kKeepPools ? n_pools - first : kKeepPools;
    int most = 0;
    for (int i = 0; i < n; ++i) {
      const int j = first + i;
      KeepPool& p = a.pool[i];
      p.p = static_cast<uint8_t*>(pools[j]);
      p.size = transposed[j] ? element_bytes[j] : 0;
      p.units = (int)(transposed[j] ? channels[j] : channels[j] * element_bytes[j] / 16);
      most = p.units > most ? p.units : most;
    }
    a.table_stride = table_stride;
    a.n_blocks = n_blocks;
    a.t = (int)t;
    a.pieces = (most + 255) / 256;
    const int64_t lanes = kMaxGroups / ((int64_t)n * a.pieces) < 65535 ? kMaxGroups / ((int64_t)n * a.pieces) : 65535;
    if (lanes < 1) return MTPK_EINVAL;
    for (int64_t at = 0; at < batch; at += lanes) {
      a.table = block_table + at * table_stride;
      a.base = base_pos + at;
      a.path = path + at * t;
      a.lengths = lengths + at;
      const int64_t m = batch - at < lanes ? batch - at : lanes;
      hipLaunchKernelGGL(k_keep_path, dim3((unsigned)a.pieces, (unsigned)n, (unsigned)m), dim3(256), 0, (hipStream_t)stream, a);
      const int rc = status_of(hipGetLastError());
      if (rc) return rc;
    }
  }
  return 0;
}

}  // extern "C"
