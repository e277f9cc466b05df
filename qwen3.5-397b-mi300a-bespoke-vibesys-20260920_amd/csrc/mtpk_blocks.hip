// Copies of cache blocks inside the pools of all layers, in one launch: forked lanes' partly filled
// blocks, blocks that a compaction moves. A block is contiguous in the K pool (16 rows) and in the V pool
// (16 rows, transposed inside), so that a pool is an array of blocks of `bytes[i]` bytes and nothing
// else is known of it. A workgroup moves up to 16 KB of one pair, all of its loads issued before the
// first store. Bound by the bytes, each read once and written once.

#include "mtpk_device.h"
#include "mtpk_host.h"

namespace mtpk {

constexpr int kCopyPools = 64;        // pools a launch takes
constexpr int kCopyPiece = 16 << 10;  // bytes a workgroup moves

struct CopyArgs {
  uint8_t* pool[kCopyPools];
  int64_t bytes[kCopyPools];  // of a block
  const void* src;
  const void* dst;
  int index_dt;
  int64_t n_blocks;
  int pools, pieces;  // pieces: of the largest block
};

__global__ __launch_bounds__(256) void k_copy_blocks(CopyArgs a) {
  constexpr int N = kCopyPiece / 256 / 16;
  const int64_t per = (int64_t)a.pools * a.pieces;
  const int64_t pair = blockIdx.x / per;  // of this launch
  const int rest = (int)(blockIdx.x - pair * per), i = rest / a.pieces, piece = rest % a.pieces;
  const int64_t from = load_index(a.src, a.index_dt, pair), to = load_index(a.dst, a.index_dt, pair);
  if (from < 0 || from >= a.n_blocks || to < 0 || to >= a.n_blocks || from == to) return;
  const int64_t bytes = a.bytes[i];
  const uint8_t* const s = a.pool[i] + from * bytes;
  uint8_t* const d = a.pool[i] + to * bytes;
  u32x4_t r[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int64_t at = (int64_t)piece * kCopyPiece + (j * 256 + threadIdx.x) * 16;
    if (at < bytes) r[j] = ld16(s + at);
  }
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int64_t at = (int64_t)piece * kCopyPiece + (j * 256 + threadIdx.x) * 16;
    if (at < bytes) *reinterpret_cast<u32x4_t*>(d + at) = r[j];
  }
}

}  // namespace mtpk

using namespace mtpk;

extern "C" int mtpk_copy_blocks(void* const* pools, const int64_t* block_bytes, int n_pools,
                                int64_t n_blocks, const void* src, const void* dst, int index_dtype,
                                int64_t pairs, void* stream) {
  if (!pools || !block_bytes || n_pools < 1 || n_blocks < 1 || pairs < 0 || pairs > INT32_MAX) return MTPK_EINVAL;
  if (index_dtype != MTPK_I32 && index_dtype != MTPK_I64) return MTPK_EINVAL;
  for (int i = 0; i < n_pools; ++i)
    if (!pools[i] || !aligned16(pools[i]) || block_bytes[i] < 16 || block_bytes[i] % 16) return MTPK_EINVAL;
  if (pairs == 0) return 0;
  if (!src || !dst) return MTPK_EINVAL;
  for (int first = 0; first < n_pools; first += kCopyPools) {
    CopyArgs a{};
    a.pools = n_pools - first < kCopyPools ? n_pools - first : kCopyPools;
    int64_t most = 0;
    for (int i = 0; i < a.pools; ++i) {
      a.pool[i] = static_cast<uint8_t*>(pools[first + i]);
      a.bytes[i] = block_bytes[first + i];
      most = a.bytes[i] > most ? a.bytes[i] : most;
    }
    const int64_t pieces = (most + kCopyPiece - 1) / kCopyPiece;
    if (pieces > kMaxGroups / a.pools) return MTPK_EINVAL;
    a.index_dt = index_dtype;
    a.n_blocks = n_blocks;
    a.pieces = (int)pieces;
    const int64_t most_pairs = kMaxGroups / (a.pools * pieces), index_bytes = index_dtype == MTPK_I64 ? 8 : 4;
    for (int64_t at = 0; at < pairs; at += most_pairs) {
      const int64_t n = pairs - at < most_pairs ? pairs - at : most_pairs;
      a.src = static_cast<const uint8_t*>(src) + at * index_bytes;
      a.dst = static_cast<const uint8_t*>(dst) + at * index_bytes;
      hipLaunchKernelGGL(k_copy_blocks, dim3((unsigned)(n * a.pools * pieces)), dim3(256), 0, (hipStream_t)stream, a);
      const int rc = status_of(hipGetLastError());
      if (rc) return rc;
    }
  }
  return 0;
}
