// Position rotation of attention heads, with the head norms and the way into the paged cache in the
// same pass.
//
// A head's first `rot` channels are rot / 2 pairs, (i, i + rot / 2) or (2 i, 2 i + 1), and pair i of a
// head at position p is turned by p * rates[i] radians and scaled by `magnitude`:
//   (a, b) -> magnitude * (a cos - b sin, b cos + a sin)
// With a weight the head is first normed, y = x * rsqrt(mean(x^2) + eps) * (1 + w). fp32 from the load
// to the store's one rounding; the angle in 64 bits up to its fraction of a turn: at position 10^6 an
// fp32 angle is off by 0.03 radians. Angles are computed here, once per token and workgroup, instead of
// read from a table: one of 10^6 positions by 64 channels would be 512 MB for its cos and sin.
//
// A lane holds 8 adjacent channels of a head (16 bytes of bf16), G lanes a head; a workgroup takes one
// token, 256 / G heads at a time. A lane's channels, and so its cos, sin and weights, are the same for
// every head, and stay in registers. The partner of a channel is in the lane's own 8 (adjacent pairs),
// in the lane rot / 16 further on (halves of whole 8s), or read again from memory (other halves).
// Bound by the bytes of the heads, read once and written once.

#include "mtpk_device.h"
#include "mtpk_host.h"

namespace mtpk {

constexpr int kRotMaxDim = 512;
constexpr int kCacheBlock = 16;  // rows of a cache block

enum RotPairs { kAdjacent = 0, kHalvesOf8 = 1, kHalves = 2 };

struct RotStrides {
  int64_t b, h, s;  // lane, head, step (elements)
};

struct RotArgs {
  const void* q;  // heads of [B, t]
  RotStrides qs;
  const void* qw;  // may be null: no norm
  void* out;
  RotStrides os;
  const uint16_t* k;  // the cache form's k and v rows, null otherwise
  RotStrides ks;
  const void* kw;
  const uint16_t* v;
  RotStrides vs;
  uint16_t* k_pool;
  uint16_t* v_pool;
  int64_t pool_rows;
  const int32_t* table;
  int64_t table_stride;
  const int64_t* base;  // position of step 0 of each lane (null: the positions alone)
  const int64_t* pos;   // positions [B, t] (null: base + s)
  const uint8_t* keep;
  int64_t keep_b, keep_s;
  const double* rates;
  int w_dt;
  float eps, magnitude;
  int rot, t, heads, kvh, dim;
  int head_chunk;         // heads a workgroup takes
  int chunks;             // workgroups a token
  int64_t row_groups;     // workgroups that rotate; the others write v
  int v_blocks, v_parts;  // cache blocks a lane's t rows can touch, and workgroups a block
};

template <typename T>
__device__ inline void rot_load8(const T* p, float* v) {
  load8(p, sizeof(T) == 4 ? MTPK_F32 : MTPK_BF16, 0, v);
}

// Physical block and slot of a position through a lane's table; -1 where there is none.
__device__ inline int64_t rot_block(const RotArgs& a, int b, int64_t p) {
  if (p < 0 || p / kCacheBlock >= a.table_stride) return -1;
  const int64_t blk = a.table[b * a.table_stride + p / kCacheBlock];
  return blk < 0 || (blk + 1) * kCacheBlock > a.pool_rows ? -1 : blk;
}

// The v rows of one cache block of one lane, transposed into its [kv head, channel, slot] slab: a
// thread takes two adjacent channels of up to 16 rows, so that it reads 4 bytes a row (256 a wave) and
// writes 64 adjacent bytes where the whole block is there.
__device__ inline void rot_write_v(const RotArgs& a, int64_t id) {
  const int part = (int)(id % a.v_parts);
  id /= a.v_parts;
  const int j = (int)(id % a.v_blocks), b = (int)(id / a.v_blocks);
  const int c2 = part * 256 + threadIdx.x;  // pair of channels, over all kv heads
  if (c2 >= a.kvh * a.dim / 2) return;
  const int h = 2 * c2 / a.dim, d = 2 * c2 - h * a.dim;
  const int64_t base = a.base[b];
  const int64_t first = (base >= 0 ? base / kCacheBlock : -((-base + kCacheBlock - 1) / kCacheBlock)) + j;
  const int64_t blk = rot_block(a, b, first * kCacheBlock);
  if (blk < 0) return;
  uint32_t w[kCacheBlock];
  uint32_t live = 0;
#pragma unroll
  for (int e = 0; e < kCacheBlock; ++e) {
    const int64_t s = first * kCacheBlock + e - base;
    const bool in = s >= 0 && s < a.t && (!a.keep || a.keep[b * a.keep_b + s * a.keep_s]);
    live |= (uint32_t)in << e;
    w[e] = in ? *reinterpret_cast<const uint32_t*>(a.v + b * a.vs.b + h * a.vs.h + s * a.vs.s + d) : 0u;
  }
  uint16_t* const to = a.v_pool + ((blk * a.kvh + h) * a.dim + d) * kCacheBlock;
  if (live == 0xffffu) {
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        u32x4_t r;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t lo = w[8 * i + 2 * e], hi = w[8 * i + 2 * e + 1];
          r[e] = x == 0 ? (lo & 0xffffu) | (hi << 16) : (lo >> 16) | (hi & 0xffff0000u);
        }
        *reinterpret_cast<u32x4_t*>(to + x * kCacheBlock + 8 * i) = r;
      }
    return;
  }
#pragma unroll
  for (int e = 0; e < kCacheBlock; ++e)
    if (live >> e & 1) {
      to[e] = (uint16_t)(w[e] & 0xffffu);
      to[kCacheBlock + e] = (uint16_t)(w[e] >> 16);
    }
}

template <typename T, int G, int PAIRS, bool CACHE>
__global__ __launch_bounds__(256) void k_rotate(RotArgs a) {
  constexpr int U = 4;  // rows in flight per lane
  __shared__ float2 turn[kRotMaxDim / 2];
  if (CACHE && blockIdx.x >= a.row_groups) return rot_write_v(a, blockIdx.x - a.row_groups);
  const int tid = threadIdx.x, gl = tid % G, e0 = gl * 8;
  const int64_t tok = blockIdx.x / a.chunks;
  const int part = (int)(blockIdx.x - tok * a.chunks);
  const int b = (int)(tok / a.t), s = (int)(tok - (int64_t)b * a.t);
  const int all = a.heads + (CACHE ? a.kvh : 0);
  const int h0 = part * a.head_chunk, h1 = min(h0 + a.head_chunk, all);
  const int half = a.rot / 2;
  const bool lane_in = e0 < a.dim;
  const int64_t p = a.pos ? a.pos[tok] : a.base[b] + s;
  const T* const q0 = static_cast<const T*>(a.q) + b * a.qs.b + s * a.qs.s;
  const T* const k0 = CACHE ? reinterpret_cast<const T*>(a.k) + b * a.ks.b + s * a.ks.s : nullptr;
  auto row = [&](int h) { return CACHE && h >= a.heads ? k0 + (h - a.heads) * a.ks.h : q0 + h * a.qs.h; };
  int64_t krow = -1;  // this token's pool row
  if (CACHE && h1 > a.heads && (!a.keep || a.keep[b * a.keep_b + s * a.keep_s])) {
    const int64_t at = a.base[b] + s, blk = rot_block(a, b, at);
    krow = blk < 0 ? -1 : blk * kCacheBlock + at % kCacheBlock;
  }
  float c8[8], s8[8], w[8], wp[8];
  bool have = false, k_now = false;
  for (int hb = h0 + tid / G; hb - tid / G < h1; hb += U * (256 / G)) {
    float v[U][8], pv[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = hb + u * (256 / G);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[u][j] = pv[u][j] = 0.f;
      if (h < h1 && lane_in) {
        const T* const r = row(h);
        rot_load8(r + e0, v[u]);
        if (PAIRS == kHalves) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int e = e0 + j;
            if (e < a.rot) pv[u][j] = load_float(r, sizeof(T) == 4 ? MTPK_F32 : MTPK_BF16, e < half ? e + half : e - half);
          }
        }
      }
    }
    if (!have) {  // uniform: the token's turns, while the first rows are on their way
      have = true;
      if (tid < half) {
        const double rev = (double)p * (a.rates[tid] * 0.15915494309189533577);
        float sn, cs;
        sincospif(2.f * (float)(rev - rint(rev)), &sn, &cs);
        turn[tid] = make_float2(cs * a.magnitude, sn * a.magnitude);
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int e = e0 + j;
        c8[j] = 1.f;
        s8[j] = 0.f;
        if (e < a.rot) {
          const bool low = PAIRS == kAdjacent ? (j & 1) == 0 : e < half;
          const float2 cs = turn[PAIRS == kAdjacent ? e / 2 : low ? e : e - half];
          c8[j] = cs.x;
          s8[j] = low ? -cs.y : cs.y;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = hb + u * (256 / G);
      const bool k_row = CACHE && h >= a.heads;
      const void* const wt = k_row ? a.kw : a.qw;
      if (wt) {
        if ((u == 0 && hb == h0 + tid / G) || k_row != k_now) {  // the first row, or the first of k
          k_now = k_row;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int e = e0 + j;
            w[j] = lane_in ? 1.f + load_float(wt, a.w_dt, e) : 0.f;
            const int pe = PAIRS == kAdjacent ? (e ^ 1) : e < half ? e + half : e - half;
            wp[j] = e < a.rot && lane_in ? 1.f + load_float(wt, a.w_dt, pe) : 0.f;
          }
        }
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss += v[u][j] * v[u][j];
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o, kWave);
        const float inv = rsqrtf(ss / (float)a.dim + a.eps);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[u][j] = v[u][j] * inv;
          pv[u][j] = pv[u][j] * inv;
        }
      }
      if (PAIRS == kAdjacent) {
#pragma unroll
        for (int j = 0; j < 8; ++j) pv[u][j] = v[u][j ^ 1];
      }
      if (PAIRS == kHalvesOf8) {
        const int lane = tid & (kWave - 1), from = e0 < half ? lane + half / 8 : lane - half / 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) pv[u][j] = __shfl(v[u][j], from & (kWave - 1), kWave);
      }
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x = wt ? v[u][j] * w[j] : v[u][j];
        const float xp = wt ? pv[u][j] * wp[j] : pv[u][j];
        y[j] = e0 + j < a.rot ? x * c8[j] + xp * s8[j] : x;
      }
      if (h >= h1 || !lane_in) continue;
      T* to;
      if (k_row) {
        if (krow < 0) continue;
        to = reinterpret_cast<T*>(a.k_pool) + (krow * a.kvh + (h - a.heads)) * a.dim;
      } else {
        to = static_cast<T*>(a.out) + b * a.os.b + h * a.os.h + s * a.os.s;
      }
      store8(to, sizeof(T) == 4 ? MTPK_F32 : MTPK_BF16, e0, y);
    }
  }
}

namespace {

template <typename T, int PAIRS, bool CACHE>
int rotate_g(const RotArgs& a, unsigned grid, hipStream_t st) {
  const int need = a.dim / 8;
#define MTPK_ROT(G_) hipLaunchKernelGGL((k_rotate<T, G_, PAIRS, CACHE>), dim3(grid), dim3(256), 0, st, a)
  if (need <= 2) MTPK_ROT(2);
  else if (need <= 4) MTPK_ROT(4);
  else if (need <= 8) MTPK_ROT(8);
  else if (need <= 16) MTPK_ROT(16);
  else if (need <= 32) MTPK_ROT(32);
  else MTPK_ROT(64);
#undef MTPK_ROT
  return status_of(hipGetLastError());
}

template <typename T, bool CACHE>
int rotate_launch(RotArgs& a, int64_t tokens, int interleaved, hipStream_t st) {
  int g = 2;
  while (g * 8 < a.dim) g *= 2;
  const int all = a.heads + (CACHE ? a.kvh : 0), step = 256 / g;
  // A workgroup a token where tokens fill the chip; else as many as the token's heads fill.
  const int fine = (all + step - 1) / step;
  a.chunks = tokens * fine <= 4096 ? fine : 1;
  a.head_chunk = a.chunks == 1 ? all : step;
  a.row_groups = tokens * a.chunks;
  int64_t grid = a.row_groups;
  if (CACHE) {
    a.v_blocks = (a.t + kCacheBlock - 2) / kCacheBlock + 1;
    a.v_parts = (a.kvh * a.dim / 2 + 255) / 256;
    grid += tokens / a.t * a.v_blocks * a.v_parts;
  }
  if (grid > INT32_MAX) return MTPK_EINVAL;
  if (interleaved) return rotate_g<T, kAdjacent, CACHE>(a, (unsigned)grid, st);
  if (a.rot % 16 == 0) return rotate_g<T, kHalvesOf8, CACHE>(a, (unsigned)grid, st);
  return rotate_g<T, kHalves, CACHE>(a, (unsigned)grid, st);
}

bool rot_ok(int64_t dim, int rot, const double* rates, float eps) {
  if (dim < 8 || dim % 8 || dim > kRotMaxDim) return false;
  return rot >= 2 && rot % 2 == 0 && rot <= dim && rates && eps >= 0.f;
}

bool strides8(const int64_t* s, int unit) { return s[0] % unit == 0 && s[1] % unit == 0 && s[2] % unit == 0; }

}  // namespace
}  // namespace mtpk

using namespace mtpk;

extern "C" {

int mtpk_rotate(const void* x, int dtype, const int64_t* x_strides, int64_t tokens, int64_t heads,
                int64_t dim, const void* w, int w_dtype, float eps, const int64_t* pos,
                const double* rates, int rot_dim, int interleaved, float magnitude, void* out,
                const int64_t* out_strides, void* stream) {
  if (!x || !out || !pos || !x_strides || !out_strides) return MTPK_EINVAL;
  if ((dtype != MTPK_F32 && dtype != MTPK_BF16) || (w && w_dtype != MTPK_F32 && w_dtype != MTPK_BF16)) return MTPK_EINVAL;
  if (!rot_ok(dim, rot_dim, rates, eps) || tokens < 0 || heads < 1 || heads > 65535) return MTPK_EINVAL;
  const int unit = dtype == MTPK_F32 ? 4 : 8;  // 16-byte accesses
  if (!aligned16(x) || !aligned16(out) || x_strides[0] % unit || x_strides[1] % unit || out_strides[0] % unit ||
      out_strides[1] % unit)
    return MTPK_EINVAL;
  if (tokens == 0) return 0;
  if (tokens > INT32_MAX) return MTPK_EINVAL;
  RotArgs a{};
  a.q = x;
  a.qs = {x_strides[0], x_strides[1], 0};  // a token a lane, of one step
  a.qw = w;
  a.out = out;
  a.os = {out_strides[0], out_strides[1], 0};
  a.pos = pos;
  a.rates = rates;
  a.w_dt = w_dtype;
  a.eps = eps;
  a.magnitude = magnitude;
  a.rot = rot_dim;
  a.t = 1;
  a.heads = (int)heads;
  a.dim = (int)dim;
  const hipStream_t st = (hipStream_t)stream;
  return dtype == MTPK_F32 ? rotate_launch<float, false>(a, tokens, interleaved, st)
                           : rotate_launch<uint16_t, false>(a, tokens, interleaved, st);
}

int mtpk_rotate_to_cache(const uint16_t* q, const int64_t* q_strides, const uint16_t* k,
                         const int64_t* k_strides, const uint16_t* v, const int64_t* v_strides,
                         const void* q_norm, const void* k_norm, int norm_dtype, float eps,
                         const double* rates, int rot_dim, int interleaved, float magnitude,
                         uint16_t* k_pool, uint16_t* v_pool, int64_t pool_rows,
                         const int32_t* block_table, int64_t table_stride, const int64_t* base_pos,
                         const int64_t* positions, const uint8_t* keep, int64_t keep_b, int64_t keep_s,
                         int64_t batch, int64_t t, int64_t heads, int64_t kv_heads, int64_t head_dim,
                         uint16_t* out, const int64_t* out_strides, void* stream) {
  if (!q || !k || !v || !k_pool || !v_pool || !block_table || !base_pos || !out) return MTPK_EINVAL;
  if (!q_strides || !k_strides || !v_strides || !out_strides) return MTPK_EINVAL;
  if (!rot_ok(head_dim, rot_dim, rates, eps)) return MTPK_EINVAL;
  if ((q_norm || k_norm) && norm_dtype != MTPK_F32 && norm_dtype != MTPK_BF16) return MTPK_EINVAL;
  if (batch < 0 || t < 1 || heads < 1 || kv_heads < 1 || heads > 65535 || kv_heads > 65535) return MTPK_EINVAL;
  if (pool_rows <= 0 || pool_rows % kCacheBlock || table_stride <= 0) return MTPK_EINVAL;
  if (keep && (keep_b < 0 || keep_s < 0)) return MTPK_EINVAL;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || !aligned16(k_pool) || !aligned16(v_pool))
    return MTPK_EINVAL;
  if (!strides8(q_strides, 8) || !strides8(k_strides, 8) || !strides8(v_strides, 8) || !strides8(out_strides, 8))
    return MTPK_EINVAL;
  if (batch == 0) return 0;
  if (batch > INT32_MAX / t) return MTPK_EINVAL;
  RotArgs a{};
  a.q = q;
  a.qs = {q_strides[0], q_strides[1], q_strides[2]};
  a.qw = q_norm;
  a.out = out;
  a.os = {out_strides[0], out_strides[1], out_strides[2]};
  a.k = k;
  a.ks = {k_strides[0], k_strides[1], k_strides[2]};
  a.kw = k_norm;
  a.v = v;
  a.vs = {v_strides[0], v_strides[1], v_strides[2]};
  a.k_pool = k_pool;
  a.v_pool = v_pool;
  a.pool_rows = pool_rows;
  a.table = block_table;
  a.table_stride = table_stride;
  a.base = base_pos;
  a.pos = positions;
  a.keep = keep;
  a.keep_b = keep_b;
  a.keep_s = keep_s;
  a.rates = rates;
  a.w_dt = norm_dtype;
  a.eps = eps;
  a.magnitude = magnitude;
  a.rot = rot_dim;
  a.t = (int)t;
  a.heads = (int)heads;
  a.kvh = (int)kv_heads;
  a.dim = (int)head_dim;
  return rotate_launch<uint16_t, true>(a, batch * t, interleaved, (hipStream_t)stream);
}

}  // extern "C"
