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
// A lane holds 8 adjacent channels of a head (16 bytes of bf16), G lanes a head, 256 / G such slots a
// workgroup. A slot takes some heads of one token, all of them where tokens fill the chip: its lanes
// compute the token's turns into LDS of their own (no barrier: a slot lies inside a wave), and a lane's
// cos, sin and weights stay in registers from head to head. The partner of a channel is in the lane's own
// 8 (adjacent pairs), or read again from memory, 16 bytes at once where a half is whole 8s: those lines
// are in L1. Bound by the bytes of the heads, read once and written once. (A workgroup a token, its turns by the
// first lanes behind a barrier and partners by shuffles, took 203 us for 8000 tokens of 34 heads, where this
// form takes 70: the instructions.)

#include <algorithm>

#include "mtpk_device.h"
#include "mtpk_host.h"

namespace mtpk {

constexpr int kRotMaxDim = 512;
constexpr int kCacheBlock = 16;  // rows of a cache block

enum RotPairs { kAdjacent = 0, kHalvesOf8 = 1, kHalves = 2 };  // of 16 channels, of any even number

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
  int64_t tokens;
  int head_chunk, chunks;  // heads a slot takes, and slots a token
  int v_groups;            // workgroups that write v, the first ones
  int v_blocks, v_parts;   // cache blocks a lane's t rows can touch, and workgroups a block
};

// Sum over a slot's G lanes, in every one of them.
template <int G>
__device__ inline float slot_sum(float v) {
  if (G >= 2) v += dpp_mov<0xB1>(v);
  if (G >= 4) v += dpp_mov<0x4E>(v);
  if (G >= 8) v += dpp_mov<0x141>(v);
  if (G >= 16) v += dpp_mov<0x140>(v);
#pragma unroll
  for (int o = 16; o < G; o *= 2) v += __shfl_xor(v, o, kWave);
  return v;
}

// Eight channels as they lie in memory.
template <typename T>
struct Raw8 {
  u32x4_t d[sizeof(T) / 2];
  __device__ inline void zero() {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) d[i] = zero16();
  }
  __device__ inline void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) d[i] = ld16(p + i * (16 / sizeof(T)));
  }
  __device__ inline void get(float* v) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (sizeof(T) == 4)
        v[j] = bits_f32(d[j / 4][j % 4]);
      else
        v[j] = bits_f32(j & 1 ? d[0][j / 2] & 0xffff0000u : d[0][j / 2] << 16);
    }
  }
};

// sin and cos of f turns, |f| <= 1/2: the quarter turn next to f, and the Taylor sums of the rest x, at most
// an eighth of a turn, up to x^9 and x^10 (x in radians below 0.786: the next terms are below 2e-9).
__device__ inline void sincos_turn(float f, float& s, float& c) {
  const float k = rintf(f * 4.f), r = fmaf(k, -0.25f, f), x = r * 6.28318530717958648f, u = x * x;
  const float sn = x * fmaf(u, fmaf(u, fmaf(u, fmaf(u, 2.75573192e-6f, -1.98412698e-4f), 8.33333333e-3f), -1.66666667e-1f), 1.f);
  const float cs = fmaf(u, fmaf(u, fmaf(u, fmaf(u, fmaf(u, -2.75573192e-7f, 2.48015873e-5f), -1.38888889e-3f), 4.16666667e-2f), -0.5f), 1.f);
  const int q = (int)k & 3;
  const float a = q & 1 ? cs : sn, b = q & 1 ? sn : cs;
  s = q & 2 ? -a : a;
  c = q == 1 || q == 2 ? -b : b;
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
  constexpr int U = sizeof(T) == 4 ? 1 : 4, kDt = sizeof(T) == 4 ? MTPK_F32 : MTPK_BF16;  // heads in flight per slot
  __shared__ float2 turns[1024];  // 256 / G slots of at most 4 G pairs
  if (CACHE && (int)blockIdx.x < a.v_groups) return rot_write_v(a, blockIdx.x);
  const int tid = threadIdx.x, gl = tid % G, e0 = gl * 8, half = a.rot / 2;
  const int64_t slot = (int64_t)((int)blockIdx.x - a.v_groups) * (256 / G) + tid / G;
  int64_t tok = slot / a.chunks;
  const int part = (int)(slot - tok * a.chunks);
  const int all = a.heads + (CACHE ? a.kvh : 0);
  const int h0 = part * a.head_chunk, h1 = tok < a.tokens ? min(h0 + a.head_chunk, all) : h0;
  tok = min(tok, a.tokens - 1);
  const int b = (int)(tok / a.t), s = (int)(tok - (int64_t)b * a.t);
  const bool lane_in = e0 < a.dim;
  const T* const q0 = static_cast<const T*>(a.q) + b * a.qs.b + s * a.qs.s;
  const T* const k0 = CACHE ? reinterpret_cast<const T*>(a.k) + b * a.ks.b + s * a.ks.s : nullptr;
  auto row = [&](int h) { return CACHE && h >= a.heads ? k0 + (h - a.heads) * a.ks.h : q0 + h * a.qs.h; };
  const int p0 = e0 < half ? e0 + half : e0 - half;  // the partners' first channel (halves)
  Raw8<T> raw[U], rawp[U];
  auto load = [&](int h) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      raw[u].zero();
      rawp[u].zero();
      if (h + u < h1 && lane_in) {
        raw[u].load(row(h + u) + e0);
        if (PAIRS == kHalvesOf8 && e0 < a.rot) rawp[u].load(row(h + u) + p0);
      }
    }
  };
  load(h0);
  // weights as 1 + w, of the lane's channels and of their partners
  float w[8], wp[8];
  const void* wt = nullptr;
  auto weights = [&](const void* from) {
    wt = from;
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = wp[j] = 0.f;
    if (!wt || !lane_in) return;
    load8(wt, a.w_dt, e0, w);
    if (PAIRS == kHalvesOf8 && e0 < a.rot) load8(wt, a.w_dt, p0, wp);
    if (PAIRS == kHalves)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (e0 + j < a.rot) wp[j] = load_float(wt, a.w_dt, e0 + j < half ? e0 + j + half : e0 + j - half);
    if (PAIRS == kAdjacent)
#pragma unroll
      for (int j = 0; j < 8; ++j) wp[j] = w[j ^ 1];
  };
  weights(CACHE && h0 >= a.heads ? a.kw : a.qw);
  int64_t krow = -1;  // this token's pool row
  if (CACHE && h1 > a.heads && (!a.keep || a.keep[b * a.keep_b + s * a.keep_s])) {
    const int64_t at = a.base[b] + s, blk = rot_block(a, b, at);
    krow = blk < 0 ? -1 : blk * kCacheBlock + at % kCacheBlock;
  }
  // the token's turns, a pair a lane
  float2* const turn = turns + tid / G * half;
  {
    const double p = (double)(a.pos ? a.pos[tok] : a.base[b] + s);
    for (int i = gl; i < half; i += G) {
      const double rev = p * (a.rates[i] * 0.15915494309189533577);
      float sn, cs;
      sincos_turn((float)(rev - rint(rev)), sn, cs);
      turn[i] = make_float2(cs * a.magnitude, sn * a.magnitude);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  // y = inv * (x cw + partner sw)
  float cw[8], sw[8];
  auto factors = [&]() {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int e = e0 + j;
      cw[j] = 1.f;
      sw[j] = 0.f;
      if (e < a.rot) {
        const bool low = PAIRS == kAdjacent ? (j & 1) == 0 : e < half;
        const float2 cs = turn[PAIRS == kAdjacent ? e / 2 : low ? e : e - half];
        cw[j] = cs.x;
        sw[j] = low ? -cs.y : cs.y;
      }
      if (wt) {
        cw[j] *= 1.f + w[j];
        sw[j] *= 1.f + wp[j];
      }
    }
  };
  factors();
  const float per = 1.f / (float)a.dim;
  for (int h = h0; h < h1; h += U) {
    if (h > h0) load(h);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int hu = h + u;
      if (hu >= h1) break;
      const bool k_row = CACHE && hu >= a.heads;
      if (CACHE && hu == a.heads && hu > h0) {  // from the q heads to the k heads
        weights(a.kw);
        factors();
      }
      float v[8], pv[8];
      raw[u].get(v);
      rawp[u].get(pv);
      if (PAIRS == kAdjacent) {
#pragma unroll
        for (int j = 0; j < 8; ++j) pv[j] = e0 + j < a.rot ? v[j ^ 1] : 0.f;
      }
      if (PAIRS == kHalves) {
        const T* const r = row(hu);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (e0 + j < a.rot) pv[j] = load_float(r, kDt, e0 + j < half ? e0 + j + half : e0 + j - half);
      }
      float inv = 1.f;
      if (wt) {
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(v[j], v[j], ss);
        inv = rsqrtf(fmaf(slot_sum<G>(ss), per, a.eps));
      }
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = inv * fmaf(pv[j], sw[j], v[j] * cw[j]);
      if (!lane_in || (k_row && krow < 0)) continue;
      T* const to = k_row ? reinterpret_cast<T*>(a.k_pool) + (krow * a.kvh + (hu - a.heads)) * a.dim
                          : static_cast<T*>(a.out) + b * a.os.b + hu * a.os.h + s * a.os.s;
      store8(to, kDt, e0, y);
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
  const int all = a.heads + (CACHE ? a.kvh : 0), slots = 256 / g;
  // Slots for four waves a SIMD, a token's heads shared out evenly among its own: few tokens take a slot a
  // head, many one for all of their heads. 4099 tokens of 16 fp32 heads of 128: 13.4 us a pass (5.0 TB/s) with
  // four slots a token, 18.8 with two, 17.4 with sixteen; 8000 tokens of 34 heads of 256 into the cache: 69.6
  // (4.2 TB/s) with one, 72.5 with two of 17 heads, 97 with 33 heads in one and the last in another.
  const int64_t want = (int64_t)device_cu_count() * 4 * slots;
  a.chunks = (int)std::min<int64_t>(std::max<int64_t>((want + tokens / 2) / tokens, 1), all);
  a.head_chunk = (all + a.chunks - 1) / a.chunks;
  a.chunks = (all + a.head_chunk - 1) / a.head_chunk;
  a.tokens = tokens;
  int64_t grid = (tokens * a.chunks + slots - 1) / slots;
  if (CACHE) {
    a.v_blocks = (a.t + kCacheBlock - 2) / kCacheBlock + 1;
    a.v_parts = (a.kvh * a.dim / 2 + 255) / 256;
    const int64_t v_groups = tokens / a.t * a.v_blocks * a.v_parts;
    if (v_groups > INT32_MAX) return MTPK_EINVAL;
    a.v_groups = (int)v_groups;
    grid += v_groups;
  }
  if (grid > kMaxGroups) return MTPK_EINVAL;
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
  if (!aligned16(x) || !aligned16(out) || (w && !aligned16(w)) || x_strides[0] % unit || x_strides[1] % unit || out_strides[0] % unit ||
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
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || !aligned16(k_pool) || !aligned16(v_pool) ||
      (q_norm && !aligned16(q_norm)) || (k_norm && !aligned16(k_norm)))
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
