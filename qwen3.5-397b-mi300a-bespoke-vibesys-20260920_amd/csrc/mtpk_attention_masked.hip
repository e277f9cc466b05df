// Attention over the paged bf16 KV cache whose scores are capped, biased by distance or masked beyond
// the causal order. For the query row at position p of lane b, q head h, and the key at position j:
//   x = scale * q . k_j;   x = cap * tanh(x / cap) with a cap;   x -= slope_h * |p - j| with slopes
//   seen: first <= j, p - j < window (with one), and j <= p or both below the lane's prefix end
//   out = sum softmax(x)_j v_j over the seen j, 0 where none is; times sigmoid(gate) with a gate
// The first three conditions and the prefix make an interval [lo, hi) of keys per row, so a row group
// reads only the tiles between its rows' first and last key, and only the tiles that some row sees in
// part are masked, score by score.
//
// Both forms work on tiles of 32 keys by 32 query rows with both products transposed, so that a lane
// holds one query row (rows token by token: row r = step r / group, q head r % group of a kv head):
//   S^T = K Q^T   v_mfma_f32_32x32x16_bf16, A = 32 keys from LDS, B = Q (registers)
//   O^T += V^T P^T  A = V^T from LDS (the cache's own layout), B = P
// Row m of a K tile is its key with bits 2 and 3 of m swapped: then the S^T values that a lane gets
// are 8 adjacent keys of each 16, which is the B operand of O^T, and P never leaves its registers. Tiles
// go straight to LDS, their 16-byte pieces permuted on the way so that the reads fall on all banks. Every
// block of a tile is a buffer of its own, based in 64 bits: the pools may be of any size.
//
// Sums and statistics are fp32. P is rounded to bf16 for the second product, and the row sum adds the
// rounded values, so that a row's weights sum to 1 as they are used. The output, with its gate, is
// rounded once.
//
// Keys that a row does not see may hold anything: their scores are replaced, and where a tile that is
// masked for some row holds a V value that is not finite, its second product takes a form of its own
// (0 times infinity would be NaN in the rows that do not see it).

#include <algorithm>

#include "mtpk_attention_common.h"
#include "mtpk_host.h"

namespace mtpk {

constexpr int kTileKeys = 32;
constexpr int kMaskedSplits = 64;       // key splits the merge takes
constexpr float kLog2e = 1.4426950408889634f;

struct MaskedArgs {
  const uint16_t* q;
  AttnRows qr;
  uint16_t* out;
  AttnRows orow;
  const uint16_t* gate;  // may be null
  AttnRows gr;
  const uint16_t* k_pool;
  const uint16_t* v_pool;
  int64_t pool_rows;
  const int32_t* table;
  int64_t table_stride;
  const int64_t* base;
  const float* slopes;  // per q head, may be null
  const void* prefix;   // per lane, may be null
  const void* first;    // per lane and step, may be null
  int prefix_dt, first_dt;
  int window;  // 0: none
  int t, heads, kvh, lanes_kvh;
  int n_split, row_groups;
  float scale2;                 // scale * log2(e)
  float cap2;                   // cap * log2(e), 0: none
  float cap_in;                 // 2 * log2(e) * scale / cap
  float poly_max, c0, c1, c2, c3;  // cap2 * tanh(s scale / cap) as s (c0 + c1 s^2 + ..) up to |s| = poly_max
  float* part_o;
  float* part_ml;
};

// The keys [lo, hi) that a row sees, and its position.
struct RowKeys {
  int pos, lo, hi;
};

__device__ inline RowKeys masked_row(const MaskedArgs& a, int b, int s) {
  const int64_t base = a.base[b], pos = base + s;
  int64_t lo = 0, hi = pos + 1;
  if (a.prefix) {
    const int64_t edge = load_index(a.prefix, a.prefix_dt, b);
    if (pos < edge) hi = edge;
  }
  if (a.window > 0) lo = max(lo, pos - a.window + 1);
  if (a.first) lo = max(lo, load_index(a.first, a.first_dt, (int64_t)b * a.t + s));
  // never past the rows of this call, nor past the lane's table
  hi = max(min(min(hi, base + a.t), a.table_stride * kAttnBlock), (int64_t)0);
  lo = min(lo, (int64_t)INT32_MAX);
  return RowKeys{(int)pos, (int)lo, (int)hi};
}

__device__ inline int wave_min_i(int v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, kWave));
  return uniform(v);
}
__device__ inline int wave_max_i(int v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor(v, o, kWave));
  return uniform(v);
}

// What 32 rows (the two halves of a wave hold them twice) see together.
struct RowSet {
  int lo_min, lo_max, hi_min, hi_max;
  __device__ inline bool touches(int key0) const { return key0 < hi_max && key0 + kTileKeys > lo_min; }
  __device__ inline bool whole(int key0) const { return key0 >= lo_max && key0 + kTileKeys <= hi_min; }
};
// A row that sees nothing makes no key worth reading, and every tile that another row touches is masked.
__device__ inline RowSet row_set(const RowKeys& r) {
  const bool none = r.hi <= r.lo;
  return RowSet{wave_min_i(none ? INT32_MAX : r.lo), wave_max_i(none ? INT32_MAX : r.lo), wave_min_i(none ? 0 : r.hi),
                wave_max_i(none ? 0 : r.hi)};
}

// The tiles [tile0, tile0 + n) of split `sp` for keys [lo, hi).
__device__ inline void masked_split(int lo, int hi, int n_split, int sp, int& tile0, int& n) {
  tile0 = hi > lo ? lo / kTileKeys : 0;
  const int all = hi > lo ? (hi + kTileKeys - 1) / kTileKeys - tile0 : 0;
  const int per = (all + n_split - 1) / n_split;
  const int from = min(sp * per, all);
  n = min(per, all - from);
  tile0 += from;
}

// Staging of one 16-row block's K or V into LDS by `loads` 1 KB loads: a lane's offsets are the same
// for every block. K as [key][piece ^ prompt_flip(row of the key)], V as [channel][piece ^ (channel / 4 & 1)].
template <int HD>
struct TileGeom {
  static constexpr int kS = HD / 16, kT = HD / 32, kP = HD / 8;  // k steps, channel tiles, 16-byte pieces of a key
  static constexpr int kHalf = kAttnBlock * HD * 2;              // bytes of a block's K (or V) of one kv head
  static constexpr int kTile = 2 * kHalf;
  static constexpr int kLoads = kHalf / 1024;  // 1 KB loads of a block
};

template <int HD>
struct BlockSource {
  rsrc_t k, v;
  __device__ inline BlockSource(const MaskedArgs& a, int blk, bool wanted) {
    const int64_t slab = (int64_t)kAttnBlock * a.kvh * HD;
    const bool ok = wanted && blk >= 0 && (int64_t)(blk + 1) * kAttnBlock <= a.pool_rows;
    const int64_t at = (int64_t)uniform(ok ? blk : 0) * slab;
    const uint32_t bytes = (uint32_t)uniform(ok ? (int)(slab * 2) : 0);  // a block outside the pool reads as zeros
    k = make_rsrc(a.k_pool + at, bytes);
    v = make_rsrc(a.v_pool + at, bytes);
  }
};

// Byte offset of K load j (of kLoads) of a block: 1 KB covers 64 / kP keys.
template <int HD>
__device__ inline uint32_t k_offset(int lane, int kvh, int kh, int half, int j) {
  using G = TileGeom<HD>;
  const int key = j * (64 / G::kP) + lane / G::kP;
  return (uint32_t)(((key * kvh + kh) * HD + ((lane % G::kP) ^ prompt_flip(prompt_swap(16 * half + key))) * 8) * 2);
}
// V load 0; load j is 1 KB further on.
template <int HD>
__device__ inline uint32_t v_offset(int lane, int kh) {
  return (uint32_t)(kh * HD * 32 + (lane >> 1) * 32 + (((lane & 1) ^ (lane >> 3 & 1)) * 16));
}

__device__ inline void load_lds(rsrc_t r, uint8_t* to, uint32_t off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void_t*)to, 16, (int)off, 0, 0, 0);
}

// One row's running softmax: m in units of log2, l over the rounded P.
struct RowSoft {
  float m, l;
};

__device__ inline float cap_exact(const MaskedArgs& a, float s) {
  return fmaf(__builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s * a.cap_in) + 1.f), -2.f * a.cap2, a.cap2);
}
__device__ inline float cap_poly(const MaskedArgs& a, float s) {
  const float u = s * s;
  return s * fmaf(u, fmaf(u, fmaf(u, a.c3, a.c2), a.c1), a.c0);
}

// Scores of a tile (this lane's row, keys key0 + 16 (i / 8) + 8 h + i % 8) into P, and what O has to be
// multiplied by first (1: nothing to do, for the whole wave).
template <bool CAP, bool SLOPES>
__device__ inline float tile_softmax(const MaskedArgs& a, f32x16_t& s, const RowKeys& row, float slope2, bool whole,
                                     int key0, int h, RowSoft& r, bf16x8_t (&p)[2]) {
  bool poly = true;
  if (CAP) {
    float am = fabsf(s[0]);
#pragma unroll
    for (int i = 1; i < 16; ++i) am = fmaxf(am, fabsf(s[i]));
    poly = __ballot(!(am <= a.poly_max)) == 0ull;
  }
  const bool direct = !SLOPES && whole && poly;  // exponents straight from the scores
  float tm;
  if (direct) {
    tm = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) tm = fmaxf(tm, s[i]);
    tm = CAP ? cap_poly(a, tm) : tm * a.scale2;
  } else {
    if (CAP && !poly) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = cap_exact(a, s[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = CAP ? cap_poly(a, s[i]) : s[i] * a.scale2;
    }
    if (SLOPES) {
      const float away = (float)(row.pos - key0 - 8 * h);
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = fmaf(fabsf(away - (float)(16 * (i >> 3) + (i & 7))), -slope2, s[i]);
    }
    if (!whole) {
      const int lo = row.lo - key0 - 8 * h, n = row.hi - row.lo;  // seen: 0 <= i - lo < n, in one comparison
#pragma unroll
      for (int i = 0; i < 16; ++i)
        s[i] = (uint32_t)(16 * (i >> 3) + (i & 7) - lo) < (uint32_t)max(n, 0) ? s[i] : -INFINITY;
    }
    tm = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) tm = fmaxf(tm, s[i]);
  }
  tm = fmaxf(tm, __shfl_xor(tm, 32, kWave));
  const float mn = fmaxf(r.m, tm);
  float alpha = 1.f;
  if (__ballot(mn > r.m) != 0ull) {  // uniform over the wave
    alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(r.m - mn);
    r.m = mn;
    r.l *= alpha;
  }
  const float ms = r.m == -INFINITY ? 0.f : r.m;  // a row with no key so far: every e below is 0
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float x;
    if (direct) {
      if (CAP) {
        const float u = s[i] * s[i];
        x = fmaf(s[i], fmaf(u, fmaf(u, fmaf(u, a.c3, a.c2), a.c1), a.c0), -ms);
      } else {
        x = fmaf(s[i], a.scale2, -ms);
      }
    } else {
      x = s[i] - ms;
    }
    p[i >> 3][i & 7] = (__bf16)__builtin_amdgcn_exp2f(x);
  }
  const bf16x2_t one = {(__bf16)1.f, (__bf16)1.f};
  float part[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    part[i & 1] = __builtin_amdgcn_fdot2_f32_bf16(bf16x2_t{p[i >> 2][2 * (i & 3)], p[i >> 2][2 * (i & 3) + 1]}, one,
                                                  part[i & 1], false);
  r.l += part[0] + part[1];
  return alpha;
}

// Whether a tile of V^T in LDS holds a value that is not finite (each wave looks at the whole tile).
template <int HD>
__device__ inline bool tile_not_finite(const uint8_t* v, uint32_t vat) {
  using G = TileGeom<HD>;
  uint32_t bad = 0;
#pragma unroll 2
  for (int i = 0; i < G::kS; ++i) {
    const u32x4_t w = lds16(v + vat + (i % G::kT) * 1024 + (i / G::kT) * G::kHalf);
#pragma unroll
    for (int e = 0; e < 4; ++e) bad |= (w[e] & 0x7f807f80u) + 0x00800080u;  // carries into bits 15, 31
  }
  return __ballot((bad & 0x80008000u) != 0u) != 0ull;
}

// V values with zeros where they are not finite: what the second product of such a tile takes.
__device__ inline u32x4_t finite_only(u32x4_t w) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t lo = (w[e] & 0x7f80u) == 0x7f80u ? 0u : 0x0000ffffu;
    const uint32_t hi = (w[e] & 0x7f800000u) == 0x7f800000u ? 0u : 0xffff0000u;
    w[e] &= lo | hi;
  }
  return w;
}

// And what is not finite, into the sums of the rows that see it: two products, of ones in its places with
// ones for the keys that a row sees, say where infinities of either sign (NaN: of both) belong.
template <int HD>
__device__ inline void add_not_finite(f32x16_t (&o)[HD / 32], const uint8_t* v, uint32_t vat, const RowKeys& row, int key0,
                                      int h) {
  using G = TileGeom<HD>;
  bf16x8_t seen[2];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int key = key0 + 16 * (i >> 3) + 8 * h + (i & 7);
    seen[i >> 3][i & 7] = (__bf16)(key >= row.lo && key < row.hi ? 1.f : 0.f);
  }
#pragma unroll
  for (int dt = 0; dt < G::kT; ++dt)
#pragma unroll
    for (int sign = 0; sign < 2; ++sign) {
      f32x16_t n;
#pragma unroll
      for (int i = 0; i < 16; ++i) n[i] = 0.f;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        u32x4_t w = lds16(v + vat + dt * 1024 + x * G::kHalf);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t ones = 0;
#pragma unroll
          for (int y = 0; y < 32; y += 16) {
            const uint32_t b = w[e] >> y & 0xffffu;
            ones |= ((b & 0x7fffu) > 0x7f80u || b == (sign ? 0xff80u : 0x7f80u) ? 0x3f80u : 0u) << y;
          }
          w[e] = ones;
        }
        n = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(w), seen[x], n, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) o[dt][i] += n[i] > 0.f ? (sign ? -INFINITY : INFINITY) : 0.f;
      ring_fence();  // the rare path: few of its registers at a time
    }
}

// A row's sum is NaN where it saw keys and all of them at minus infinity, 0 where it saw none.
__device__ inline float row_sum(float m, float l, bool seen) { return seen && m == -INFINITY ? __builtin_nanf("") : l; }
__device__ inline bool row_sees(const RowKeys& row, int k0, int k1) { return max(row.lo, k0) < min(row.hi, k1); }

__device__ inline float row_inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }

__device__ inline float sigmoid_of(uint16_t g) {
  // exp2 and reciprocal, 1 ulp each; scaled, as the reciprocal of a value above 2^126 would be flushed
  return __builtin_amdgcn_rcpf((1.f + __builtin_amdgcn_exp2f(-kLog2e * bf16_to_f32(g))) * 0x1p-32f) * 0x1p-32f;
}

// Eight values of an output row, gated, rounded once.
__device__ inline void store_out8(const MaskedArgs& a, int b, int hq, int st, int d, const float* v) {
  float y[8];
  uint16_t* const to = a.out + a.orow.at(b, hq, st) + d;
  if (a.gate) {
    const u32x4_t g = ld16(a.gate + a.gr.at(b, hq, st) + d);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      y[2 * e] = v[2 * e] * sigmoid_of((uint16_t)(g[e] & 0xffffu));
      y[2 * e + 1] = v[2 * e + 1] * sigmoid_of((uint16_t)(g[e] >> 16));
    }
    store8(to, MTPK_BF16, 0, y);
  } else {
    store8(to, MTPK_BF16, 0, v);
  }
}

// ---------------------------------------------------------------- many rows
//
// W waves of 32 rows to a workgroup, tiles shared by its waves, one tile ahead in two buffers with one
// barrier per tile: prompts, and verify rows of more than one wave.
template <int HD, int W, bool CAP, bool SLOPES>
__global__ __launch_bounds__(W* kWave, 2) void k_masked_rows(MaskedArgs a) {
  using G = TileGeom<HD>;
  constexpr int kRows = 32 * W;
  __shared__ __attribute__((aligned(16))) uint8_t smem[4 * G::kTile];  // two buffers of (K, V)
  __shared__ int wg_lo[W], wg_hi[W];
  const int group = a.heads / a.kvh, R = group * a.t;
  const int rg = a.row_groups - 1 - (int)blockIdx.x / a.lanes_kvh;  // the last rows, which see most, first
  const int bkh = (int)blockIdx.x % a.lanes_kvh, kh = bkh % a.kvh, b = bkh / a.kvh, sp = blockIdx.y;
  const int tid = threadIdx.x, wave = uniform(tid / kWave), lane = tid & (kWave - 1);
  const int h = lane >> 5, c = lane & 31;
  const int r = min(kRows * rg + 32 * wave + c, R - 1);  // rows past R repeat the last one
  const int step = r / group, hq = kh * group + r % group;
  const RowKeys row = masked_row(a, b, step);
  const RowSet set = row_set(row);
  if (lane == 0) {
    wg_lo[wave] = set.lo_min;
    wg_hi[wave] = set.hi_max;
  }
  __syncthreads();
  int lo = wg_lo[0], hi = wg_hi[0];
#pragma unroll
  for (int w = 1; w < W; ++w) {
    lo = min(lo, wg_lo[w]);
    hi = max(hi, wg_hi[w]);
  }
  lo = uniform(lo);
  hi = uniform(hi);
  int tile0, tiles;
  masked_split(lo, hi, a.n_split, sp, tile0, tiles);
  tile0 = uniform(tile0);
  tiles = uniform(tiles);

  bf16x8_t q[G::kS];
  {
    const uint16_t* const qrow = a.q + a.qr.at(b, hq, step) + 8 * h;
    u32x4_t d[G::kS];
#pragma unroll
    for (int s = 0; s < G::kS; ++s) d[s] = ld16(qrow + 16 * s);
#pragma unroll
    for (int s = 0; s < G::kS; ++s) {
      asm volatile("" : "+v"(d[s]));  // landed before the loop: its waits count the tiles' loads alone
      q[s] = as_bf16x8(d[s]);
    }
  }
  const float slope2 = SLOPES ? a.slopes[hq] * kLog2e : 0.f;
  const int32_t* const trow = a.table + (int64_t)b * a.table_stride;
  const int last_block = (int)min(a.table_stride, (int64_t)INT32_MAX) - 1;

  // This wave loads one of the tile's two blocks, or half of one, K and V.
  constexpr int kShare = W / 2, kMine = G::kLoads / kShare;
  const int half = wave / kShare;
  uint32_t koff[kMine];
#pragma unroll
  for (int j = 0; j < kMine; ++j) koff[j] = k_offset<HD>(lane, a.kvh, kh, half, (wave % kShare) * kMine + j);
  const uint32_t voff = v_offset<HD>(lane, kh) + (uint32_t)((wave % kShare) * kMine * 1024);
  auto block = [&](int key0) { return sload(trow, min(key0 / kAttnBlock + half, last_block)); };
  auto stage = [&](int buf, int key0, int blk) {
    const int at = key0 + kAttnBlock * half;
    const BlockSource<HD> src(a, uniform(blk), at < hi && at + kAttnBlock > lo);
    uint8_t* const to = smem + buf + wave * (kMine * 1024);
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      load_lds(src.k, to + j * 1024, koff[j]);
      load_lds(src.v, to + G::kTile + j * 1024, voff + 1024u * j);
    }
  };

  RowSoft soft{-INFINITY, 0.f};
  f32x16_t o[G::kT];
#pragma unroll
  for (int dt = 0; dt < G::kT; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;
  // this lane's K pieces: 2 s + h of tile row c, whose place is that of piece h with bits of s flipped
  const uint32_t kat = (uint32_t)(prompt_swap(c) * HD * 2 + ((h ^ prompt_flip(c)) * 16));
  // and its V^T keys: 8 h .. 8 h + 7 of each block, channel 32 dt + c
  const uint32_t vat = (uint32_t)(c * 32 + (h ^ (c >> 2 & 1)) * 16);

  int key0 = tile0 * kTileKeys, buf = 0, next = 0;
  if (tiles > 0) {
    stage(0, key0, block(key0));
    next = block(key0 + kTileKeys);
  }
  for (int n = 0; n < tiles; ++n, key0 += kTileKeys, buf ^= 2 * G::kTile) {
    ring_fence();
    vmcnt_wait<0>();  // this tile, issued a tile ago
    __builtin_amdgcn_s_barrier();
    ring_fence();
    if (n + 1 < tiles) {
      stage(buf ^ (2 * G::kTile), key0 + kTileKeys, next);  // last read a tile ago, before the barrier
      next = block(key0 + 2 * kTileKeys);
    }
    ring_fence();
    if (!set.touches(key0)) continue;
    const bool whole = set.whole(key0);
    const uint8_t* const kt = smem + buf;
    const uint8_t* const vt = smem + buf + G::kTile;
    f32x16_t s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.f;
    // operands come from LDS four products ahead, fenced
    u32x4_t f[4];
    auto kfrag = [&](int i) { return lds16(kt + (kat ^ (32u * (i & 3))) + 128 * (i >> 2)); };
    auto vfrag = [&](int i) { return lds16(vt + vat + (i % G::kT) * 1024 + (i / G::kT) * G::kHalf); };
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = kfrag(i);
    ring_fence();
#pragma unroll
    for (int i = 0; i < G::kS; ++i) {
      s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(f[i & 3]), q[i], s, 0, 0, 0);
      f[i & 3] = i + 4 < G::kS ? kfrag(i + 4) : vfrag(i + 4 - G::kS);
      ring_fence();
    }
    bf16x8_t p[2];
    const float alpha = tile_softmax<CAP, SLOPES>(a, s, row, slope2, whole, key0, h, soft, p);
    if (__ballot(alpha != 1.f) != 0ull) {
#pragma unroll
      for (int dt = 0; dt < G::kT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[dt][i] *= alpha;
    }
    const bool bad = !whole && tile_not_finite<HD>(vt, vat);  // uniform over the wave
    if (bad) {
      add_not_finite<HD>(o, vt, vat, row, key0, h);
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = vfrag(i);  // again: not held over the rare path
    }
#pragma unroll
    for (int i = 0; i < G::kS; ++i) {
      if (bad) f[i & 3] = finite_only(f[i & 3]);
      o[i % G::kT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(f[i & 3]), p[i / G::kT], o[i % G::kT], 0, 0, 0);
      if (i + 4 < G::kS) f[i & 3] = vfrag(i + 4);
      ring_fence();
    }
  }
  const float l = row_sum(soft.m, soft.l + __shfl_xor(soft.l, 32, kWave),
                          row_sees(row, tile0 * kTileKeys, (tile0 + tiles) * kTileKeys));
  // o[dt][4 i + e] is channel 32 dt + 8 i + 4 h + e of the row
  if (a.n_split == 1) {
    // Through LDS, half of the channels at a time, into whole rows: a lane holds 8 bytes here and there
    // of its row. A wave's 32 rows are its own; 16-byte pieces (4 floats) at [row][piece ^ row].
    constexpr int kRow = HD * 2, kPieces = HD / 8, kFlip = kPieces - 1;  // bytes and pieces of half a row
    const float inv = row_inverse(l);
    uint8_t* const mine = smem + wave * (32 * kRow);
    __syncthreads();  // the last tile's reads are done
#pragma unroll
    for (int part = 0; part < 2; ++part) {
#pragma unroll
      for (int dt = 0; dt < G::kT / 2; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int piece = 8 * dt + 2 * i + h;
          const f32x16_t& x = o[part * (G::kT / 2) + dt];
          *reinterpret_cast<f32x4_t*>(mine + c * kRow + ((piece ^ c) & kFlip) * 16) =
              f32x4_t{x[4 * i] * inv, x[4 * i + 1] * inv, x[4 * i + 2] * inv, x[4 * i + 3] * inv};
        }
      __syncthreads();
#pragma unroll 2
      for (int i = lane; i < 32 * kPieces / 2; i += kWave) {
        const int rl = i / (kPieces / 2), pc = i % (kPieces / 2), ro = kRows * rg + 32 * wave + rl;
        if (ro >= R) continue;
        float y[8];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const f32x4_t w = *reinterpret_cast<const f32x4_t*>(mine + rl * kRow + (((2 * pc + e) ^ rl) & kFlip) * 16);
#pragma unroll
          for (int g = 0; g < 4; ++g) y[4 * e + g] = w[g];
        }
        store_out8(a, b, kh * group + ro % group, ro / group, part * (HD / 2) + 8 * pc, y);
      }
      __syncthreads();
    }
  } else {
    if (kRows * rg + 32 * wave + c >= R) return;
    const int64_t pr = (((int64_t)bkh * a.row_groups + rg) * a.n_split + sp) * kRows + 32 * wave + c;
    float* const po = a.part_o + pr * HD;
    if (tiles > 0) {
#pragma unroll
      for (int dt = 0; dt < G::kT; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<f32x4_t*>(po + 32 * dt + 8 * i + 4 * h) =
              f32x4_t{o[dt][4 * i], o[dt][4 * i + 1], o[dt][4 * i + 2], o[dt][4 * i + 3]};
    }
    if (h == 0) {
      a.part_ml[pr * 2] = soft.m;
      a.part_ml[pr * 2 + 1] = l;
    }
  }
}

// ---------------------------------------------------------------- few rows
//
// Up to 32 rows of a (lane, kv head) to a workgroup; its four waves take every fourth tile each, over
// all of the rows, and stage it for themselves alone: no barrier until their results are merged. K's
// place is loaded again as soon as the first product has read it, V's after the second.
template <int HD, bool CAP, bool SLOPES>
__global__ __launch_bounds__(256, 1) void k_masked_few(MaskedArgs a) {
  using G = TileGeom<HD>;
  __shared__ __attribute__((aligned(16))) uint8_t smem[4][2 * G::kTile];  // a wave's K and V tile
  __shared__ float ml[4][32][2];
  __shared__ bool sees[32];
  const int group = a.heads / a.kvh, R = group * a.t;
  const int bkh = blockIdx.x, kh = bkh % a.kvh, b = bkh / a.kvh, sp = blockIdx.y;
  const int tid = threadIdx.x, wave = uniform(tid / kWave), lane = tid & (kWave - 1);
  const int h = lane >> 5, c = lane & 31;
  const int r = min(c, R - 1);  // rows past R repeat the last one
  const int step = r / group, hq = kh * group + r % group;
  const RowKeys row = masked_row(a, b, step);
  const RowSet set = row_set(row);
  const int lo = set.lo_min, hi = set.hi_max;
  const float slope2 = SLOPES ? a.slopes[hq] * kLog2e : 0.f;
  bf16x8_t q[G::kS];
  {
    const uint16_t* const qrow = a.q + a.qr.at(b, hq, step) + 8 * h;
    u32x4_t d[G::kS];
#pragma unroll
    for (int s = 0; s < G::kS; ++s) d[s] = ld16(qrow + 16 * s);
#pragma unroll
    for (int s = 0; s < G::kS; ++s) {
      asm volatile("" : "+v"(d[s]));  // landed before the loop: its waits count the tiles' loads alone
      q[s] = as_bf16x8(d[s]);
    }
  }
  int tile0, tiles;
  masked_split(lo, hi, a.n_split, sp, tile0, tiles);
  tile0 = uniform(tile0);
  tiles = uniform(tiles);
  const int32_t* const trow = a.table + (int64_t)b * a.table_stride;
  const int last_block = (int)min(a.table_stride, (int64_t)INT32_MAX) - 1;
  uint8_t* const kt = smem[wave];
  uint8_t* const vt = kt + G::kTile;
  uint32_t koff[2][G::kLoads];
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int j = 0; j < G::kLoads; ++j) koff[x][j] = k_offset<HD>(lane, a.kvh, kh, x, j);
  const uint32_t voff = v_offset<HD>(lane, kh);
  auto block = [&](int key0, int x) { return sload(trow, min(key0 / kAttnBlock + x, last_block)); };
  auto wanted = [&](int key0, int x) { return key0 + kAttnBlock * x < hi && key0 + kAttnBlock * (x + 1) > lo; };
  auto stage_k = [&](int key0, int b0, int b1) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const BlockSource<HD> src(a, uniform(x ? b1 : b0), wanted(key0, x));
#pragma unroll
      for (int j = 0; j < G::kLoads; ++j) load_lds(src.k, kt + x * G::kHalf + j * 1024, koff[x][j]);
    }
  };
  auto stage_v = [&](int key0, int b0, int b1) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const BlockSource<HD> src(a, uniform(x ? b1 : b0), wanted(key0, x));
#pragma unroll
      for (int j = 0; j < G::kLoads; ++j) load_lds(src.v, vt + x * G::kHalf + j * 1024, voff + 1024u * j);
    }
  };

  RowSoft soft{-INFINITY, 0.f};
  f32x16_t o[G::kT];
#pragma unroll
  for (int dt = 0; dt < G::kT; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;
  const uint32_t kat = (uint32_t)(prompt_swap(c) * HD * 2 + ((h ^ prompt_flip(c)) * 16));
  const uint32_t vat = (uint32_t)(c * 32 + (h ^ (c >> 2 & 1)) * 16);
  constexpr int kStep = 4 * kTileKeys;
  const int end = (tile0 + tiles) * kTileKeys;
  int key0 = (tile0 + wave) * kTileKeys;
  int b0 = 0, b1 = 0;
  if (key0 < end) {
    b0 = block(key0, 0);
    b1 = block(key0, 1);
    stage_k(key0, b0, b1);
    stage_v(key0, b0, b1);
    b0 = block(key0 + kStep, 0);
    b1 = block(key0 + kStep, 1);
  }
  for (; key0 < end; key0 += kStep) {
    const bool more = key0 + kStep < end;
    ring_fence();
    vmcnt_wait<2 * G::kLoads>();  // K has landed, V may be on its way
    ring_fence();
    f32x16_t s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.f;
    u32x4_t f[4];
    auto kfrag = [&](int i) { return lds16(kt + (kat ^ (32u * (i & 3))) + 128 * (i >> 2)); };
    auto vfrag = [&](int i) { return lds16(vt + vat + (i % G::kT) * 1024 + (i / G::kT) * G::kHalf); };
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = kfrag(i);
    ring_fence();
#pragma unroll
    for (int i = 0; i < G::kS; ++i) {
      s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(f[i & 3]), q[i], s, 0, 0, 0);
      if (i + 4 < G::kS) f[i & 3] = kfrag(i + 4);
      ring_fence();
    }
    if (more) stage_k(key0 + kStep, b0, b1);  // every read of K went into a product above
    ring_fence();
    const bool whole = set.whole(key0);
    bf16x8_t p[2];
    const float alpha = tile_softmax<CAP, SLOPES>(a, s, row, slope2, whole, key0, h, soft, p);
    if (__ballot(alpha != 1.f) != 0ull) {
#pragma unroll
      for (int dt = 0; dt < G::kT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[dt][i] *= alpha;
    }
    ring_fence();
    if (more)
      vmcnt_wait<2 * G::kLoads>();  // V has landed, the next K may be on its way
    else
      vmcnt_wait<0>();
    ring_fence();
    const bool bad = !whole && tile_not_finite<HD>(vt, vat);  // uniform over the wave
    if (bad) add_not_finite<HD>(o, vt, vat, row, key0, h);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = vfrag(i);
    ring_fence();
#pragma unroll
    for (int i = 0; i < G::kS; ++i) {
      if (bad) f[i & 3] = finite_only(f[i & 3]);
      o[i % G::kT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(f[i & 3]), p[i / G::kT], o[i % G::kT], 0, 0, 0);
      if (i + 4 < G::kS) f[i & 3] = vfrag(i + 4);
      ring_fence();
    }
    if (more) {
      __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): every read of V is done
      ring_fence();
      stage_v(key0 + kStep, b0, b1);
      b0 = block(key0 + 2 * kStep, 0);
      b1 = block(key0 + 2 * kStep, 1);
    }
  }
  // The four waves' results through their own tiles' LDS: 32 rows of HD floats.
  const float l = soft.l + __shfl_xor(soft.l, 32, kWave);
  constexpr int kRow = HD * 4, kFlip = HD / 4 - 1;
#pragma unroll
  for (int dt = 0; dt < G::kT; ++dt)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int piece = 8 * dt + 2 * i + h;
      *reinterpret_cast<f32x4_t*>(kt + c * kRow + ((piece ^ c) & kFlip) * 16) =
          f32x4_t{o[dt][4 * i], o[dt][4 * i + 1], o[dt][4 * i + 2], o[dt][4 * i + 3]};
    }
  if (h == 0) {
    ml[wave][c][0] = soft.m;
    ml[wave][c][1] = l;
    if (wave == 0) sees[c] = row_sees(row, tile0 * kTileKeys, end);
  }
  __syncthreads();
  for (int i = tid; i < 32 * G::kP; i += 256) {
    const int rl = i / G::kP, pc = i % G::kP;
    if (rl >= R) break;
    float m = -INFINITY, sum = 0.f, y[8];
#pragma unroll
    for (int w = 0; w < 4; ++w) m = fmaxf(m, ml[w][rl][0]);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float mw = ml[w][rl][0], lw = ml[w][rl][1];
      const float wt = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - m);
      sum += lw * (mw == -INFINITY ? 1.f : wt);  // a sum without a maximum is 0 or NaN
      if (mw == -INFINITY) continue;             // such a wave holds nothing
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const f32x4_t x = *reinterpret_cast<const f32x4_t*>(smem[w] + rl * kRow + (((2 * pc + e) ^ rl) & kFlip) * 16);
#pragma unroll
        for (int g = 0; g < 4; ++g) y[4 * e + g] = fmaf(x[g], wt, y[4 * e + g]);
      }
    }
    sum = row_sum(m, sum, sees[rl]);
    if (a.n_split == 1) {
      const float inv = row_inverse(sum);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] *= inv;
      store_out8(a, b, kh * group + rl % group, rl / group, 8 * pc, y);
    } else {
      const int64_t pr = ((int64_t)bkh * a.n_split + sp) * 32 + rl;
      float* const po = a.part_o + pr * HD + 8 * pc;
      *reinterpret_cast<f32x4_t*>(po) = f32x4_t{y[0], y[1], y[2], y[3]};
      *reinterpret_cast<f32x4_t*>(po + 4) = f32x4_t{y[4], y[5], y[6], y[7]};
      if (pc == 0) {
        a.part_ml[pr * 2] = m;
        a.part_ml[pr * 2 + 1] = sum;
      }
    }
  }
}

// Merge of the key splits: out = sum_s o_s 2^(m_s - M) / sum_s l_s 2^(m_s - M), M = max_s m_s. W waves a
// row: each weighs all splits at once (lane s split s), then takes every W-th split, four of them in
// flight; the waves' sums are added in order.
template <int HD, int W>
__global__ __launch_bounds__(256) void k_masked_merge(MaskedArgs a, int rows, int group_rows) {
  constexpr int NV = HD / kWave;
  typedef float vec_t __attribute__((ext_vector_type(NV)));
  __shared__ vec_t red[W][kWave];
  const int group = a.heads / a.kvh;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = W == 1 ? 0 : uniform(tid / kWave);
  const int id = W == 1 ? uniform((int)blockIdx.x * 4 + tid / kWave) : (int)blockIdx.x;
  if (id >= rows) return;  // uniform over the wave (W == 1: no barrier below)
  const int hq = id % a.heads, bs = id / a.heads, st = bs % a.t, b = bs / a.t, kh = hq / group;
  const int r = st * group + hq % group, rg = r / group_rows, rl = r % group_rows;
  const int64_t base = (((int64_t)(b * a.kvh + kh) * a.row_groups + rg) * a.n_split) * group_rows + rl;
  const bool live = lane < a.n_split;
  const float m = live ? a.part_ml[(base + (int64_t)lane * group_rows) * 2] : -INFINITY;
  const float l = live ? a.part_ml[(base + (int64_t)lane * group_rows) * 2 + 1] : 0.f;
  const float mx = wave_max(m);
  const float w = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mx);
  const float inv = row_inverse(wave_sum(m == -INFINITY ? l : l * w));
  const uint64_t held = __ballot(m != -INFINITY);  // the other splits hold nothing: their rows are not written
  vec_t acc = {};
  for (int s0 = wave; s0 < a.n_split; s0 += 4 * W) {
    vec_t v[4];
    float ws[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int s = s0 + W * i;
      ws[i] = __shfl(w, s & (kWave - 1), kWave);
      v[i] = vec_t{};
      if (s < a.n_split && (held >> s & 1ull)) v[i] = *reinterpret_cast<const vec_t*>(a.part_o + (base + (int64_t)s * group_rows) * HD + NV * lane);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) acc += v[i] * ws[i];
  }
  if (W > 1) {
    red[wave][lane] = acc;
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int i = 1; i < W; ++i) acc += red[i][lane];
  }
  uint16_t* const orow = a.out + a.orow.at(b, hq, st) + NV * lane;
  const uint16_t* const grow = a.gate ? a.gate + a.gr.at(b, hq, st) + NV * lane : nullptr;
#pragma unroll
  for (int e = 0; e < NV; ++e) {
    const float y = acc[e] * inv;
    orow[e] = f32_to_bf16(grow ? y * sigmoid_of(grow[e]) : y);
  }
}

namespace {

// Rows of a workgroup: one wave's, two's or four's.
int64_t masked_group_rows(int64_t rows) { return rows <= 32 ? 32 : rows <= 64 ? 64 : 128; }
int64_t masked_row_groups(int64_t rows) { return (rows + masked_group_rows(rows) - 1) / masked_group_rows(rows); }

// Key splits: as many as bring the workgroups near the device's compute units, of at least 8 tiles each.
int masked_splits(int64_t batch, int64_t kvh, int64_t rows, int64_t hd, int64_t keys) {
  const int64_t wgs = std::max<int64_t>(batch * kvh * masked_row_groups(rows), 1);
  const int64_t per_cu = hd == 256 && rows <= 32 ? 1 : 2;
  const int64_t tiles = (keys + kTileKeys - 1) / kTileKeys;
  int64_t n = std::min<int64_t>(device_cu_count() * per_cu / wgs, tiles / 8);
  n = std::min<int64_t>(n, kMaskedSplits);
  return n < 1 ? 1 : (int)n;
}

template <int HD, bool CAP, bool SLOPES>
int masked_launch(const MaskedArgs& a, int64_t batch, hipStream_t st) {
  const int64_t rows = (int64_t)(a.heads / a.kvh) * a.t;
  const dim3 grid((unsigned)(batch * a.kvh * a.row_groups), (unsigned)a.n_split);
  if (rows <= 32)
    hipLaunchKernelGGL((k_masked_few<HD, CAP, SLOPES>), grid, dim3(256), 0, st, a);
  else if (rows <= 64)
    hipLaunchKernelGGL((k_masked_rows<HD, 2, CAP, SLOPES>), grid, dim3(128), 0, st, a);
  else
    hipLaunchKernelGGL((k_masked_rows<HD, 4, CAP, SLOPES>), grid, dim3(256), 0, st, a);
  int rc = status_of(hipGetLastError());
  if (rc || a.n_split == 1) return rc;
  const int out_rows = (int)(batch * a.heads * a.t), group_rows = (int)masked_group_rows(rows);
  if (a.n_split <= 8)
    hipLaunchKernelGGL((k_masked_merge<HD, 1>), dim3((unsigned)((out_rows + 3) / 4)), dim3(256), 0, st, a, out_rows, group_rows);
  else
    hipLaunchKernelGGL((k_masked_merge<HD, 4>), dim3((unsigned)out_rows), dim3(256), 0, st, a, out_rows, group_rows);
  return status_of(hipGetLastError());
}

template <int HD>
int masked_flags(const MaskedArgs& a, int64_t batch, hipStream_t st) {
  const bool cap = a.cap2 > 0.f;
  if (a.slopes) return cap ? masked_launch<HD, true, true>(a, batch, st) : masked_launch<HD, false, true>(a, batch, st);
  return cap ? masked_launch<HD, true, false>(a, batch, st) : masked_launch<HD, false, false>(a, batch, st);
}

bool masked_shape(int64_t batch, int64_t t, int64_t heads, int64_t kv_heads, int64_t head_dim) {
  return batch > 0 && t > 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0 &&
         (head_dim == 64 || head_dim == 128 || head_dim == 256) && batch <= INT32_MAX / 64 / t &&
         heads <= INT32_MAX / 64 / (batch * t);
}

}  // namespace
}  // namespace mtpk

using namespace mtpk;

extern "C" {

int mtpk_attention_masked_splits(int64_t batch, int64_t t, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                 int64_t max_ctx, int64_t window) {
  if (!masked_shape(batch, t, heads, kv_heads, head_dim) || max_ctx < 0 || window < 0) return 0;
  const int64_t rows = heads / kv_heads * t;
  int64_t keys = max_ctx;
  if (window > 0) keys = std::min(keys, window + masked_group_rows(rows) / (heads / kv_heads) + kTileKeys);
  return masked_splits(batch, kv_heads, rows, head_dim, keys);
}

int64_t mtpk_attention_masked_workspace_bytes(int64_t batch, int64_t t, int64_t heads, int64_t kv_heads,
                                              int64_t head_dim, int n_split) {
  if (!masked_shape(batch, t, heads, kv_heads, head_dim) || n_split <= 1) return 0;
  const int64_t rows = heads / kv_heads * t;
  return batch * kv_heads * masked_row_groups(rows) * masked_group_rows(rows) * n_split * (head_dim + 2) * 4;
}

int mtpk_paged_attention_masked(const uint16_t* q, const int64_t* q_strides, const uint16_t* gate,
                                const int64_t* gate_strides, int64_t batch, int64_t t, int64_t heads,
                                int64_t kv_heads, int64_t head_dim, const uint16_t* k_pool,
                                const uint16_t* v_pool, int64_t pool_rows, const int32_t* block_table,
                                int64_t table_stride, const int64_t* base_pos, float scale, float softcap,
                                int64_t window, const float* slopes, const void* prefix, int prefix_dtype,
                                const void* first, int first_dtype, int n_split, void* workspace,
                                int64_t workspace_bytes, uint16_t* out, const int64_t* out_strides,
                                void* stream) {
  if (!q || !k_pool || !v_pool || !block_table || !base_pos || !out || !q_strides || !out_strides) return MTPK_EINVAL;
  if (gate && !gate_strides) return MTPK_EINVAL;
  if (batch == 0 && t > 0) return 0;
  if (!masked_shape(batch, t, heads, kv_heads, head_dim)) return MTPK_EINVAL;
  if (pool_rows <= 0 || pool_rows % kAttnBlock || table_stride <= 0 || table_stride > (1 << 26) ||
      kv_heads > 4096) return MTPK_EINVAL;
  if (!(scale > 0.f) || !(softcap >= 0.f) || !(scale < INFINITY) || !(softcap < INFINITY)) return MTPK_EINVAL;
  if (window < 0 || n_split < 1 || n_split > kMaskedSplits) return MTPK_EINVAL;
  if (prefix && prefix_dtype != MTPK_I32 && prefix_dtype != MTPK_I64) return MTPK_EINVAL;
  if (first && first_dtype != MTPK_I32 && first_dtype != MTPK_I64) return MTPK_EINVAL;
  // 16-byte accesses to query, gate and output rows and to the pools
  if (!aligned16(q) || !aligned16(k_pool) || !aligned16(v_pool) || !aligned16(out) || (gate && !aligned16(gate)))
    return MTPK_EINVAL;
  for (int i = 0; i < 3; ++i)
    if (q_strides[i] % 8 || out_strides[i] % 8 || (gate && gate_strides[i] % 8)) return MTPK_EINVAL;
  if (n_split > 1 && (!workspace || !aligned16(workspace) ||
                      workspace_bytes < mtpk_attention_masked_workspace_bytes(batch, t, heads, kv_heads, head_dim, n_split)))
    return MTPK_EINVAL;
  const int64_t rows = heads / kv_heads * t;
  MaskedArgs a{};
  a.q = q;
  a.qr = {q_strides[0], q_strides[1], q_strides[2]};
  a.out = out;
  a.orow = {out_strides[0], out_strides[1], out_strides[2]};
  a.gate = gate;
  if (gate) a.gr = {gate_strides[0], gate_strides[1], gate_strides[2]};
  a.k_pool = k_pool;
  a.v_pool = v_pool;
  a.pool_rows = pool_rows;
  a.table = block_table;
  a.table_stride = table_stride;
  a.base = base_pos;
  a.slopes = slopes;
  a.prefix = prefix;
  a.prefix_dt = prefix_dtype;
  a.first = first;
  a.first_dt = first_dtype;
  a.window = (int)std::min<int64_t>(window, INT32_MAX);
  a.t = (int)t;
  a.heads = (int)heads;
  a.kvh = (int)kv_heads;
  a.lanes_kvh = (int)(batch * kv_heads);
  a.n_split = n_split;
  a.row_groups = (int)masked_row_groups(rows);
  a.scale2 = scale * kLog2e;
  if (softcap > 0.f) {
    // cap * tanh(u) log2(e), u = s * scale / cap: u - u^3 / 3 + 2 u^5 / 15 - 17 u^7 / 315 is within 3e-7 of
    // tanh(u), relative, up to |u| = 0.23
    const double k = (double)scale / softcap, c = (double)softcap * 1.4426950408889634;
    a.cap2 = (float)c;
    a.cap_in = (float)(2. * 1.4426950408889634 * k);
    a.poly_max = (float)(0.23 / k);
    a.c0 = (float)(c * k);
    a.c1 = (float)(-c * k * k * k / 3.);
    a.c2 = (float)(c * k * k * k * k * k * 2. / 15.);
    a.c3 = (float)(-c * k * k * k * k * k * k * k * 17. / 315.);
  }
  a.part_o = (float*)workspace;
  a.part_ml = a.part_o ? a.part_o + batch * kv_heads * a.row_groups * masked_group_rows(rows) * n_split * head_dim : nullptr;
  const hipStream_t st = (hipStream_t)stream;
  switch (head_dim) {
    case 64: return masked_flags<64>(a, batch, st);
    case 128: return masked_flags<128>(a, batch, st);
    default: return masked_flags<256>(a, batch, st);
  }
}

}  // extern "C"
