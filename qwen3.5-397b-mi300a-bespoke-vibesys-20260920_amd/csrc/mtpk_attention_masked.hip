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
// rounded once: 1.9e-3 to 2.4e-3 of the 2-norm from 64 bits, where the output's rounding alone makes 1.7e-3. P in two
// bf16 parts, a second product for the rest, comes down to that; it took 5 % more for a short context of one lane, 1 %
// for 48 lanes in a window, 2 to 8 % for verify rows, and prompts, half products as they are, would pay most.
//
// Keys that a row does not see may hold anything: their scores are replaced, and V is zeroed where no row of
// the workgroup sees the key. Nor do finite ones that no row sees choose the form in which a tile's scores are capped;
// the rows of a tile share it (each score's form by that score alone took two forms and a selection for every one of
// a tile past the cubic: 8000 rows of 16 heads of 128, scores of std 4 under a cap of 30, 390 -> 597 us). A value that
// is not finite and that some of the rows sharing a tile see makes all of them NaN (0 times infinity): such rows are
// found at the end and done again one by one.

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "mtpk_attention_common.h"
#include "mtpk_host.h"
#include "mtpk_tree.h"

namespace mtpk {

constexpr int kTileKeys = 32;
constexpr int kMaskedSplits = 64;       // key splits the merge takes
constexpr int kMergeOne = 8;            // up to these, with a wave a row; beyond, a workgroup
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
  uint32_t pool_blocks;  // at most 2^31: a table's entries are int32
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
  float cap2;                   // cap * log2(e), 0: none
  float cap_in;                 // 2 * log2(e) * scale / cap
  // cap2 * tanh(s scale / cap) as s (c0 + c1 s^2) up to |s| = cubic_max (s c0 without a cap), and as
  // s (e0 + e1 u + e2 u^2), u = (s cap_k)^2, up to |s cap_k| = 0.25
  float cubic_max, c0, c1, cap_k, e0, e1, e2;
  float* part_o;
  float* part_ml;
  TreeParents tree;  // the TREE form alone
};

// The keys [lo, hi) that a row sees, and its position (for distances); in a tree of the keys from `pos` on, the lane's
// first node, only those whose bits are set.
struct RowKeys {
  int pos, lo, hi;
  uint64_t nodes;
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
  const int64_t end = a.table_stride * kAttnBlock;
  hi = max(min(min(hi, base + a.t), end), (int64_t)0);
  lo = min(lo, (int64_t)INT32_MAX);
  // A row past the table is as if at its end: one distance more or less for all of its keys is no change, and
  // int and float hold the others' differences.
  return RowKeys{(int)min(pos, end), (int)lo, (int)hi, 0ull};
}

// A tree's row: the lane's whole context, then nodes by their bits. (An absent node's row, without bits, goes along as if it
// saw the context, and is done again in the end, which makes it zeros.)
__device__ inline RowKeys tree_row(const MaskedArgs& a, int b) {
  const int64_t base = a.base[b], end = a.table_stride * kAttnBlock;
  return RowKeys{(int)min(max(base, (int64_t)0), end), 0, (int)max(min(base + a.t, end), (int64_t)0), 0ull};
}

// Bit i: whether the row sees key key0 + i, for keys below `end`.
__device__ inline uint32_t tree_seen(const RowKeys& row, int key0) {
  const int at = key0 - row.pos, left = row.hi - key0;
  uint64_t w = at >= kTreeNodes ? 0ull : at >= 0 ? row.nodes >> at : at <= -32 ? ~0ull : row.nodes << -at | ((1ull << -at) - 1ull);
  return left >= 32 ? (uint32_t)w : left <= 0 ? 0u : (uint32_t)w & ((1u << left) - 1u);
}

// Over the 16 lanes of a row by DPP, then the two rows of a half.
__device__ inline int wave_min_i(int v) {
  v = min(v, __builtin_amdgcn_mov_dpp(v, 0xB1, 0xf, 0xf, false));
  v = min(v, __builtin_amdgcn_mov_dpp(v, 0x4E, 0xf, 0xf, false));
  v = min(v, __builtin_amdgcn_mov_dpp(v, 0x141, 0xf, 0xf, false));
  v = min(v, __builtin_amdgcn_mov_dpp(v, 0x140, 0xf, 0xf, false));
  return min(uniform(v), __builtin_amdgcn_readlane(v, 16));
}
__device__ inline int wave_max_i(int v) { return -1 - wave_min_i(-1 - v); }

// What 32 rows (the two halves of a wave hold them twice) see together.
struct RowSet {
  int lo_min, lo_max, hi_min, hi_max;
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
// for every block. K as [key][piece ^ k_flip(row of the key)], V as [channel][piece ^ v_swap(channel)].
template <int HD>
struct TileGeom {
  static constexpr int kS = HD / 16, kT = HD / 32, kP = HD / 8;  // k steps, channel tiles, 16-byte pieces of a key
  static constexpr int kHalf = kAttnBlock * HD * 2;              // bytes of a block's K (or V) of one kv head
  static constexpr int kTile = 2 * kHalf;                        // of a tile's V
  static constexpr int kKTile = kTile + (HD == 256 ? 1024 : 0);   // of a tile's K, with its rows' shifts
  static constexpr int kLoads = kHalf / 1024;  // 1 KB loads of a block
};

template <int HD>
struct BlockSource {
  rsrc_t k, v;
  __device__ inline BlockSource(const MaskedArgs& a, int blk, bool wanted) {
    const int64_t slab = (int64_t)kAttnBlock * a.kvh * HD;
    const bool ok = wanted && (uint32_t)blk < a.pool_blocks;
    const int64_t at = (int64_t)uniform(ok ? blk : 0) * slab;
    const uint32_t bytes = (uint32_t)uniform(ok ? (int)(slab * 2) : 0);  // a block outside the pool reads as zeros
    k = make_rsrc(a.k_pool + at, bytes);
    v = make_rsrc(a.v_pool + at, bytes);
  }
};

// The places of a tile's 16-byte pieces in LDS. One cycle of a read serves 16 lanes with 256 bytes: lanes 0-3, 8-11,
// 20-23 and 28-31, then 4-7, 12-15, 16-19 and 24-27, and so on in the upper half (the counted bank conflicts are those
// that this makes). So what a lane's c is to choose among 16 places is bits 0 to 3 of c. K's row for c
// (prompt_swap(c)) has its pieces flipped by three of them. Heads of 64, two rows to 256 bytes, have bit 0 in the row
// itself; heads of 256 have their rows shifted by 128 bytes for every 4, which is bit 3 (4095 packed rows: 94.0
// without, 93.2 us with it); heads of 128 are left with K's conflicts of two, as the same shift, though it ends
// them, made 8000 rows slower (318 to 322 us). V's channel d holds two pieces of a block, exchanged by bits 2 and 3 of d.
template <int HD>
__device__ inline int k_flip(int c) {
  return HD == 64 ? c >> 1 & 7 : ((c & 3) << 1) | (c >> 2 & 1);
}
template <int HD>
__device__ inline constexpr int k_row(int r) {
  return r * HD * 2 + (HD == 256 ? (r >> 2) * 128 : 0);
}
__device__ inline int v_swap(int d) { return ((d >> 2) ^ (d >> 3)) & 1; }

// Byte offset of K load j (of kLoads) of a block: 1 KB covers 64 / kP keys.
template <int HD>
__device__ inline uint32_t k_offset(int lane, int kvh, int kh, int half, int j) {
  using G = TileGeom<HD>;
  const int key = j * (64 / G::kP) + lane / G::kP;
  return (uint32_t)(((key * kvh + kh) * HD + ((lane % G::kP) ^ k_flip<HD>(prompt_swap(16 * half + key))) * 8) * 2);
}
// V load 0; load j is 1 KB further on.
template <int HD>
__device__ inline uint32_t v_offset(int lane, int kh) {
  return (uint32_t)(kh * HD * 32 + (lane >> 1) * 32 + (((lane & 1) ^ v_swap(lane >> 1)) * 16));
}

// V of `blocks` blocks in LDS, the first one's keys from key0 on: zeros at the keys outside [lo, hi). A wave takes 8 keys
// of 64 channels at a time, so that what of them is seen is one scalar mask.
template <int HD>
__device__ inline void zero_unseen(uint8_t* v, int blocks, int key0, int lo, int hi, int tid, int threads) {
  for (int i = tid; i < blocks * HD * 2; i += threads) {
    const int x = uniform(i / HD), d = i % HD, from = lo - key0 - 8 * x, to = hi - key0 - 8 * x;
    if (from <= 0 && to >= 8) continue;
    uint8_t* const at = v + (x >> 1) * (HD * 32) + d * 32 + ((x & 1) ^ v_swap(d)) * 16;
    u32x4_t w = lds16(at);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      w[e] &= (2 * e >= from && 2 * e < to ? 0x0000ffffu : 0u) | (2 * e + 1 >= from && 2 * e + 1 < to ? 0xffff0000u : 0u);
    lds16_store(at, w);
  }
}

// 1 KB from off + AT of each lane to `to` + AT (at most 4095).
template <int AT = 0>
__device__ inline void load_lds(rsrc_t r, uint8_t* to, uint32_t off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void_t*)to, 16, (int)off, 0, AT, 0);
}

// Scores are worked on in units of log2. What a row does not see becomes kUnseen, and a row's maximum starts
// at kNoKey, far above it and far below any score in use: neither needs a comparison later on, and
// both stay finite where the cap's line squares them. Capped scores up to 2^kCapMost need no maximum at all:
// their exponentials and sums stay inside fp32's and bf16's range as they are, and so the largest part of
// the work between the two products falls away. A row whose sum all the same comes out below least_sum (its
// keys all far below, or none: 0), or that holds a value that is not finite, is done again by masked_row_slow.
// In a tree the maximum that a row's weights are taken against moves only when a score passes it by more than kRise: the weights
// stay below 2^kRise, which fp32 sums and bf16 hold as well as those below 1, and the sums of a wave, which some of its 32
// rows would have multiplied again in nearly every tile, in few.
constexpr float kRise = 8.f;
constexpr float kUnseen = -1e18f, kNoKey = -1e17f, kCapMost = 100.f;

// The cap alone leaves every key at least 2^-100. A bias may take keys below 2^-126, where they are lost: up to 2^20
// of them are then less than 2^-26 of a sum that is at least 2^-80.
__device__ inline float least_sum(const MaskedArgs& a) { return a.slopes ? 0x1p-80f : 0x1p-102f; }

struct RowSoft {
  float m, l;
};

__device__ inline float cap_exact(const MaskedArgs& a, float s) {
  return fmaf(__builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s * a.cap_in) + 1.f), -2.f * a.cap2, a.cap2);
}

__device__ inline float cap_quintic(const MaskedArgs& a, float s, float u) { return s * fmaf(u, fmaf(u, a.e2, a.e1), a.e0); }

// The cap of a score, however wide: cap_exact is off by 2^-23 of the cap, which is more than a whole score where the
// cap is far above it, so it takes over only where scores are of the cap's own size.
__device__ inline float cap_any(const MaskedArgs& a, float s) {
  const float x = s * a.cap_k, u = x * x;
  return u <= 0.0625f ? cap_quintic(a, s, u) : cap_exact(a, s);
}

// The larger of a value and of the other half's (lane ^ 32).
__device__ inline float halves_max(float v) {
  const uint32_t u = f32_bits(v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(bits_f32(r[0]), bits_f32(r[1]));
}

// One tile of scores on its way to P, in steps that the caller puts between its products: scan (every value once),
// finish, and each value's exponent.
template <bool CAP, bool SLOPES, bool TREE = false>
struct TileSoftmax {
  float c0, c1, ms;  // exponent of a score s: s (c0 + c1 s^2) with a cap, s c0 - ms without one
  float top;         // the largest score, with a cap the largest magnitude
  float held;

  __device__ inline void begin() { top = CAP ? 0.f : -INFINITY; }
  __device__ inline void scan(float s) { top = fmaxf(top, CAP ? fabsf(s) : s); }

  // Scores to where `exponent` takes them from there, and without a cap the row's new maximum. Returns what the
  // row's sums are multiplied by, 1 for the whole wave in most tiles.
  // Inlined by force, as the steps around it in k_masked_rows are: a call would keep the wave's sums in memory.
  __device__ __forceinline__ float finish(const MaskedArgs& a, f32x16_t& s, const RowKeys& row, float slope2, bool whole, int key0,
                                 int h, RowSoft& r) {
    c0 = a.c0;
    c1 = a.c1;
    const int lo = row.lo - key0 - 8 * h, n = max(row.hi - row.lo, 0);  // seen: 0 <= i - lo < n, in one comparison
    const uint32_t bits = TREE && !whole ? tree_seen(row, key0 + 8 * h) : 0u;
    auto seen = [&](int i) {
      if constexpr (TREE)
        return (bits >> (16 * (i >> 3) + (i & 7)) & 1u) != 0u;
      else
        return (uint32_t)(16 * (i >> 3) + (i & 7) - lo) < (uint32_t)n;
    };
    auto past = [&]() { return __ballot(!(top <= a.cubic_max)) != 0ull; };
    bool bent = CAP ? past() : !TREE && a.cap2 > 0.f;  // past the cap's cubic part
    if (CAP && bent && !whole) {  // keys that no row sees have no part in the choice of the form
      begin();
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[i] = seen(i) ? s[i] : 0.f;
        scan(s[i]);
      }
      bent = past();
    }
    if (SLOPES || !whole || bent) {  // uniform over the wave: in full here, and the exponent is the score
      if (!bent) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = CAP ? s[i] * fmaf(s[i] * s[i], c1, c0) : s[i] * c0;
      } else if (CAP && __ballot(!(top * a.cap_k <= 0.25f)) == 0ull) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float x = s[i] * a.cap_k;
          s[i] = cap_quintic(a, s[i], x * x);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = CAP ? cap_exact(a, s[i]) : cap_any(a, s[i]);
      }
      if (SLOPES) {
        const float away = (float)(row.pos - key0 - 8 * h);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = fmaf(fabsf(away - (float)(16 * (i >> 3) + (i & 7))), -slope2, s[i]);
      }
      if (!whole) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = seen(i) ? s[i] : kUnseen;
      }
      c0 = 1.f;
      c1 = 0.f;
      if (!CAP) {
        begin();
#pragma unroll
        for (int i = 0; i < 16; ++i) scan(s[i]);
      }
    }
    if (CAP) return 1.f;
    if constexpr (TREE) {
      const float now = halves_max(top * c0);
      const bool up = now > r.m + kRise;
      ms = up ? now : r.m;
      if (__ballot(up) == 0ull) return 1.f;  // uniform
      const float alpha = __builtin_amdgcn_exp2f(r.m - ms);
      r.m = ms;
      r.l *= alpha;
      return alpha;
    }
    ms = fmaxf(r.m, halves_max(top * c0));
    const float alpha = __builtin_amdgcn_exp2f(r.m - ms);
    r.m = ms;
    r.l *= alpha;
    return alpha;
  }
  __device__ __forceinline__ float prepare(const MaskedArgs& a, f32x16_t& s, const RowKeys& row, float slope2, bool whole, int key0,
                                  int h, RowSoft& r) {
    begin();
#pragma unroll
    for (int i = 0; i < 16; ++i) scan(s[i]);
    return finish(a, s, row, slope2, whole, key0, h, r);
  }

  // Value I of a tile; the odd ones, after their even neighbour, store both.
  template <int I>
  __device__ inline void exponent(const f32x16_t& s, u32x4_t (&p)[2], RowSoft& r) {
    const float x = s[I], y = __builtin_amdgcn_exp2f(CAP ? x * fmaf(x * x, c1, c0) : fmaf(x, c0, -ms));
    if constexpr (I % 2 == 0) {
      held = y;
    } else {
      const bf16x2_t one = {(__bf16)1.f, (__bf16)1.f}, e = {(__bf16)held, (__bf16)y};
      uint32_t w = __builtin_bit_cast(uint32_t, e);
      asm volatile("" : "+v"(w));  // here, beside the products around it, and not where the second product is
      p[I >> 3][I >> 1 & 3] = w;
      // the sum of what the product uses
      r.l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w), one, r.l, false);
      asm volatile("" : "+v"(r.l));
    }
  }
};

// Steps of a loop as constants.
template <int N, typename F, int I = 0>
__device__ inline void static_for(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    static_for<N, F, I + 1>(static_cast<F&&>(f));
  }
}

// What a wave wrote to LDS, before its other lanes read it.
__device__ inline void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
  __builtin_amdgcn_wave_barrier();
}

// NaN where the sum has left fp32's range, as a bias that raises the weights makes it: the row is then done again.
__device__ inline float row_inverse(float l) { return l == 0.f ? 0.f : 1.f / l + (l - l); }

__device__ inline float sigmoid_of(uint16_t g) {
  // exp2 and reciprocal, 1 ulp each, of 2^-32 (1 + exp(-g)): the reciprocal of a value above 2^126 would be flushed
  return __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(fmaf(-kLog2e, bf16_to_f32(g), -32.f)) + 0x1p-32f) * 0x1p-32f;
}

// Eight values of an output row, gated, rounded once.
__device__ inline u32x4_t gate8(const MaskedArgs& a, int b, int hq, int st, int d) {
  return a.gate ? ld16(a.gate + a.gr.at(b, hq, st) + d) : zero16();
}
__device__ inline void store_out8(const MaskedArgs& a, int b, int hq, int st, int d, const float* v, u32x4_t g) {
  float y[8];
  uint16_t* const to = a.out + a.orow.at(b, hq, st) + d;
  if (a.gate) {
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

// One row by one wave, key by key in fp32 straight from memory: for the rows whose result above is not
// finite (a value or score that is not, seen by this row or by another one that shares its tiles), or
// whose keys all weigh too little. What the row does not see is not read.
template <int HD, bool TREE = false>
__device__ void masked_row_slow(const MaskedArgs& a, int b, int hq, int step, int lane) {
  constexpr int NV = HD / kWave;
  RowKeys row = TREE ? tree_row(a, b) : masked_row(a, b, step);
  if (TREE) {
    row.nodes = lane_bits(tree_ancestors(a.tree.at(b, lane, a.t), lane), step);
    if (row.nodes == 0ull) row.hi = row.lo;
  }
  const int kh = hq / (a.heads / a.kvh);
  const uint16_t* const q = a.q + a.qr.at(b, hq, step);
  const int32_t* const trow = a.table + (int64_t)b * a.table_stride;
  const float slope2 = a.slopes ? a.slopes[hq] * kLog2e : 0.f;
  float acc[NV], odd[NV], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < NV; ++e) acc[e] = odd[e] = 0.f;
#pragma unroll 1
  for (int key0 = row.lo; key0 < row.hi; key0 += kWave) {
    const int key = key0 + lane;
    bool live = key < row.hi;
    if (TREE && key >= row.pos) live = live && (row.nodes >> (key - row.pos & 63) & 1ull);
    const int id = live ? trow[key / kAttnBlock] : -1;
    const bool held = (uint32_t)id < a.pool_blocks;  // else the block reads as zeros
    float s = 0.f;
    if (held) {
      const uint16_t* const k = a.k_pool + (((int64_t)id * kAttnBlock + key % kAttnBlock) * a.kvh + kh) * HD;
#pragma unroll 1
      for (int d = 0; d < HD; d += 8) {
        float x[8], y[8];
        load8(q, MTPK_BF16, d, x);
        load8(k, MTPK_BF16, d, y);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(x[e], y[e], s);
      }
    }
    s = a.cap2 > 0.f ? cap_any(a, s) : s * a.c0;  // c0 without a cap: the scale
    s = live ? fmaf(fabsf((float)(row.pos - key)), -slope2, s) : -INFINITY;
    const float mn = fmaxf(m, wave_max(s)), ms = mn == -INFINITY ? 0.f : mn;
    const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn), p = live ? __builtin_amdgcn_exp2f(s - ms) : 0.f;
    m = mn;
    l = l * alpha + wave_sum(p);
#pragma unroll
    for (int e = 0; e < NV; ++e) acc[e] *= alpha;
#pragma unroll 1
    for (int j = 0; j < kWave && key0 + j < row.hi; ++j) {
      const float pj = __shfl(p, j, kWave);
      const int blk = __shfl(held ? id : -1, j, kWave);
      if (blk < 0) continue;  // uniform
      const uint16_t* const v = a.v_pool + (((int64_t)blk * a.kvh + kh) * HD + NV * lane) * kAttnBlock + (key0 + j) % kAttnBlock;
#pragma unroll
      for (int e = 0; e < NV; ++e) {
        const float x = bf16_to_f32(v[e * kAttnBlock]);
        if (fabsf(x) < INFINITY)
          acc[e] = fmaf(pj, x, acc[e]);
        else
          odd[e] += x;
      }
    }
  }
  const float inv = row.hi <= row.lo ? 0.f : 1.f / l;  // keys all at minus infinity: 0 / 0
  uint16_t* const to = a.out + a.orow.at(b, hq, step) + NV * lane;
  const uint16_t* const gate = a.gate ? a.gate + a.gr.at(b, hq, step) + NV * lane : nullptr;
#pragma unroll
  for (int e = 0; e < NV; ++e) {
    const float y = acc[e] * inv + odd[e];
    to[e] = f32_to_bf16(gate ? y * sigmoid_of(gate[e]) : y);
    if (TREE && row.hi <= row.lo) to[e] = 0;  // an absent node, whatever its gate holds
  }
}

// ---------------------------------------------------------------- many rows
//
// W waves of 32 rows to a workgroup, which share stages of ST tiles, one stage ahead in two buffers with
// one barrier per stage: prompts, and verify rows of more than one wave. With heads up to 128 a tile's first
// product runs one tile ahead of its second (AHEAD): between the products of S^T of tile t + 1 and the first half of
// O^T of tile t stand the exponents of tile t, spread evenly, between the others the scan of tile t + 1. Heads
// of 256, whose sums fill the registers, have half of a tile's exponents between its own O^T's products.
//
// 8000 rows of 16 heads of 128: 306-335 us by box, 0.93 PFLOP/s of visible products, at 1.9 GHz, 45 % of the cycles being
// products: 70 cycles a product, of which the same mix of instructions alone takes 50 at 1.77 GHz (the card's power), and
// the rest are stalls, bank conflicts in a third of the LDS cycles among them. 4095 rows of 32
// heads of 256 in documents of 700, gated: 84-90 us, 46 us of which the rows, gates and outputs take from memory at the copy
// rate; a workgroup spends 7 us on its rows, 19 on 12 tiles, 11 on gates and outputs, and the card holds just two
// rounds of them. Left out: two sets of 32 rows a wave, which read each operand once for both but leave one wave a
// SIMD (heads of 128: 317 -> 361 us); three waves a SIMD there (453 -> 477, an earlier form).
template <int HD, int W, bool CAP, bool SLOPES, bool TREE = false>
__global__ __launch_bounds__(W* kWave, 2) void k_masked_rows(MaskedArgs a) {
  using G = TileGeom<HD>;
  constexpr bool AHEAD = HD <= 128;
  constexpr int ST = AHEAD ? 2 : 1, kRows = 32 * W, kLead = AHEAD ? kTileKeys : 0;  // keys that K is staged ahead of V
  constexpr int RD = 4;  // products that an operand is read ahead
  constexpr int QL = AHEAD ? 0 : 3;  // pieces of Q that stay in LDS, where the registers hold no more
  constexpr int kStageKeys = ST * kTileKeys, kVAt = ST * G::kKTile;  // a buffer: K tiles, then V tiles
  constexpr int kBuffer = kVAt + ST * G::kTile;
  constexpr int kMine = 2 * ST * G::kLoads / W;                        // 1 KB loads of a stage and tensor that a wave makes
  constexpr int kBlocks = kMine >= G::kLoads ? kMine / G::kLoads : 1;  // blocks that it takes part in
  constexpr int kPer = kMine < G::kLoads ? kMine : G::kLoads;          // and of each its loads
  constexpr int kFirst = 2 * G::kLoads / W;                            // of the first tile of K
  static_assert(kFirst >= 1 && kFirst <= G::kLoads, "a wave loads from one block of the first tile");
  // Two objects, and two stages written out below: what the loads write is then known not to be what is read, and no
  // read waits for them.
  __shared__ __attribute__((aligned(16))) uint8_t buf0[kBuffer], buf1[kBuffer];
  __shared__ __attribute__((aligned(16))) uint8_t q_smem[QL ? W * QL * 1024 : 16];
  __shared__ int wg_lo[W], wg_hi[W];
  const int group = a.heads / a.kvh, R = group * a.t;
  const int rg = a.row_groups - 1 - (int)blockIdx.x / a.lanes_kvh;  // the last rows, which see most, first
  const int bkh = (int)blockIdx.x % a.lanes_kvh, kh = bkh % a.kvh, b = bkh / a.kvh, sp = blockIdx.y;
  const int tid = threadIdx.x, wave = uniform(tid / kWave), lane = tid & (kWave - 1);
  const int h = lane >> 5, c = lane & 31;
  const int row0 = kRows * rg + 32 * wave;  // this wave's first row
  const int r = min(row0 + c, R - 1);       // rows past R repeat the last one
  const int step = r / group, hq = kh * group + r % group;
  u32x4_t qd[G::kS];
  {
    const uint16_t* const qrow = a.q + a.qr.at(b, hq, step) + 8 * h;
#pragma unroll
    for (int s = 0; s < G::kS; ++s) qd[s] = ld16(qrow + 16 * s);
  }
  RowKeys row;
  RowSet set;
  int lo, hi;
  if constexpr (TREE) {  // the same keys for all rows
    row = tree_row(a, b);
    lo = 0;
    hi = uniform(row.hi);
    set = RowSet{0, 0, min(uniform(row.pos), hi), hi};
  } else {
    row = masked_row(a, b, step);
    set = row_set(row);
    if (lane == 0) {
      wg_lo[wave] = set.lo_min;
      wg_hi[wave] = set.hi_max;
    }
    __syncthreads();
    lo = wg_lo[0];
    hi = wg_hi[0];
#pragma unroll
    for (int w = 1; w < W; ++w) {
      lo = min(lo, wg_lo[w]);
      hi = max(hi, wg_hi[w]);
    }
    lo = uniform(lo);
    hi = uniform(hi);
  }
  int tile0, tiles;
  masked_split(lo, hi, a.n_split, sp, tile0, tiles);
  tile0 = uniform(tile0);
  tiles = uniform(tiles);
  const int end = (tile0 + tiles) * kTileKeys;
  // This split's keys alone: its last stage may reach into the next one's.
  row.hi = min(row.hi, end);
  set.hi_min = min(set.hi_min, end);
  hi = min(hi, end);

  const float slope2 = SLOPES ? a.slopes[hq] * kLog2e : 0.f;
  const int32_t* const trow = a.table + (int64_t)b * a.table_stride;
  const int last_block = (int)min(a.table_stride, (int64_t)INT32_MAX) - 1;

  // Stage s holds V of the tiles from ST s on and K of those kLead further on. This wave's loads of each are
  // [wave kMine, (wave + 1) kMine) of them, block by block.
  const int g0 = wave * kMine, block0 = g0 / G::kLoads, j0 = g0 % G::kLoads;
  const uint32_t kpiece = (uint32_t)(((lane / G::kP * a.kvh + kh) * HD + (lane % G::kP) * 8) * 2);
  const uint32_t kstep = (uint32_t)(64 / G::kP * a.kvh * HD * 2);  // bytes between loads of a block
  const uint32_t vpiece = v_offset<HD>(lane, kh);
  const int klane = lane / G::kP;
  auto wanted = [&](int at) { return at < hi && at + kAttnBlock > lo; };
  auto block = [&](int key) { return sload(trow, min(key / kAttnBlock, last_block)); };
  // Load J of a block of K, into its tile's place: two to a setting of the LDS address, the second one's offset in the
  // instruction, which counts for both sides. Its lanes' pieces ^ flip of the key's row: the flip of
  // 16 (block % 2) + key, of which the lane has its own share.
  auto load_k = [&](rsrc_t src, uint8_t* to, int half, int first, auto j) {
    const int at = 16 * half + (first + j / 2 * 2) * (64 / G::kP), key = at + j % 2 * (64 / G::kP) + klane;
    const uint32_t off = (kpiece ^ (uint32_t)(k_flip<HD>(prompt_swap(key)) * 16)) + (uint32_t)(first + j) * kstep;
    load_lds<j % 2 * 1024>(src, to + k_row<HD>(at), off - j % 2 * 1024u);
  };
  int kid[kBlocks], vid[kBlocks];
  auto blocks = [&](int key) {
#pragma unroll
    for (int x = 0; x < kBlocks; ++x) {
      vid[x] = block(key + kAttnBlock * (block0 + x));
      kid[x] = block(key + kLead + kAttnBlock * (block0 + x));
    }
  };
  // Load J of the 2 kMine of the stage at key: of each block K, then V. What lies past the keys is zeros, unread.
  rsrc_t from;
  auto load = [&](uint8_t* to, int key, auto j) {
    constexpr int x = j / (2 * kPer), i = j % (2 * kPer);
    const int at = key + kAttnBlock * (block0 + x);
    if constexpr (i == 0) from = BlockSource<HD>(a, uniform(kid[x]), wanted(at + kLead)).k;
    if constexpr (i == kPer) from = BlockSource<HD>(a, uniform(vid[x]), wanted(at)).v;
    if constexpr (i < kPer) {
      load_k(from, to + (block0 + x) / 2 * G::kKTile, (block0 + x) & 1, j0, std::integral_constant<int, i>{});
    } else {
      constexpr int n = (i - kPer) / 4 * 4, m = (i - kPer) % 4;
      load_lds<m * 1024>(from, to + kVAt + (block0 + x) * G::kHalf + (j0 + n) * 1024, vpiece + 1024u * (j0 + n));
    }
  };
  // The stage at `key` beside product `slot` of the first S of the one before: in one go its loads hold a wave up for
  // 760 cycles of a stage's 3600 (heads of 128).
  auto loads = [&](auto slot, auto slots, uint8_t* to, int key) {
    constexpr int first = (slot * 2 * kMine + slots - 1) / slots, last = ((slot + 1) * 2 * kMine + slots - 1) / slots;
    static_for<last - first>([&](auto j) { load(to, key, std::integral_constant<int, first + j>{}); });
  };

  RowSoft soft{CAP ? 0.f : kNoKey, 0.f};
  f32x16_t o[G::kT];
#pragma unroll
  for (int dt = 0; dt < G::kT; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;
  // this lane's K pieces: 2 s + h of tile row c, whose place is that of piece h with bits of s flipped
  const uint32_t kat = (uint32_t)(k_row<HD>(prompt_swap(c)) + ((h ^ k_flip<HD>(c)) * 16));
  // and its V^T keys: 8 h .. 8 h + 7 of each block, channel 32 dt + c
  const uint32_t vat = (uint32_t)(kVAt + c * 32 + (h ^ v_swap(c)) * 16);

  uint8_t* const q_mine = q_smem + (wave * QL * 64 + lane) * 16;
  int key0 = tile0 * kTileKeys;
  if (tiles > 0) {
    if constexpr (AHEAD) {  // the first tile of K, as the last one of a stage before the first
      const int g = wave * kFirst, x = g / G::kLoads;
      const BlockSource<HD> src(a, uniform(block(key0 + kAttnBlock * x)), wanted(key0 + kAttnBlock * x));
      static_for<kFirst>([&](auto j) { load_k(src.k, buf1 + (ST - 1) * G::kKTile, x, g % G::kLoads, j); });
    }
    blocks(key0);
    static_for<2 * kMine>([&](auto j) { load(buf0, key0, j); });
    blocks(key0 + kStageKeys);
  }
  if constexpr (TREE) {
    const uint64_t nodes = tree_ancestors(a.tree.at(b, lane, a.t), lane);
    row.nodes = (uint64_t)(uint32_t)__shfl((int)(nodes >> 32), step, kWave) << 32 | (uint32_t)__shfl((int)nodes, step, kWave);
  }
  bf16x8_t q[G::kS - QL];
#pragma unroll
  for (int s = 0; s < G::kS; ++s) {
    asm volatile("" : "+v"(qd[s]));  // landed before the loop: its waits count the tiles' loads alone
    if (s >= QL)
      q[s - QL] = as_bf16x8(qd[s]);
    else
      lds16_store(q_mine + s * 1024, qd[s]);
  }

  TileSoftmax<CAP, SLOPES, TREE> soft_tile;
  u32x4_t p[2], f[RD];
  const f32x16_t zero = {};
  auto kfrag = [&](const uint8_t* k, int i) { return lds16(k + (kat ^ (32u * (i & 3))) + 128 * (i >> 2)); };
  auto vfrag = [&](const uint8_t* v, int i) { return lds16(v + vat + (i % G::kT) * 1024 + (i / G::kT) * G::kHalf); };
  auto begin = [&](const uint8_t* k) {
#pragma unroll
    for (int i = 0; i < RD; ++i) f[i] = kfrag(k, i);
    ring_fence();
  };
  auto qpiece = [&](auto i) {
    if constexpr (i < QL)
      return as_bf16x8(lds16(q_mine + i * 1024));
    else
      return q[i - QL];
  };
  auto rescale = [&](float alpha) {
    if (!CAP && __ballot(alpha != 1.f) != 0ull) {
#pragma unroll
      for (int dt = 0; dt < G::kT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[dt][i] *= alpha;
    }
    ring_fence();
  };
  auto finish = [&](f32x16_t& s, int key) __attribute__((always_inline)) {
    return soft_tile.finish(a, s, row, slope2, set.whole(key), key, h, soft);
  };
  // Exponents [from, to) of a tile's 16.
  auto exponents = [&](auto from, auto to, const f32x16_t& s) {
    static_for<to - from>([&](auto j) { soft_tile.template exponent<from + j>(s, p, soft); });
  };
  // S^T of the tile at k into sn and O^T of the one at v with the scores sc. `next` (or null): where the K after that
  // is; `to` (or null): where the next stage goes.
  auto tile = [&](const uint8_t* k, const uint8_t* v, auto next, const f32x16_t& sc, f32x16_t& sn, auto to) __attribute__((always_inline)) {
    constexpr bool kNext = !std::is_same_v<decltype(next), std::nullptr_t>;
    constexpr bool kStage = !std::is_same_v<decltype(to), std::nullptr_t>;
    constexpr int kSlots = G::kS + G::kT;  // products beside which the exponents stand, two thirds before O^T begins
    auto beside = [&](auto slot) {
      if constexpr (kStage) loads(slot, std::integral_constant<int, 2 * G::kS>{}, to, key0 + kStageKeys);
      if constexpr (slot < kSlots)
        exponents(std::integral_constant<int, (slot * 16 + kSlots - 1) / kSlots>{},
                  std::integral_constant<int, ((slot + 1) * 16 + kSlots - 1) / kSlots>{}, sc);
    };
    static_for<G::kS>([&](auto i) {
      sn = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(f[i % RD]), qpiece(i), i == 0 ? zero : sn, 0, 0, 0);
      f[i % RD] = i + RD < G::kS ? kfrag(k, i + RD) : vfrag(v, i + RD - G::kS);
      beside(i);
      ring_fence();
    });
    soft_tile.begin();
    static_for<G::kS>([&](auto i) {
      if constexpr (i == G::kT) __builtin_amdgcn_s_setprio(1);  // few instructions beside these
      o[i % G::kT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(f[i % RD]), as_bf16x8(p[i / G::kT]), o[i % G::kT], 0, 0, 0);
      if constexpr (i + RD < G::kS)
        f[i % RD] = vfrag(v, i + RD);
      else if constexpr (kNext)
        f[i % RD] = kfrag(next, i + RD - G::kS);
      beside(std::integral_constant<int, G::kS + i>{});
      if constexpr (i >= G::kT) {
#pragma unroll
        for (int e = 0; e < 16 / G::kT; ++e) soft_tile.scan(sn[(i - G::kT) * (16 / G::kT) + e]);
        asm volatile("" : "+v"(soft_tile.top));  // here as well
      }
      ring_fence();
    });
    __builtin_amdgcn_s_setprio(0);
  };
  // The stage in `at`; the next one's loads go to `to`.
  f32x16_t s0, s1;
  auto stage = [&](uint8_t* at, uint8_t* to) __attribute__((always_inline)) {
    ring_fence();
    vmcnt_wait<0>();  // this stage, loaded during the last one, which has been the last to read `to`
    __builtin_amdgcn_s_barrier();
    ring_fence();
    if (key0 < lo || key0 + kStageKeys > hi) {  // uniform: V at keys that no row of the workgroup sees becomes zeros
      zero_unseen<HD>(at + kVAt, 2 * ST, key0, lo, hi, tid, W * kWave);
      __syncthreads();
    }
    begin(at);
    if constexpr (AHEAD) {
      tile(at, at, at + G::kKTile, s0, s1, to);
      blocks(key0 + 2 * kStageKeys);
      if (key0 + kTileKeys < end) {
        rescale(finish(s1, key0 + kTileKeys));
        tile(at + G::kKTile, at + G::kTile, nullptr, s1, s0, nullptr);
        if (key0 + kStageKeys < end) rescale(finish(s0, key0 + kStageKeys));
      }
    } else {  // four operands ahead where no exponents are in the registers yet, two across the softmax (90.0 -> 88.9 us)
      static_for<G::kS>([&](auto i) {
        s0 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(f[i % RD]), qpiece(i), i == 0 ? zero : s0, 0, 0, 0);
        if constexpr (i + RD < G::kS) f[i % RD] = kfrag(at, i + RD);
        loads(i, std::integral_constant<int, G::kS>{}, to, key0 + kStageKeys);
        ring_fence();
      });
      blocks(key0 + 2 * kStageKeys);
      const float alpha = soft_tile.prepare(a, s0, row, slope2, set.whole(key0), key0, h, soft);
      f[0] = vfrag(at, 0);
      f[1] = vfrag(at, 1);
      exponents(std::integral_constant<int, 0>{}, std::integral_constant<int, 8>{}, s0);
      rescale(alpha);
      __builtin_amdgcn_s_setprio(1);
      static_for<G::kS>([&](auto i) {
        o[i % G::kT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(f[i % RD]), as_bf16x8(p[i / G::kT]), o[i % G::kT], 0, 0, 0);
        if constexpr (i < 2) {
          f[(2 * i + 2) % RD] = vfrag(at, 2 * i + 2);
          f[(2 * i + 3) % RD] = vfrag(at, 2 * i + 3);
        } else if constexpr (i + RD < G::kS) {
          f[i % RD] = vfrag(at, i + RD);
        }
        if constexpr (i < 8) exponents(std::integral_constant<int, 8 + i>{}, std::integral_constant<int, 9 + i>{}, s0);
        ring_fence();
      });
      __builtin_amdgcn_s_setprio(0);
    }
    key0 += kStageKeys;
  };
  if constexpr (AHEAD) {
    if (tiles > 0) {
      vmcnt_wait<2 * kMine>();  // K of the first tile, the stage behind it may be on its way
      __builtin_amdgcn_s_barrier();
      ring_fence();
      const uint8_t* const k = buf1 + (ST - 1) * G::kKTile;
      begin(k);
      static_for<G::kS>([&](auto i) {
        s0 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(f[i % RD]), qpiece(i), i == 0 ? zero : s0, 0, 0, 0);
        if (i + RD < G::kS) f[i % RD] = kfrag(k, i + RD);
        ring_fence();
      });
      soft_tile.prepare(a, s0, row, slope2, set.whole(key0), key0, h, soft);  // no sums yet to multiply
      ring_fence();
    }
  }
  while (key0 < end) {
    stage(buf0, buf1);
    if (key0 >= end) break;
    stage(buf1, buf0);
  }
  float l = soft.l + __shfl_xor(soft.l, 32, kWave);
  if (TREE && row.nodes == 0ull) l = 0.f;
  const bool real = row0 + c < R;
  // o[dt][4 i + e] is channel 32 dt + 8 i + 4 h + e of the row
  if (a.n_split == 1) {
    // Through LDS, half of the channels at a time, into whole rows: a lane holds 8 bytes here and there
    // of its row. A wave's 32 rows are its own; 16-byte pieces (4 floats) at [row][piece ^ row].
    constexpr int kRow = HD * 2, kPieces = HD / 8, kFlip = kPieces - 1;  // bytes and pieces of half a row
    static_assert(W / 2 * 32 * kRow <= kBuffer, "half of the rows' floats fit the buffers");
    constexpr int kEach = 32 * kPieces / 2 / kWave;  // pieces of 8 channels that a lane stores of a half
    // the gates, all on their way before the first is used: one memory latency for the workgroup's last step
    u32x4_t gates[2 * kEach];
#pragma unroll
    for (int i = 0; i < 2 * kEach; ++i) {
      const int at = lane + kWave * (i % kEach), ro = min(row0 + at / (kPieces / 2), R - 1);
      gates[i] = gate8(a, b, kh * group + ro % group, ro / group, i / kEach * (HD / 2) + 8 * (at % (kPieces / 2)));
    }
    const float inv = row_inverse(l);
    float top = 0.f;  // the row's largest magnitude, NaN where a value is
    uint8_t* const mine = (wave & 1 ? buf1 : buf0) + wave / 2 * (32 * kRow);
    vmcnt_wait<0>();  // loads into the buffers, zeros behind the last stage, are over,
    __syncthreads();  // and the reads of it
#pragma unroll
    for (int part = 0; part < 2; ++part) {
#pragma unroll
      for (int dt = 0; dt < G::kT / 2; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int piece = 8 * dt + 2 * i + h;
          const f32x16_t& x = o[part * (G::kT / 2) + dt];
          const f32x4_t y = {x[4 * i] * inv, x[4 * i + 1] * inv, x[4 * i + 2] * inv, x[4 * i + 3] * inv};
#pragma unroll
          for (int e = 0; e < 4; ++e) top = __builtin_elementwise_maximum(top, fabsf(y[e]));
          *reinterpret_cast<f32x4_t*>(mine + c * kRow + ((piece ^ c) & kFlip) * 16) = y;
        }
      wave_lds_fence();
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int at = lane + kWave * i, rl = at / (kPieces / 2), pc = at % (kPieces / 2), ro = row0 + rl;
        if (ro >= R) continue;
        float y[8];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const f32x4_t w = *reinterpret_cast<const f32x4_t*>(mine + rl * kRow + (((2 * pc + e) ^ rl) & kFlip) * 16);
#pragma unroll
          for (int g = 0; g < 4; ++g) y[4 * e + g] = w[g];
        }
        store_out8(a, b, kh * group + ro % group, ro / group, part * (HD / 2) + 8 * pc, y, gates[part * kEach + i]);
      }
      wave_lds_fence();
    }
    uint64_t again = __ballot(real && (!(top < INFINITY) || (l < least_sum(a) && row.hi > row.lo)));
    again = (again | again >> 32) & 0xffffffffull;
    while (again != 0ull) {
      const int rl = uniform(__builtin_ctzll(again)), ro = row0 + rl;
      again &= again - 1ull;
      masked_row_slow<HD, TREE>(a, b, kh * group + ro % group, ro / group, lane);
    }
  } else {
    if (!real) return;
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
      a.part_ml[pr * 2] = tiles > 0 ? soft.m : -INFINITY;  // of a split without tiles nothing else is written
      a.part_ml[pr * 2 + 1] = l;
    }
  }
}

// ---------------------------------------------------------------- few rows
//
// Up to 32 rows of a (lane, kv head) to a workgroup; its W waves take every W-th tile each, over
// all of the rows, and stage it for themselves alone: no barrier until their results are merged. K's
// place is loaded again as soon as the first product has read it, V's after the second. 48 lanes of 2 kv heads of 256,
// windows of 4096: 81 us with the merge, 5.2 TB/s in this kernel; 65,000 and 31,000 keys of 4 kv heads of 128: 50 us.
template <int HD, int W, bool CAP, bool SLOPES, bool TREE = false>
__global__ __launch_bounds__(W* kWave, 1) void k_masked_few(MaskedArgs a) {
  using G = TileGeom<HD>;
  __shared__ __attribute__((aligned(16))) uint8_t smem[W][G::kKTile + G::kTile];  // a wave's K and V tile
  __shared__ float ml[W][32][2];
  __shared__ int again[32];
  const int group = a.heads / a.kvh, R = group * a.t;
  const int bkh = blockIdx.x, kh = bkh % a.kvh, b = bkh / a.kvh, sp = blockIdx.y;
  const int tid = threadIdx.x, wave = uniform(tid / kWave), lane = tid & (kWave - 1);
  const int h = lane >> 5, c = lane & 31;
  const int r = min(c, R - 1);  // rows past R repeat the last one
  const int step = r / group, hq = kh * group + r % group;
  u32x4_t qd[G::kS];
  {
    const uint16_t* const qrow = a.q + a.qr.at(b, hq, step) + 8 * h;
#pragma unroll
    for (int s = 0; s < G::kS; ++s) qd[s] = ld16(qrow + 16 * s);
  }
  RowKeys row = TREE ? tree_row(a, b) : masked_row(a, b, step);
  const RowSet set = TREE ? RowSet{0, 0, min(uniform(row.pos), uniform(row.hi)), uniform(row.hi)} : row_set(row);
  const int lo = set.lo_min, hi = set.hi_max;
  const float slope2 = SLOPES ? a.slopes[hq] * kLog2e : 0.f;
  int tile0, tiles;
  masked_split(lo, hi, a.n_split, sp, tile0, tiles);
  tile0 = uniform(tile0);
  tiles = uniform(tiles);
  const int32_t* const trow = a.table + (int64_t)b * a.table_stride;
  const int last_block = (int)min(a.table_stride, (int64_t)INT32_MAX) - 1;
  uint8_t* const kt = smem[wave];
  uint8_t* const vt = kt + G::kKTile;
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
      for (int j = 0; j < G::kLoads; ++j) load_lds(src.k, kt + k_row<HD>(16 * x + j * (64 / G::kP)), koff[x][j]);
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

  RowSoft soft{CAP ? 0.f : kNoKey, 0.f};
  f32x16_t o[G::kT];
#pragma unroll
  for (int dt = 0; dt < G::kT; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;
  const uint32_t kat = (uint32_t)(k_row<HD>(prompt_swap(c)) + ((h ^ k_flip<HD>(c)) * 16));
  const uint32_t vat = (uint32_t)(c * 32 + (h ^ v_swap(c)) * 16);
  constexpr int kStep = W * kTileKeys;
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
  if constexpr (TREE) {
    const uint64_t nodes = tree_ancestors(a.tree.at(b, lane, a.t), lane);
    row.nodes = (uint64_t)(uint32_t)__shfl((int)(nodes >> 32), step, kWave) << 32 | (uint32_t)__shfl((int)nodes, step, kWave);
  }
  bf16x8_t q[G::kS];
#pragma unroll
  for (int s = 0; s < G::kS; ++s) {
    asm volatile("" : "+v"(qd[s]));  // landed before the loop: its waits count the tiles' loads alone
    q[s] = as_bf16x8(qd[s]);
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
    TileSoftmax<CAP, SLOPES, TREE> soft_tile;
    u32x4_t p[2];
    const float alpha = soft_tile.prepare(a, s, row, slope2, set.whole(key0), key0, h, soft);
    static_for<16>([&](auto i) { soft_tile.template exponent<i>(s, p, soft); });
    if (!CAP && __ballot(alpha != 1.f) != 0ull) {
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
    if (key0 < lo || key0 + kTileKeys > hi) {  // uniform: V at keys that no row sees becomes zeros
      zero_unseen<HD>(vt, 2, key0, lo, hi, lane, kWave);
      wave_lds_fence();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = vfrag(i);
    ring_fence();
#pragma unroll
    for (int i = 0; i < G::kS; ++i) {
      o[i % G::kT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(f[i & 3]), as_bf16x8(p[i / G::kT]), o[i % G::kT], 0, 0, 0);
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
  // The waves' results through their own tiles' LDS: 32 rows of HD floats.
  float l = soft.l + __shfl_xor(soft.l, 32, kWave);
  if (TREE && row.nodes == 0ull) l = 0.f;
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
    if (wave == 0) again[c] = 0;
  }
  __syncthreads();
  for (int i = tid; i < 32 * G::kP; i += W * kWave) {
    const int rl = i / G::kP, pc = i % G::kP;
    if (rl >= R) break;
    const u32x4_t gate = a.n_split == 1 ? gate8(a, b, kh * group + rl % group, rl / group, 8 * pc) : zero16();
    float m = kNoKey, sum = 0.f, y[8];
#pragma unroll
    for (int w = 0; w < W; ++w) m = fmaxf(m, ml[w][rl][0]);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float wt = __builtin_amdgcn_exp2f(ml[w][rl][0] - m);
      sum = fmaf(ml[w][rl][1], wt, sum);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const f32x4_t x = *reinterpret_cast<const f32x4_t*>(smem[w] + rl * kRow + (((2 * pc + e) ^ rl) & kFlip) * 16);
#pragma unroll
        for (int g = 0; g < 4; ++g) y[4 * e + g] = fmaf(x[g], wt, y[4 * e + g]);
      }
    }
    if (a.n_split == 1) {
      const float inv = row_inverse(sum);
      float odd = sum < least_sum(a) ? 1.f : 0.f;  // not 0: the row is done again, below
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y[e] *= inv;
        odd = fmaf(y[e], 0.f, odd);
      }
      store_out8(a, b, kh * group + rl % group, rl / group, 8 * pc, y, gate);
      if (odd != 0.f) again[rl] = 1;
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
  if (a.n_split > 1) return;
  __syncthreads();
  for (int rl = wave; rl < min(R, 32); rl += W) {
    if (uniform(again[rl]) != 0) masked_row_slow<HD, TREE>(a, b, kh * group + rl % group, rl / group, lane);
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
  const float mx = fmaxf(wave_max(m), kNoKey);
  const float w = __builtin_amdgcn_exp2f(m - mx), sum = wave_sum(l * w), inv = row_inverse(sum);
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
  float odd = sum < least_sum(a) ? 1.f : 0.f;
#pragma unroll
  for (int e = 0; e < NV; ++e) {
    const float y = acc[e] * inv;
    odd = fmaf(y, 0.f, odd);
    orow[e] = f32_to_bf16(grow ? y * sigmoid_of(grow[e]) : y);
  }
  if (__ballot(odd != 0.f) != 0ull) masked_row_slow<HD>(a, b, hq, st, lane);
}

// The same of a tree's rows, workgroup (x, y) of node x of all lanes: everything that a row is made of is on its way at once,
// the splits' sums before their weights are known (a split without keys has none written, and its garbage is left out). Up
// to 8 splits with a wave a row, 4 heads to a workgroup, which weighs them without a word between lanes (24,576 rows of 2
// splits of 256: 14.8 us, with the form above 19.7); beyond, a workgroup a row (2016 of 32 splits of 128: 8.7, 10.0).
template <int HD, int W, int N>
__global__ __launch_bounds__(256, N* HD > 2048 ? 4 : 6) void k_tree_merge(MaskedArgs a, int group_rows) {
  constexpr int NV = HD / kWave;
  typedef float vec_t __attribute__((ext_vector_type(NV)));
  __shared__ vec_t red[W][kWave];
  const int lane = threadIdx.x & (kWave - 1), part = uniform((int)threadIdx.x / kWave), wave = W == 1 ? 0 : part;
  const int hq = W == 1 ? (int)blockIdx.y * 4 + part : (int)blockIdx.y, bs = (int)blockIdx.x;
  if (hq >= a.heads) return;  // uniform over the wave (W == 1: no barrier below)
  const int group = a.heads / a.kvh, b = bs / a.t, st = bs - b * a.t, kh = hq / group;
  const int r = st * group + hq - kh * group, rg = r / group_rows, rl = r - rg * group_rows;
  const int64_t base = (((int64_t)(b * a.kvh + kh) * a.row_groups + rg) * a.n_split) * group_rows + rl;
  uint16_t* const orow = a.out + a.orow.at(b, hq, st) + NV * lane;
  const uint16_t* const grow = a.gate ? a.gate + a.gr.at(b, hq, st) + NV * lane : nullptr;
  uint16_t gate[NV] = {};
  if (grow) {
#pragma unroll
    for (int e = 0; e < NV; ++e) gate[e] = grow[e];
  }
  vec_t v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int s = min(wave + W * i, a.n_split - 1);  // no branch around a load: past the last split, that one again
    v[i] = *reinterpret_cast<const vec_t*>(a.part_o + (base + (int64_t)s * group_rows) * HD + NV * lane);
  }
  float w[N], sum = 0.f;
  const float* const ml = a.part_ml + base * 2;
  if constexpr (W == 1) {
    float m[N], l[N], mx = kNoKey;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float2 x = *reinterpret_cast<const float2*>(ml + (int64_t)min(i, a.n_split - 1) * group_rows * 2);
      m[i] = i < a.n_split ? x.x : -INFINITY;
      l[i] = i < a.n_split ? x.y : 0.f;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) mx = fmaxf(mx, m[i]);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      w[i] = __builtin_amdgcn_exp2f(m[i] - mx);
      sum = fmaf(l[i], w[i], sum);
      if (m[i] == -INFINITY) v[i] = vec_t{};
    }
  } else {
    const bool live = lane < a.n_split;
    const float2 x = *reinterpret_cast<const float2*>(ml + (int64_t)min(lane, a.n_split - 1) * group_rows * 2);
    const float m = live ? x.x : -INFINITY, l = live ? x.y : 0.f;
    const float mx = fmaxf(wave_max(m), kNoKey), wt = __builtin_amdgcn_exp2f(m - mx);
    sum = wave_sum(l * wt);
    const uint64_t held = __ballot(m != -INFINITY);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int s = wave + W * i;
      w[i] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wt), s));
      if (!(held >> s & 1ull)) v[i] = vec_t{};  // nor past the last split
    }
  }
  vec_t acc = {};
#pragma unroll
  for (int i = 0; i < N; ++i) acc += v[i] * w[i];
  if (W > 1) {
    red[wave][lane] = acc;
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int i = 1; i < W; ++i) acc += red[i][lane];
  }
  const float inv = row_inverse(sum);
  float odd = sum < least_sum(a) ? 1.f : 0.f;
#pragma unroll
  for (int e = 0; e < NV; ++e) {
    const float y = acc[e] * inv;
    odd = fmaf(y, 0.f, odd);
    orow[e] = f32_to_bf16(grow ? y * sigmoid_of(gate[e]) : y);
  }
  if (__ballot(odd != 0.f) != 0ull) masked_row_slow<HD, true>(a, b, hq, st, lane);
}

namespace {

// Rows of a workgroup: one wave's, two's or four's.
int64_t masked_group_rows(int64_t rows) { return rows <= 32 ? 32 : rows <= 64 ? 64 : 128; }
int64_t masked_row_groups(int64_t rows) { return (rows + masked_group_rows(rows) - 1) / masked_group_rows(rows); }

// Up to 32 rows: eight waves a workgroup while the lanes' workgroups stay within the compute units, where more of a
// lane's keys are on their way at once and fewer splits are left to merge (one lane of 300 keys, heads of 64: 7.4 -> 6.3
// us; 48 of 4000 keys, 4 kv heads of 128: 79.5 -> 72 us); four, and two workgroups a unit, for more of them (48 of 500
// keys, 8 kv heads: 20.3 us with four, 23.9 with eight). The tiles of eight waves of 256 channels do not fit LDS.
bool masked_eight(int64_t lanes_kvh, int64_t hd) { return hd < 256 && lanes_kvh <= device_cu_count(); }

// Key splits. At most what the device holds at once: 48 lanes of 2 kv heads of 256 (96 workgroups), one step with a
// window of 4096, one workgroup a compute unit: 2 splits 82 us, 4 89, 8 90; four steps over 8000 keys, two a unit: 5 splits
// 149 us, 4 153, 6 202. At most sqrt(32 tiles / workgroups): a split's tiles get fewer with each, but its start, its
// partial sums and their merge are there for every workgroup (8 of these lanes, four steps over 1000 keys: 4 splits
// 21.6 us, 8 20.1, 16 22.0; 24 lanes: 4 24.1, 6 23.6, 12 35). And some tiles for each: with up to 32 rows 4 for eight waves,
// 3 for four, and none split below 3 tiles a wave (one lane, heads of 64: 700 keys 7.3 us whole, 7.7 as 4; 1500 keys 10.2
// whole, 8.4 as 5, 7.7 as 12); else 2 (one lane, four steps over 700 keys: whole 33 us, 2 splits 22.6, 8 13.2, 12 12.4).
int masked_splits(int64_t batch, int64_t kvh, int64_t rows, int64_t hd, int64_t keys) {
  const int64_t wgs = std::max<int64_t>(batch * kvh * masked_row_groups(rows), 1);
  const int64_t per_cu = hd > 64 && rows <= 32 ? 1 : 2;  // what LDS holds
  const int64_t tiles = (keys + kTileKeys - 1) / kTileKeys;
  const int64_t waves = masked_eight(batch * kvh, hd) ? 8 : 4;
  if (rows <= 32 && tiles <= 3 * waves) return 1;
  int64_t n = std::min<int64_t>(device_cu_count() * per_cu / wgs, tiles / (rows > 32 ? 2 : waves == 8 ? 4 : 3));
  n = std::min<int64_t>(n, (int64_t)std::sqrt(32. * (double)tiles / (double)wgs));
  n = std::min<int64_t>(n, kMaskedSplits);
  return n < 1 ? 1 : (int)n;
}

template <int HD, bool CAP, bool SLOPES, bool TREE>
void masked_few_launch(const MaskedArgs& a, dim3 grid, hipStream_t st) {
  if constexpr (HD < 256) {
    if (masked_eight(a.lanes_kvh, HD)) {
      hipLaunchKernelGGL((k_masked_few<HD, 8, CAP, SLOPES, TREE>), grid, dim3(512), 0, st, a);
      return;
    }
  }
  hipLaunchKernelGGL((k_masked_few<HD, 4, CAP, SLOPES, TREE>), grid, dim3(256), 0, st, a);
}

template <int HD, bool CAP, bool SLOPES, bool TREE = false>
int masked_launch(const MaskedArgs& a, int64_t batch, hipStream_t st) {
  const int64_t rows = (int64_t)(a.heads / a.kvh) * a.t;
  const dim3 grid((unsigned)(batch * a.kvh * a.row_groups), (unsigned)a.n_split);
  if (rows <= 32)
    masked_few_launch<HD, CAP, SLOPES, TREE>(a, grid, st);
  else if (rows <= 64)
    hipLaunchKernelGGL((k_masked_rows<HD, 2, CAP, SLOPES, TREE>), grid, dim3(128), 0, st, a);
  else
    hipLaunchKernelGGL((k_masked_rows<HD, 4, CAP, SLOPES, TREE>), grid, dim3(256), 0, st, a);
  int rc = status_of(hipGetLastError());
  if (rc || a.n_split == 1) return rc;
  const int out_rows = (int)(batch * a.heads * a.t), group_rows = (int)masked_group_rows(rows);
  if constexpr (TREE) {
    const unsigned nodes = (unsigned)(batch * a.t), heads = (unsigned)a.heads;
    auto merge = [&](auto waves, auto n) {
      const unsigned y = waves == 1 ? (heads + 3) / 4 : heads;
      hipLaunchKernelGGL((k_tree_merge<HD, decltype(waves)::value, decltype(n)::value>), dim3(nodes, y), dim3(256), 0, st, a, group_rows);
    };
    constexpr std::integral_constant<int, 1> one{};
    constexpr std::integral_constant<int, 2> two{};
    constexpr std::integral_constant<int, 4> four{};
    constexpr std::integral_constant<int, 8> eight{};
    constexpr std::integral_constant<int, 16> sixteen{};
    if (a.n_split <= 2)
      merge(one, two);
    else if (a.n_split <= 4)
      merge(one, four);
    else if (a.n_split <= 8)
      merge(one, eight);
    else if (a.n_split <= 16)
      merge(four, four);
    else if (a.n_split <= 32)
      merge(four, eight);
    else
      merge(four, sixteen);
  } else if (a.n_split <= kMergeOne)
    hipLaunchKernelGGL((k_masked_merge<HD, 1>), dim3((unsigned)((out_rows + 3) / 4)), dim3(256), 0, st, a, out_rows, group_rows);
  else
    hipLaunchKernelGGL((k_masked_merge<HD, 4>), dim3((unsigned)out_rows), dim3(256), 0, st, a, out_rows, group_rows);
  return status_of(hipGetLastError());
}

template <int HD>
int masked_flags(const MaskedArgs& a, int64_t batch, hipStream_t st) {
  const bool cap = a.cap2 > 0.f && a.cap2 <= kCapMost;  // a wider one: in full for every tile, with a maximum
  if (a.slopes) return cap ? masked_launch<HD, true, true>(a, batch, st) : masked_launch<HD, false, true>(a, batch, st);
  return cap ? masked_launch<HD, true, false>(a, batch, st) : masked_launch<HD, false, false>(a, batch, st);
}

bool masked_shape(int64_t batch, int64_t t, int64_t heads, int64_t kv_heads, int64_t head_dim) {
  return batch > 0 && t > 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0 &&
         (head_dim == 64 || head_dim == 128 || head_dim == 256) && batch <= INT32_MAX / 64 / t &&
         heads <= INT32_MAX / 64 / (batch * t) && batch * kv_heads * masked_row_groups(heads / kv_heads * t) <= kMaxGroups;
}

int64_t masked_workspace(int64_t batch, int64_t t, int64_t heads, int64_t kv_heads, int64_t head_dim, int n_split) {
  if (!masked_shape(batch, t, heads, kv_heads, head_dim) || n_split <= 1) return 0;
  const int64_t rows = heads / kv_heads * t;
  return batch * kv_heads * masked_row_groups(rows) * masked_group_rows(rows) * n_split * (head_dim + 2) * 4;
}

// The operands that every call has, checked and taken down. False: refused.
bool masked_operands(MaskedArgs& a, const uint16_t* q, const int64_t* q_strides, const uint16_t* gate, const int64_t* gate_strides,
                     int64_t batch, int64_t t, int64_t heads, int64_t kv_heads, int64_t head_dim, const uint16_t* k_pool,
                     const uint16_t* v_pool, int64_t pool_rows, const int32_t* block_table, int64_t table_stride,
                     const int64_t* base_pos, float scale, int n_split, void* workspace, int64_t workspace_bytes, uint16_t* out,
                     const int64_t* out_strides) {
  if (!masked_shape(batch, t, heads, kv_heads, head_dim)) return false;
  if (pool_rows <= 0 || pool_rows % kAttnBlock || table_stride <= 0 || table_stride > (1 << 26) || kv_heads > 4096) return false;
  if (!(scale > 0.f) || !(scale < INFINITY)) return false;
  if (n_split < 1 || n_split > kMaskedSplits) return false;
  if (n_split > kMergeOne && batch * t * heads > kMaxGroups) return false;  // the merge's workgroups
  // 16-byte accesses to query, gate and output rows and to the pools
  if (!aligned16(q) || !aligned16(k_pool) || !aligned16(v_pool) || !aligned16(out) || (gate && !aligned16(gate))) return false;
  for (int i = 0; i < 3; ++i)
    if (q_strides[i] % 8 || out_strides[i] % 8 || (gate && gate_strides[i] % 8)) return false;
  if (n_split > 1 && (!workspace || !aligned16(workspace) ||
                      workspace_bytes < masked_workspace(batch, t, heads, kv_heads, head_dim, n_split)))
    return false;
  const int64_t rows = heads / kv_heads * t;
  a.q = q;
  a.qr = {q_strides[0], q_strides[1], q_strides[2]};
  a.out = out;
  a.orow = {out_strides[0], out_strides[1], out_strides[2]};
  a.gate = gate;
  if (gate) a.gr = {gate_strides[0], gate_strides[1], gate_strides[2]};
  a.k_pool = k_pool;
  a.v_pool = v_pool;
  a.pool_blocks = (uint32_t)std::min<int64_t>(pool_rows / kAttnBlock, (int64_t)1 << 31);
  a.table = block_table;
  a.table_stride = table_stride;
  a.base = base_pos;
  a.t = (int)t;
  a.heads = (int)heads;
  a.kvh = (int)kv_heads;
  a.lanes_kvh = (int)(batch * kv_heads);
  a.n_split = n_split;
  a.row_groups = (int)masked_row_groups(rows);
  a.c0 = scale * kLog2e;
  a.part_o = (float*)workspace;
  a.part_ml = a.part_o ? a.part_o + batch * kv_heads * a.row_groups * masked_group_rows(rows) * n_split * head_dim : nullptr;
  return true;
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
  if (window > 0 && window < keys) keys = std::min(keys, window + masked_group_rows(rows) / (heads / kv_heads) + kTileKeys);
  return masked_splits(batch, kv_heads, rows, head_dim, keys);
}

int64_t mtpk_attention_masked_workspace_bytes(int64_t batch, int64_t t, int64_t heads, int64_t kv_heads,
                                              int64_t head_dim, int n_split) {
  return masked_workspace(batch, t, heads, kv_heads, head_dim, n_split);
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
  MaskedArgs a{};
  if (!masked_operands(a, q, q_strides, gate, gate_strides, batch, t, heads, kv_heads, head_dim, k_pool, v_pool, pool_rows,
                       block_table, table_stride, base_pos, scale, n_split, workspace, workspace_bytes, out, out_strides))
    return MTPK_EINVAL;
  if (!(softcap >= 0.f) || !(softcap < INFINITY) || window < 0) return MTPK_EINVAL;
  if (prefix && prefix_dtype != MTPK_I32 && prefix_dtype != MTPK_I64) return MTPK_EINVAL;
  if (first && first_dtype != MTPK_I32 && first_dtype != MTPK_I64) return MTPK_EINVAL;
  a.slopes = slopes;
  a.prefix = prefix;
  a.prefix_dt = prefix_dtype;
  a.first = first;
  a.first_dt = first_dtype;
  a.window = (int)std::min<int64_t>(window, INT32_MAX);
  if (softcap > 0.f) {
    // tanh(u) / u by polynomials in u^2 of least relative error: 8.4e-6 on |u| <= 0.15, which is 9e-5 of an exponent
    // at cap 50 (a rounded probability is off by up to 2^-8), and 4e-7 on |u| <= 0.25
    // (scores of 1e-30 caps are as good as infinite ones: the constants, and a score of 0 times them, stay finite)
    const double k = std::min((double)scale / softcap, 1e30), c = (double)softcap * 1.4426950408889634;
    a.cap2 = (float)std::min(c, 1.7e38);  // twice it stays finite
    a.cap_in = (float)(2. * 1.4426950408889634 * k);
    a.cubic_max = (float)(0.15 / k);
    a.cap_k = (float)k;
    a.e0 = (float)(c * k * 0.99999961);
    a.e1 = (float)(c * k * -0.33321928);
    a.e2 = (float)(c * k * 0.12841935);
    if (c <= kCapMost) {
      a.c0 = (float)(c * k * 0.99999165);
      a.c1 = (float)std::max(c * k * k * k * -0.33035765, -3e38);
    }
  }
  const hipStream_t st = (hipStream_t)stream;
  switch (head_dim) {
    case 64: return masked_flags<64>(a, batch, st);
    case 128: return masked_flags<128>(a, batch, st);
    default: return masked_flags<256>(a, batch, st);
  }
}

int mtpk_attention_tree_splits(int64_t batch, int64_t t, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t max_ctx) {
  if (t > kTreeNodes || !masked_shape(batch, t, heads, kv_heads, head_dim) || max_ctx < 0) return 0;
  return masked_splits(batch, kv_heads, heads / kv_heads * t, head_dim, max_ctx);
}

int64_t mtpk_attention_tree_workspace_bytes(int64_t batch, int64_t t, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                            int n_split) {
  return t > kTreeNodes ? 0 : mtpk_attention_masked_workspace_bytes(batch, t, heads, kv_heads, head_dim, n_split);
}

int mtpk_paged_attention_tree(const uint16_t* q, const int64_t* q_strides, const uint16_t* gate, const int64_t* gate_strides,
                              int64_t batch, int64_t t, int64_t heads, int64_t kv_heads, int64_t head_dim, const uint16_t* k_pool,
                              const uint16_t* v_pool, int64_t pool_rows, const int32_t* block_table, int64_t table_stride,
                              const int64_t* base_pos, float scale, const void* parents, int parents_dtype,
                              const int64_t* parents_strides, int n_split, void* workspace, int64_t workspace_bytes, uint16_t* out,
                              const int64_t* out_strides, void* stream) {
  if (!q || !k_pool || !v_pool || !block_table || !base_pos || !parents || !out || !q_strides || !out_strides || !parents_strides)
    return MTPK_EINVAL;
  if (gate && !gate_strides) return MTPK_EINVAL;
  if (t < 1 || t > kTreeNodes || (parents_dtype != MTPK_I32 && parents_dtype != MTPK_I64)) return MTPK_EINVAL;
  if (batch == 0) return 0;
  MaskedArgs a{};
  if (!masked_operands(a, q, q_strides, gate, gate_strides, batch, t, heads, kv_heads, head_dim, k_pool, v_pool, pool_rows,
                       block_table, table_stride, base_pos, scale, n_split, workspace, workspace_bytes, out, out_strides))
    return MTPK_EINVAL;
  // the merge's grid
  if (heads > 65535 || (n_split > 1 && batch * t * (n_split <= 8 ? (heads + 3) / 4 : heads) > kMaxGroups)) return MTPK_EINVAL;
  a.tree = {parents, parents_dtype, parents_strides[0], parents_strides[1]};
  const hipStream_t st = (hipStream_t)stream;
  switch (head_dim) {
    case 64: return masked_launch<64, false, false, true>(a, batch, st);
    case 128: return masked_launch<128, false, false, true>(a, batch, st);
    default: return masked_launch<256, false, false, true>(a, batch, st);
  }
}

}  // extern "C"
