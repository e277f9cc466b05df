// The Gated DeltaNet rows of a tree of drafts (mtpk_tree.h): the delta rule's inputs, with the convolution along
// each node's own path; the rule itself, each node from its parent's state; and the advance of the stored
// state and convolution window along the accepted path.

#include <algorithm>

#include "mtpk_deltanet_step.h"
#include "mtpk_host.h"
#include "mtpk_tree.h"

namespace mtpk {

constexpr int kTreeConvMost = 8;  // conv_k - 1 at most
constexpr int kTreeHeadMost = 256;  // widest head of the preparation

// ---------------------------------------------------------------- inputs
//
// As mtpk_deltanet_prep, but the columns before a node are its ancestors' (then the stored window's), which are the
// highest bits of its ancestors. A wave takes one head unit (the q heads, the k heads, the v heads, and one more for g
// and beta) of up to R nodes of a lane: lane l holds channels 2 l, 2 l + 1 (+ 128), and the columns of all
// nodes and taps are on their way at once.
//
// The convolution's output is a tensor of the model's type. Next to a rounding's border the order of the products decides
// to which side a value goes, half a step of bf16 either way: the few outputs of bf16 rows that lie nearer to one than 32
// bits tell (1 in some 500) are done again in 64, from the products, which are exact. Of f32 rows there is nothing to round,
// and the sums run as in mtpk_deltanet_prep.
constexpr int kPrepThreads = 256;

struct TreePrepArgs {
  const void* proj;  // [B * t, proj_stride]: qkv (C), z, b (vh), a (vh)
  int64_t proj_stride;
  const void* conv;  // [slots, C, k1]
  const int64_t* slot;
  int64_t slots_total;
  const void* conv_w;  // [C, conv_k]
  const float* a_log;
  const float* dt_bias;
  TreeParents parents;
  int B, t, kh, kd, vh, vd, conv_k;
  float eps, q_scale;
  float *q, *k, *v, *g, *beta;
};

template <typename T>
__device__ inline float tree_float(const void* p, int64_t i) {
  if constexpr (sizeof(T) == 2)
    return bf16_to_f32(static_cast<const uint16_t*>(p)[i]);
  else
    return static_cast<const float*>(p)[i];
}

// Channels c, c + 1 of row `row` of the lane's rows in `r`, `stride` bytes apart; `two`: both exist. PAIR: a dword of two bf16.
template <typename T, bool PAIR>
__device__ inline float2 tree_pair(rsrc_t r, int c, int row, int stride, bool two) {
  const int off = c * (int)sizeof(T), at = row * stride;
  if constexpr (PAIR) {
    const uint32_t d = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(r, off, at, 0);
    return make_float2(bits_f32(d << 16), bits_f32(d & 0xffff0000u));
  } else if constexpr (sizeof(T) == 2) {
    const uint32_t d = (uint32_t)__builtin_amdgcn_raw_buffer_load_b16(r, off, at, 0) & 0xffffu;
    const uint32_t e = (uint32_t)__builtin_amdgcn_raw_buffer_load_b16(r, two ? off + 2 : off, at, 0) & 0xffffu;
    return make_float2(bits_f32(d << 16), two ? bits_f32(e << 16) : 0.f);
  } else {
    typedef uint32_t pair_t __attribute__((ext_vector_type(2)));
    const pair_t d = __builtin_bit_cast(pair_t, __builtin_amdgcn_raw_buffer_load_b64(r, off, at, 0));
    return make_float2(bits_f32(d[0]), two ? bits_f32(d[1]) : 0.f);
  }
}

__device__ inline float tree_silu(float x) { return x / (1.f + expf(-x)); }

// The same within 8 units of the last place, in half of the instructions: e^-x as 2^p (1 + what p was rounded by), the
// division by a reciprocal and a step towards the exact quotient.
__device__ inline float tree_silu_near(float x) {
  constexpr float kLog2eHi = 1.44269502f, kLog2eLo = 1.92596303e-8f;
  const float p = -x * kLog2eHi, rest = fmaf(-x, kLog2eLo, fmaf(-x, kLog2eHi, -p)), e = __builtin_amdgcn_exp2f(p);
  const float d = 1.f + fmaf(e, rest * 0.693147182f, e), r = __builtin_amdgcn_rcpf(d), y = x * r;
  return d < INFINITY ? fmaf(fmaf(-d, y, x), r, y) : y;
}

// K: conv_k, or 0 for any. NI: 128-channel parts of a head.
template <typename T, int K, bool PAIR, int NI, int R>
__global__ __launch_bounds__(kPrepThreads) void k_tree_prep(TreePrepArgs a) {
  constexpr int KM = K ? K : kTreeConvMost + 1;
  const int lane = threadIdx.x & (kWave - 1);
  const int conv_k = K ? K : a.conv_k, k1 = conv_k - 1;
  const int units = 2 * a.kh + a.vh + 1, groups = (a.t + R - 1) / R;
  const int64_t id = (int64_t)blockIdx.x * (kPrepThreads / kWave) + uniform((int)threadIdx.x / kWave);
  if (id >= (int64_t)a.B * groups * units) return;
  const int u = (int)(id % units), br = (int)(id / units), b = br / groups, s0 = (br - b * groups) * R;
  const int64_t row0 = (int64_t)b * a.t;
  const int C = 2 * a.kh * a.kd + a.vh * a.vd;
  const int parent = a.parents.at(b, lane, a.t);
  if (u == units - 1) {
    const uint64_t seen = tree_ancestors(parent, lane);
    const uint64_t nodes = __ballot(seen != 0ull);
    for (int i = lane; i < min(R, a.t - s0) * a.vh; i += kWave) {
      const int s = s0 + i / a.vh, h = i % a.vh;
      const int64_t at = (row0 + s) * a.proj_stride + C + a.vh * a.vd + h;
      const bool present = nodes >> s & 1ull;
      const float x = __fadd_rn(tree_float<T>(a.proj, at + a.vh), a.dt_bias[h]);
      const float sp = x > 20.f ? x : log1pf(expf(x));
      a.beta[(row0 + s) * a.vh + h] = present ? 1.f / (1.f + expf(-tree_float<T>(a.proj, at))) : 0.f;
      a.g[(row0 + s) * a.vh + h] = present ? -expf(a.a_log[h]) * sp : 0.f;
    }
    return;
  }
  const bool is_v = u >= 2 * a.kh;
  const int dim = is_v ? a.vd : a.kd;
  const int c0 = is_v ? 2 * a.kh * a.kd + (u - 2 * a.kh) * a.vd : u * a.kd;
  const int64_t slot = a.slot[b];
  const bool slot_ok = slot >= 0 && slot < a.slots_total;
  float2 w[NI][KM], stored[NI][KM - 1];
#pragma unroll
  for (int n = 0; n < NI; ++n) {
    const int ch = 2 * lane + 128 * n, c = c0 + (ch < dim ? ch : 0);
    const bool two = ch + 1 < dim;
    if constexpr (PAIR && K == 4) {  // two channels of 4 taps, and of 3 columns
      const u32x4_t d = ld16(static_cast<const uint16_t*>(a.conv_w) + (int64_t)c * 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t x = d[j / 2], y = d[2 + j / 2];
        w[n][j] = make_float2(bits_f32(j % 2 ? x & 0xffff0000u : x << 16), bits_f32(j % 2 ? y & 0xffff0000u : y << 16));
      }
      uint32_t e[3] = {0u, 0u, 0u};
      if (slot_ok) {
        const uint32_t* const p = reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(a.conv) + (slot * C + c) * 3);
#pragma unroll
        for (int j = 0; j < 3; ++j) e[j] = p[j];
      }
      stored[n][0] = make_float2(bits_f32(e[0] << 16), bits_f32(e[1] & 0xffff0000u));
      stored[n][1] = make_float2(bits_f32(e[0] & 0xffff0000u), bits_f32(e[2] << 16));
      stored[n][2] = make_float2(bits_f32(e[1] << 16), bits_f32(e[2] & 0xffff0000u));
    } else {
#pragma unroll
      for (int j = 0; j < KM; ++j) {
        w[n][j] = make_float2(0.f, 0.f);
        if (j < conv_k) {
          const int64_t i = (int64_t)c * conv_k + j;
          w[n][j] = make_float2(tree_float<T>(a.conv_w, i), two ? tree_float<T>(a.conv_w, i + conv_k) : 0.f);
        }
        if (j == KM - 1) continue;
        stored[n][j] = make_float2(0.f, 0.f);
        if (j < k1 && slot_ok) {
          const int64_t i = (slot * C + c) * k1 + j;
          stored[n][j] = make_float2(tree_float<T>(a.conv, i), two ? tree_float<T>(a.conv, i + k1) : 0.f);
        }
      }
    }
  }
  const uint64_t seen = tree_ancestors(parent, lane);
  // tap j of node s0 + r: its ancestor conv_k - 1 - j generations up, or column `from` of the stored window
  float2 x[R][NI][KM];
  uint64_t way[R];
  const int stride = (int)(a.proj_stride * (int)sizeof(T));
  const rsrc_t rows = make_rsrc(static_cast<const T*>(a.proj) + row0 * a.proj_stride, (uint32_t)((a.t - 1) * stride + C * (int)sizeof(T)));
#pragma unroll
  for (int r = 0; r < R; ++r) {
    way[r] = s0 + r < a.t ? lane_bits(seen, s0 + r) : 0ull;
    uint64_t m = way[r];
#pragma unroll
    for (int j = KM - 1; j >= 0; --j) {
      if (j >= conv_k) continue;
      const bool raw = m != 0ull;
      const int i = raw ? 63 - __builtin_clzll(m) : 0;  // else loaded for nothing: no branch around the loads
      m &= ~(1ull << i);
#pragma unroll
      for (int n = 0; n < NI; ++n) {
        const int ch = 2 * lane + 128 * n, c = c0 + (ch < dim ? ch : 0);
        x[r][n][j] = tree_pair<T, PAIR>(rows, c, i, stride, ch + 1 < dim);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (s0 + r >= a.t) continue;
    const int above = __builtin_popcountll(way[r]);  // columns of the tree
    // the columns before those are the stored window's last ones: tap j has column j + above - 1
    if (above < conv_k) {  // uniform, and rare past the first generations
#pragma unroll
      for (int d = 0; d < KM; ++d) {
        if (d != above) continue;
#pragma unroll
        for (int j = 0; j < KM; ++j)
#pragma unroll
          for (int n = 0; n < NI; ++n)
            if (j + d < conv_k) x[r][n][j] = j + d > 0 ? stored[n][j + d - 1 < KM - 1 ? j + d - 1 : 0] : make_float2(0.f, 0.f);
      }
    }
    float2 y[NI];
    float ss = 0.f;
#pragma unroll
    for (int n = 0; n < NI; ++n) {
      const int ch = 2 * lane + 128 * n;
      float f[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float acc = 0.f, size = 0.f, prod[KM];
#pragma unroll
        for (int j = 0; j < KM; ++j) {
          if (j >= conv_k) continue;
          prod[j] = __fmul_rn(e ? x[r][n][j].y : x[r][n][j].x, e ? w[n][j].y : w[n][j].x);
          acc = j == 0 ? prod[j] : __fadd_rn(acc, prod[j]);
          size += fabsf(prod[j]);
        }
        if constexpr (sizeof(T) == 2) {
          // An addition is off by 2^-24 of what it gives, which is at most the products' size, SiLU's slope is below 1.1, and
          // its own error at most 1.25 x 2^-22 of the value (2^-23 of the exponential, 2^-24 of the sum, the quotient and its step each).
          float y = tree_silu_near(acc);
          const float border = bits_f32((f32_bits(y) & 0xffff0000u) | 0x8000u);  // between two bf16 values
          if (!(fabsf(y - border) > fmaf((float)k1 * 0x1.2p-24f, size, 0x1.4p-22f * fabsf(y)))) {
            double exact = 0.;
#pragma unroll
            for (int j = 0; j < KM; ++j)
              if (j < conv_k) exact += (double)prod[j];
            y = (float)(exact / (1.0 + exp(-exact)));
          }
          f[e] = bf16_to_f32(f32_to_bf16(y));
        } else {
          f[e] = tree_silu(acc);
        }
        if (ch + e >= dim) f[e] = 0.f;
        ss += f[e] * f[e];
      }
      y[n] = make_float2(f[0], f[1]);
    }
    float scale = 1.f;
    if (!is_v) scale = rsqrtf(wave_sum(ss) + a.eps);
    const int64_t rs = row0 + s0 + r;
    float* const to = is_v ? a.v + (rs * a.vh + (u - 2 * a.kh)) * a.vd
                           : (u < a.kh ? a.q + (rs * a.kh + u) * a.kd : a.k + (rs * a.kh + (u - a.kh)) * a.kd);
#pragma unroll
    for (int n = 0; n < NI; ++n) {
      const int ch = 2 * lane + 128 * n;
      float2 o = y[n];
      if (!is_v) {
        o = make_float2(o.x * scale, o.y * scale);
        if (u < a.kh) o = make_float2(o.x * a.q_scale, o.y * a.q_scale);
      }
      if (above == 0) o = make_float2(0.f, 0.f);  // an absent node
      if constexpr (PAIR) {
        if (ch < dim) *reinterpret_cast<float2*>(to + ch) = o;
      } else {
        if (ch < dim) to[ch] = o.x;
        if (ch + 1 < dim) to[ch + 1] = o.y;
      }
    }
  }
}

// Nodes of a wave: the way to a node and the weights are the wave's, four nodes share them where there are waves enough. bf16, 96
// head units, two / four: one lane of 7 nodes 4.2 / 5.9 us, 8 of 16 8.0 / 8.6, 48 of 4 10.6 / 10.3, 48 of 16 26.2 / 23.3 (eight 32).
// Bound by its instructions, of which SiLU and its border are the most: 60.8 MB in 23.3 us.
template <typename T, int K, bool PAIR, int NI, int R>
int launch_tree_prep_nodes(const TreePrepArgs& a, hipStream_t st) {
  const int64_t waves = (int64_t)a.B * ((a.t + R - 1) / R) * (2 * a.kh + a.vh + 1), n = (waves + 3) / 4;
  if (n > kMaxGroups) return MTPK_EINVAL;
  hipLaunchKernelGGL((k_tree_prep<T, K, PAIR, NI, R>), dim3((unsigned)n), dim3(kPrepThreads), 0, st, a);
  return status_of(hipGetLastError());
}

template <typename T, int K, bool PAIR, int NI>
int launch_tree_prep_heads(const TreePrepArgs& a, hipStream_t st) {
  if (a.t <= 2) return launch_tree_prep_nodes<T, K, PAIR, NI, 2>(a, st);
  if ((int64_t)a.B * a.t * (2 * a.kh + a.vh) >= 64 * (int64_t)device_cu_count()) return launch_tree_prep_nodes<T, K, PAIR, NI, 4>(a, st);
  return launch_tree_prep_nodes<T, K, PAIR, NI, 2>(a, st);
}

template <typename T, int K, bool PAIR>
int launch_tree_prep(const TreePrepArgs& a, hipStream_t st) {
  return a.kd > 128 || a.vd > 128 ? launch_tree_prep_heads<T, K, PAIR, 2>(a, st) : launch_tree_prep_heads<T, K, PAIR, 1>(a, st);
}

// ---------------------------------------------------------------- the rule, step by step
//
// A lane of the wave owns a column of the state, as in the chain's form, and takes the nodes in order. The state that it
// holds is the last node's: a node that hangs below it goes on from there, any other one starts from the stored state
// and walks its way from the root. So a chain costs a step a node, a tree its nodes' depths.
template <int DK>
__device__ __forceinline__ void tree_rule_column(const float* __restrict__ state, int64_t s_idx, int heads, int head, int row, int t,
                                                 int rep, int dv, int col, const float* __restrict__ q, const float* __restrict__ k,
                                                 const float* __restrict__ v, const float* __restrict__ g,
                                                 const float* __restrict__ beta, float* __restrict__ out, uint64_t seen, int lane,
                                                 float* kq) {
  constexpr int kPer = (DK + kWave - 1) / kWave;
  const bool live = col < dv;
  const rsrc_t rsm = make_rsrc(state + ((s_idx * heads + head) * DK) * (int64_t)dv, (uint32_t)(DK * dv * 4));
  const uint32_t vcol = live ? (uint32_t)col * 4u : kOutOfRange, drow = (uint32_t)dv * 4u;
  const int qk_heads = heads / rep, kh = head / rep;
  float s[DK];
  uint64_t held = 0ull;  // the node whose state s is, with its ancestors
  for (int node = 0; node < t; ++node) {
    const uint64_t way = lane_bits(seen, node);
    float* const to = out + (((int64_t)row * t + node) * heads + head) * dv + col;
    if (way == 0ull) {
      if (live) *to = 0.f;
      continue;
    }
    uint64_t left = way;
    if (held != 0ull && (held & ~way) == 0ull) {
      left = way & ~held;
    } else {
#pragma unroll
      for (int i = 0; i < DK; ++i)
        s[i] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rsm, (int)vcol, (int)(drow * i), 0));
    }
    held = way;
    while (left != 0ull) {
      const int at = __builtin_ctzll(left);
      left &= left - 1ull;
      const int64_t rs = (int64_t)row * t + at, hv = rs * heads + head;
      float nk[kPer], nq[kPer];
#pragma unroll
      for (int p = 0; p < kPer; ++p) {
        const int i = p * kWave + lane;
        nk[p] = i < DK ? k[(rs * qk_heads + kh) * DK + i] : 0.f;
        nq[p] = i < DK ? q[(rs * qk_heads + kh) * DK + i] : 0.f;
      }
      const float vv = live ? v[hv * dv + col] : 0.f, decay = __expf(g[hv]), bt = beta[hv];
      __syncthreads();  // the last step's reads are over (a one-wave workgroup, or all waves alike)
#pragma unroll
      for (int p = 0; p < kPer; ++p) {
        const int i = p * kWave + lane;
        if (i < DK) {
          kq[i] = nk[p];
          kq[DK + i] = nq[p];
        }
      }
      __syncthreads();
      const float4* const kk = reinterpret_cast<const float4*>(kq);
      const float4* const qq = reinterpret_cast<const float4*>(kq + DK);
      float mem = 0.f, o = 0.f;
#pragma unroll
      for (int i4 = 0; i4 < DK / 4; ++i4) {
        const float4 kv = kk[i4];
        const float kr[4] = {kv.x, kv.y, kv.z, kv.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[4 * i4 + e] *= decay;
          mem = fmaf(s[4 * i4 + e], kr[e], mem);
        }
      }
      const float delta = (vv - mem) * bt;
      asm volatile("" ::: "memory");  // k is read again rather than kept: the state takes DK registers
#pragma unroll
      for (int i4 = 0; i4 < DK / 4; ++i4) {
        const float4 kv = kk[i4], qv = qq[i4];
        const float kr[4] = {kv.x, kv.y, kv.z, kv.w}, qr[4] = {qv.x, qv.y, qv.z, qv.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[4 * i4 + e] = fmaf(kr[e], delta, s[4 * i4 + e]);
          o = fmaf(s[4 * i4 + e], qr[e], o);
        }
      }
      if (left == 0ull && live) *to = o;
    }
  }
}

template <int DK>
__global__ __launch_bounds__(kWave) void k_tree_rule_steps(const float* __restrict__ state, int64_t slots_total,
                                                           const int64_t* __restrict__ slot, int t, int heads, int rep, int dv,
                                                           const float* __restrict__ q, const float* __restrict__ k,
                                                           const float* __restrict__ v, const float* __restrict__ g,
                                                           const float* __restrict__ beta, TreeParents parents,
                                                           float* __restrict__ out) {
  __shared__ __attribute__((aligned(16))) float kq[2 * DK];
  const int nblk = (dv + kWave - 1) / kWave, bh = (int)blockIdx.x / nblk, row = bh / heads, head = bh - row * heads;
  const int lane = threadIdx.x, col = ((int)blockIdx.x - bh * nblk) * kWave + lane;
  const int64_t s_idx = slot ? slot[row] : row;
  const int parent = parents.at(row, lane, t);
  uint64_t seen = tree_ancestors(parent, lane);
  if (s_idx < 0 || s_idx >= slots_total) {  // no such slot: zero outputs, no state access
    if (col < dv)
      for (int i = 0; i < t; ++i) out[(((int64_t)row * t + i) * heads + head) * dv + col] = 0.f;
    return;
  }
  tree_rule_column<DK>(state, s_idx, heads, head, row, t, rep, dv, col, q, k, v, g, beta, out, seen, lane, kq);
}

// ---------------------------------------------------------------- the rule, all nodes at once
//
// With A(s) node s and its ancestors, G_s the sum of g over A(s), and S the stored state, the steps along every way are
//   u_s = beta_s (v_s - e^(G_s) S^T k_s - sum over a in A(s), a != s, of e^(G_s - G_a) (k_a . k_s) u_a)
//   out_s = e^(G_s) S^T q_s + sum over a in A(s) of e^(G_s - G_a) (k_a . q_s) u_a
// which is the chunk form of a chain (mtpk_deltanet_chunk.h) with the ancestors in place of the earlier steps: parents come
// first, so the system is unit lower triangular again. The state is read once, whatever the tree's depth, and passes
// through two matrix products, K S and Q S.
//
// The products run on v_mfma_f32_16x16x32_bf16 at fp32's accuracy: each operand is three bf16 parts, 24 bits, each the rest of
// the ones before it rounded, and of the nine products of parts the six largest are taken; what is left out is below
// 2^-25 of the product. That is 96 cycles for 16 x 16 x 32 where v_mfma_f32_16x16x4_f32 takes 256. G is summed and
// differenced in 64 bits, in units of log2.
//
// A wave takes 64 columns of a (row, head)'s state, as four column tiles of every fourth column, so that a lane's load of the
// state is 16 bytes and a wave's 256 of a row. It streams through the products: 32 rows of it are multiplied with all
// nodes' k and q, held in LDS in parts, while the next ones are on their way. W waves to a workgroup, of the heads that
// share q and k and their columns.
//
// A masked element is a product with zero, so that what is not finite at one node would reach nodes off its way. Where
// a correction u comes out not finite, or the inputs are not the layer's (|k|^2 at most 1.01, g <= 0, beta in [0, 1]), the
// wave does its columns again one by one, and adds a node's own ancestors alone (48 lanes of 16 nodes, one head of one lane 204 us,
// all 937; one lane of 7 nodes 74).
struct TreeRuleArgs {
  const float* state;
  int64_t slots_total;
  const int64_t* slot;
  int t, heads, qk_heads, rep, dv, slabs;  // slabs: of 64 columns
  const float *q, *k, *v, *g, *beta;
  TreeParents parents;
  float* out;
};

// Three bf16 parts of four floats, in pairs.
struct Parts4 {
  uint32_t p[3][2];
};
__device__ inline Parts4 parts_of(f32x4_t x) {
  Parts4 r;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float a = x[2 * h], b = x[2 * h + 1];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const bf16x2_t y = {(__bf16)a, (__bf16)b};
      const uint32_t u = __builtin_bit_cast(uint32_t, y);
      r.p[i][h] = u;
      a -= bits_f32(u << 16);
      b -= bits_f32(u & 0xffff0000u);
    }
  }
  return r;
}

// Part i of eight values.
__device__ inline bf16x8_t part8(const Parts4& x, const Parts4& y, int i) {
  return as_bf16x8(u32x4_t{x.p[i][0], x.p[i][1], y.p[i][0], y.p[i][1]});
}

// The products that are taken, the smallest first: parts of the left and of the right operand.
constexpr int kPartProducts = 6;
__device__ inline constexpr int left_part(int i) { return i == 0 ? 2 : i == 2 || i == 4 ? 1 : 0; }
__device__ inline constexpr int right_part(int i) { return i == 1 ? 2 : i == 2 || i == 3 ? 1 : 0; }

// K's and Q's parts lie in `both` until the products with the state are done (as they are, and taken apart by every wave for
// itself, they were as fast for many lanes and slower for few: one lane of 7 nodes 10.3 against 11.9 us, of 30 14.5 against
// 17.4). k . k, q . k and the diagonal blocks lie behind them, and at 64 nodes, where LDS does not hold both, in their place.
template <int DK, int NT, int W>
struct TreeRuleLds {
  static constexpr int N = 16 * NT, kRow = (DK < 32 ? 32 : DK) + 8, kSq = N + 4, kDRow = 20, kDBlock = 16 * kDRow + 8;
  static constexpr bool OVER = NT == 4;
  struct Pairs {
    float kk[N][kSq], qk[N][kSq];
    float diag[W][NT][kDBlock];
  };
  struct Wave {
    double g[N];
    uint64_t seen[N];
    float beta[N], eg[N];
  };
  static constexpr int kPartBytes = 2 * 3 * N * kRow * 2, kPairBytes = (int)sizeof(Pairs);
  static constexpr int kPairsAt = OVER ? 0 : kPartBytes;
  static constexpr int kBytes = OVER ? (kPartBytes > kPairBytes ? kPartBytes : kPairBytes) : kPartBytes + kPairBytes;
  Wave w[W];
  __attribute__((aligned(16))) uint8_t both[kBytes];
  __device__ inline uint16_t* part(int of, int p, int row) { return reinterpret_cast<uint16_t*>(both) + ((of * 3 + p) * N + row) * kRow; }
  __device__ inline Pairs& pairs() { return *reinterpret_cast<Pairs*>(both + kPairsAt); }
};

// Node `lane`'s ancestors and itself, and the sum of x over them.
__device__ inline uint64_t tree_sums(int parent, int lane, double& x) {
  uint64_t m = parent >= -1 ? 1ull << lane : 0ull;
  int up = parent;
  while (__ballot(up >= 0) != 0ull) {
    const int at = up < 0 ? lane : up;
    const uint32_t lo = __shfl((uint32_t)m, at, kWave), hi = __shfl((uint32_t)(m >> 32), at, kWave);
    const double above = __shfl(x, at, kWave);
    const int next = __shfl(up, at, kWave);
    if (up >= 0) {
      m |= (uint64_t)hi << 32 | lo;
      x += above;
      up = next;
    }
  }
  return up == -1 ? m : 0ull;
}

// e to the difference of two sums in log2 units; 2^-25 of 1 at most from the rounding of the exponent.
__device__ inline float tree_decay(double x) { return __builtin_amdgcn_exp2f((float)x); }

// Column col of the wave's (row, head), node by node: the corrections into `out`, then, from the last node back, each
// one's output in its place, which no later one needs any more.
template <int DK, int NT, int W>
__device__ __forceinline__ void tree_rule_again(const TreeRuleArgs& a, TreeRuleLds<DK, NT, W>& s, int wave, const float* state, int row,
                                                int kh, int head, int col) {
  const auto& mine = s.w[wave];
  if (col >= a.dv) return;
  const int64_t hv = (int64_t)row * a.t * a.heads + head;
  auto along = [&](const float* xs, const float (*near)[TreeRuleLds<DK, NT, W>::kSq], int node, uint64_t others) {
    const float* const x = xs + (((int64_t)row * a.t + node) * a.qk_heads + kh) * DK;
    float dot = 0.f;
#pragma unroll 4
    for (int i = 0; i < DK; ++i) dot = fmaf(state[(int64_t)i * a.dv + col], x[i], dot);
    float sum = mine.eg[node] * dot;
#pragma unroll 1
    while (others != 0ull) {
      const int at = __builtin_ctzll(others);
      others &= others - 1ull;
      sum = fmaf(tree_decay(mine.g[node] - mine.g[at]) * near[node][at], a.out[(hv + (int64_t)at * a.heads) * a.dv + col], sum);
    }
    return sum;
  };
#pragma unroll 1
  for (int node = 0; node < a.t; ++node) {
    const uint64_t way = mine.seen[node];
    const int64_t at = (hv + (int64_t)node * a.heads) * a.dv + col;
    a.out[at] = way ? mine.beta[node] * (a.v[at] - along(a.k, s.pairs().kk, node, way & ~(1ull << node))) : 0.f;
  }
#pragma unroll 1
  for (int node = a.t - 1; node >= 0; --node) {
    const uint64_t way = mine.seen[node];
    if (way) a.out[(hv + (int64_t)node * a.heads) * a.dv + col] = along(a.q, s.pairs().qk, node, way);
  }
}

template <int DK, int NT, int W>
__global__ __launch_bounds__(W* kWave, NT > 2 ? 2 : 3) void k_tree_rule(TreeRuleArgs a) {
  using Lds = TreeRuleLds<DK, NT, W>;
  constexpr int N = Lds::N, DKP = DK < 32 ? 32 : DK, KB = DKP / 32, RING = NT < 4 && KB > 1 ? 2 : 1;
  __shared__ __attribute__((aligned(16))) Lds s;
  const int units = a.rep * a.slabs, wgs = (units + W - 1) / W;
  int id = blockIdx.x;
  const int part = id % wgs;
  id /= wgs;
  const int kh = id % a.qk_heads, row = id / a.qk_heads;
  const int tid = threadIdx.x, wave = uniform(tid / kWave), lane = tid & (kWave - 1), gq = lane >> 4, c = lane & 15;
  const int unit = part * W + wave;
  const bool on = unit < units;  // uniform over the wave
  const int head = kh * a.rep + (on ? unit / a.slabs : 0), col = (on ? unit % a.slabs : 0) * kWave + 4 * c;
  const bool live = on && col < a.dv;
  const int64_t s_idx = a.slot ? a.slot[row] : row;
  const int64_t hv0 = (int64_t)row * a.t * a.heads + head;
  if (s_idx < 0 || s_idx >= a.slots_total) {  // no such slot: zero outputs, no state access; uniform over the workgroup
    for (int i = gq; i < a.t; i += 4)
      if (live) *reinterpret_cast<f32x4_t*>(a.out + (hv0 + (int64_t)i * a.heads) * a.dv + col) = f32x4_t{0.f, 0.f, 0.f, 0.f};
    return;
  }
  const float* const state = a.state + (s_idx * a.heads + head) * DK * (int64_t)a.dv;
  const rsrc_t rs = make_rsrc(state, (uint32_t)(DK * a.dv * 4));
  const uint32_t drow = (uint32_t)a.dv * 4u;
  const uint32_t voff = live && 8 * gq < DK ? (uint32_t)(8 * gq) * drow + (uint32_t)col * 4u : kOutOfRange;
  f32x4_t st[RING][8];  // rows 32 kb + 8 gq + j, columns col .. col + 3
  auto load_state = [&](int kb) {
#pragma unroll
    for (int j = 0; j < 8; ++j) st[kb % RING][j] = __builtin_bit_cast(f32x4_t, buf16(rs, voff, drow * (uint32_t)(32 * kb + j)));
  };
  const int parent = a.parents.at(row, lane, a.t);
  const bool node = lane < a.t;
  const float gl = node ? a.g[hv0 + (int64_t)lane * a.heads] : 0.f, bl = node ? a.beta[hv0 + (int64_t)lane * a.heads] : 0.f;
  // K and Q, eight values of a node to a thread
  constexpr int kPieces = 2 * N * DKP / 8, kEach = (kPieces + W * kWave - 1) / (W * kWave);
  f32x4_t in[kEach][2];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int p = tid + i * W * kWave, of = p / (N * DKP / 8), n = p / (DKP / 8) % N, d = p % (DKP / 8) * 8;
    in[i][0] = in[i][1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    if (of < 2 && n < a.t && d < DK) {
      const float* const at = (of ? a.q : a.k) + (((int64_t)row * a.t + n) * a.qk_heads + kh) * DK + d;
      in[i][0] = *reinterpret_cast<const f32x4_t*>(at);
      in[i][1] = *reinterpret_cast<const f32x4_t*>(at + 4);
    }
  }
#pragma unroll
  for (int kb = 0; kb < RING; ++kb) load_state(kb);
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int p = tid + i * W * kWave, of = p / (N * DKP / 8), n = p / (DKP / 8) % N, d = p % (DKP / 8) * 8;
    if (kPieces % (W * kWave) && of > 1) continue;
    const Parts4 x = parts_of(in[i][0]), y = parts_of(in[i][1]);
#pragma unroll
    for (int j = 0; j < 3; ++j) *reinterpret_cast<bf16x8_t*>(s.part(of, j, n) + d) = part8(x, y, j);
  }
  // the lane's node, in this wave's head
  auto& mine = s.w[wave];
  // e^-1000 is 0 in fp32, and a finite sum keeps G_s - G_a defined
  double gs = (double)(gl < -1000.f ? -1000.f : gl) * 1.4426950408889634;
  const uint64_t seen = tree_sums(parent, lane, gs);
  if (lane < N) {
    mine.g[lane] = seen ? gs : 0.;
    mine.seen[lane] = seen;
    mine.beta[lane] = seen ? bl : 0.f;
    mine.eg[lane] = seen ? tree_decay(gs) : 0.f;
  }
  __syncthreads();
  const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
  auto piece = [&](int of, int rt, int kb, int p) {  // row 16 rt + c, k index 32 kb + 8 gq + j
    return as_bf16x8(*reinterpret_cast<const u32x4_t*>(s.part(of, p, 16 * rt + c) + 32 * kb + 8 * gq));
  };
  // k . k and q . k of the node pairs, in turn over the waves: rows 16 rt + 4 gq + i, column 16 ct + c
  constexpr int kTiles = NT * (NT + 1), kTurns = (kTiles + W - 1) / W;
  f32x4_t pair[kTurns];
  auto pairs = [&](auto f) {  // (index of this wave's tile, which matrix, row tile, column tile)
    int at = 0;
#pragma unroll
    for (int rt = 0; rt < NT; ++rt)
#pragma unroll
      for (int ct = 0; ct <= rt; ++ct)
#pragma unroll
        for (int of = 0; of < 2; ++of, ++at)
          if (at % W == wave) f(at / W, of, rt, ct);
  };
  auto store_pairs = [&]() {
    pairs([&](int n, int of, int rt, int ct) {
#pragma unroll
      for (int i = 0; i < 4; ++i) (of ? s.pairs().qk : s.pairs().kk)[16 * rt + 4 * gq + i][16 * ct + c] = pair[n][i];
    });
  };
  pairs([&](int n, int of, int rt, int ct) {
    f32x4_t acc[2] = {zero, zero};
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      bf16x8_t x[3], y[3];
#pragma unroll
      for (int p = 0; p < 3; ++p) x[p] = piece(of, rt, kb, p), y[p] = piece(0, ct, kb, p);
#pragma unroll
      for (int p = 0; p < kPartProducts; ++p) acc[kb & 1] = mfma16x16x32(x[left_part(p)], y[right_part(p)], acc[kb & 1]);
    }
    pair[n] = acc[0] + acc[1];
  });
  if (!Lds::OVER) {
    store_pairs();
    __syncthreads();  // kk and qk are whole, and no wave waits for another any more
    if (!on) return;
  }
  // K S and Q S: lane (gq, c) gets rows 4 gq + i of a tile, columns col + e
  f32x4_t ks[NT][4], qs[NT][4];
#pragma unroll
  for (int rt = 0; rt < NT; ++rt)
#pragma unroll
    for (int e = 0; e < 4; ++e) ks[rt][e] = qs[rt][e] = zero;
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    bf16x8_t b[4][3];
    {
      const f32x4_t(&x)[8] = st[kb % RING];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const Parts4 lo = parts_of(f32x4_t{x[0][e], x[1][e], x[2][e], x[3][e]}), hi = parts_of(f32x4_t{x[4][e], x[5][e], x[6][e], x[7][e]});
#pragma unroll
        for (int p = 0; p < 3; ++p) b[e][p] = part8(lo, hi, p);
      }
    }
    if (kb + RING < KB) load_state(kb + RING);
#pragma unroll
    for (int rt = 0; rt < NT; ++rt) {
      bf16x8_t ka[3], qa[3];
#pragma unroll
      for (int p = 0; p < 3; ++p) ka[p] = piece(0, rt, kb, p), qa[p] = piece(1, rt, kb, p);
#pragma unroll
      for (int p = 0; p < kPartProducts; ++p)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          ks[rt][e] = mfma16x16x32(ka[left_part(p)], b[e][right_part(p)], ks[rt][e]);
          qs[rt][e] = mfma16x16x32(qa[left_part(p)], b[e][right_part(p)], qs[rt][e]);
        }
    }
  }
  // v of a tile's nodes, in the products' layout
  f32x4_t vv[2][4];
  auto load_v = [&](int rt) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = 16 * rt + 4 * gq + i;
      vv[rt & 1][i] = zero;
      if (n < a.t && live) vv[rt & 1][i] = *reinterpret_cast<const f32x4_t*>(a.v + (hv0 + (int64_t)n * a.heads) * a.dv + col);
    }
  };
  load_v(0);
  if (Lds::OVER) {
    __syncthreads();  // nobody reads the parts any more
    store_pairs();
    __syncthreads();  // kk and qk are whole
    if (!on) return;
  }
  auto& sq = s.pairs();
  const int own = lane < N ? lane : 0;
  const bool plain = !seen || (sq.kk[own][own] <= 1.01f && gl <= 0.f && bl >= 0.f && bl <= 1.f);
  bool odd = __ballot(!plain) != 0ull;
  // A tile of the two masked matrices, -L and that of out: row 16 rt + c, columns 16 ct + 4 gq + e.
  auto masked = [&](int rt, int ct, f32x4_t& l, f32x4_t& m) {
    const int i = 16 * rt + c, j0 = 16 * ct + 4 * gq;
    const double gi = mine.g[i];
    const float bi = mine.beta[i];
    const f32x4_t kv = *reinterpret_cast<const f32x4_t*>(&sq.kk[i][j0]), qv = *reinterpret_cast<const f32x4_t*>(&sq.qk[i][j0]);
    const uint32_t bits = (uint32_t)(mine.seen[i] >> j0) & 15u;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float d = tree_decay(gi - mine.g[j0 + e]);
      const bool above = (bits >> e & 1u) != 0u;
      l[e] = above && j0 + e != i ? -bi * d * kv[e] : 0.f;
      m[e] = above ? d * qv[e] : 0.f;
    }
  };
  float(*const diag)[Lds::kDBlock] = sq.diag[wave];
  f32x4_t am[NT];
#pragma unroll
  for (int rt = 0; rt < NT; ++rt) {
    f32x4_t l;
    masked(rt, rt, l, am[rt]);
    *reinterpret_cast<f32x4_t*>(&diag[rt][c * Lds::kDRow + 4 * gq]) = l;
  }
  auto own_lds = [&]() {  // the wave reads back only what it wrote
    ring_fence();
    __builtin_amdgcn_s_waitcnt(0xC07F);
    ring_fence();
  };
  own_lds();
  // the diagonal blocks' inverses, side by side: column c of block gq, D[i] = [i == c] + sum over m < i of -L[i][m] D[m]
  {
    const float* const block = diag[gq < NT ? gq : 0];
    float dc[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float acc = c == i ? 1.f : 0.f;
#pragma unroll
      for (int m4 = 0; m4 < (i + 3) / 4; ++m4) {
        const f32x4_t lr = *reinterpret_cast<const f32x4_t*>(&block[i * Lds::kDRow + 4 * m4]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (4 * m4 + e < i) acc = fmaf(lr[e], dc[4 * m4 + e], acc);
      }
      if (i % 4 == 3) asm volatile("" : "+v"(acc) : : "memory");  // or all of the block is read into registers first
      dc[i] = acc;
    }
    own_lds();
    if (gq < NT) {
#pragma unroll
      for (int i = 0; i < 16; ++i) diag[gq][i * Lds::kDRow + c] = dc[i];
    }
    own_lds();
  }
  uint32_t most = 0;  // bits of the largest |u|; infinity and NaN lie above every number
  Parts4 u[NT][4];
#pragma unroll
  for (int rt = 0; rt < NT; ++rt) {
    const int n0 = 16 * rt + 4 * gq;
    const f32x4_t bv = *reinterpret_cast<const f32x4_t*>(&mine.beta[n0]), ev = *reinterpret_cast<const f32x4_t*>(&mine.eg[n0]);
    const f32x4_t inv = *reinterpret_cast<const f32x4_t*>(&diag[rt][c * Lds::kDRow + 4 * gq]);
    bool present[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) present[i] = mine.seen[n0 + i] != 0ull;
    f32x4_t y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        y[e][i] = present[i] ? bv[i] * (vv[rt & 1][i][e] - ev[i] * ks[rt][e][i]) : 0.f;
        qs[rt][e][i] *= ev[i];
      }
    if (rt + 1 < NT) load_v(rt + 1);
    // the earlier tiles, two at a time: element j < 4 of an operand is of the first one's columns, the others of the second one's
#pragma unroll
    for (int ct = 0; ct < rt; ct += 2) {
      f32x4_t l[2] = {zero, zero}, m[2] = {zero, zero};
      masked(rt, ct, l[0], m[0]);
      if (ct + 1 < rt) masked(rt, ct + 1, l[1], m[1]);
      const Parts4 l0 = parts_of(l[0]), l1 = parts_of(l[1]), m0 = parts_of(m[0]), m1 = parts_of(m[1]);
      const Parts4 none = {};
#pragma unroll
      for (int p = 0; p < kPartProducts; ++p)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bf16x8_t x = part8(u[ct][e], ct + 1 < rt ? u[ct + 1][e] : none, right_part(p));
          y[e] = mfma16x16x32(part8(l0, l1, left_part(p)), x, y[e]);
          qs[rt][e] = mfma16x16x32(part8(m0, m1, left_part(p)), x, qs[rt][e]);
        }
    }
    f32x4_t un[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) un[e] = dn_mma(inv, y[e], zero);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      qs[rt][e] = dn_mma(am[rt], un[e], qs[rt][e]);
#pragma unroll
      for (int i = 0; i < 4; ++i) most = max(most, f32_bits(un[e][i]) & 0x7fffffffu);
      if (rt + 1 < NT) u[rt][e] = parts_of(un[e]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = n0 + i;
      if (n < a.t && live)
        *reinterpret_cast<f32x4_t*>(a.out + (hv0 + (int64_t)n * a.heads) * a.dv + col) =
            present[i] ? f32x4_t{qs[rt][0][i], qs[rt][1][i], qs[rt][2][i], qs[rt][3][i]} : zero;
    }
  }
  odd |= __ballot(most >= 0x7f800000u) != 0ull;
  if (odd) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the stores above, before those of the same places
    tree_rule_again<DK, NT, W>(a, s, wave, state, row, kh, head, col - 4 * c + lane);
  }
}

// ---------------------------------------------------------------- the accepted path
//
// The chain's commit (mtpk_deltanet_step.h) over the rows that a path names, and behind its workgroups the
// window's: its last conv_k - 1 columns after the path's. Bound by the states, read and written: 417 MB in 95 us (48 lanes of 64
// heads of 128 x 128, up to 6 rows).
struct DnStepsOnPath {
  const int64_t* path;
  const int64_t* lengths;
  int node = 0;
  __device__ inline int begin(int row, int t) {
    const TreePath p(path + (int64_t)row * t, lengths[row], t, threadIdx.x);
    node = p.node;
    return uniform(p.steps);
  }
  __device__ inline int64_t row(int r, int t, int st) const { return (int64_t)r * t + __builtin_amdgcn_readlane(node, st); }
};

struct PathWindow {
  void* conv;
  int dt;
  const int64_t* slot;
  int64_t slots_total;
  const void* proj;
  int64_t proj_stride;
  const int64_t* path;
  const int64_t* lengths;
  int C, k1, t, per_row;  // per_row: waves of a lane
};

__device__ inline void path_window(const PathWindow& j, int id, int lane) {
  const int b = id / j.per_row, c = (id - b * j.per_row) * kWave + lane;
  const int64_t slot = j.slot[b];
  if (slot < 0 || slot >= j.slots_total) return;  // uniform
  const TreePath path(j.path + (int64_t)b * j.t, j.lengths[b], j.t, lane);
  const int n = uniform(path.steps);
  const bool on = c < j.C;
  const int64_t base = (slot * j.C + (on ? c : 0)) * j.k1;
  float v[kTreeConvMost];
#pragma unroll
  for (int w = 0; w < kTreeConvMost; ++w) {
    if (w >= j.k1) continue;
    const int p = n + w;  // of [the stored window | the path's columns]
    const int at = p < j.k1 ? 0 : path.at(p - j.k1);
    if (on) v[w] = p < j.k1 ? load_float(j.conv, j.dt, base + p) : load_float(j.proj, j.dt, ((int64_t)b * j.t + at) * j.proj_stride + c);
  }
#pragma unroll
  for (int w = 0; w < kTreeConvMost; ++w)
    if (w < j.k1 && on) store_float(j.conv, j.dt, base + w, v[w]);
}

__global__ __launch_bounds__(kWave, 3) void k_path_commit(float* __restrict__ state, int64_t slots_total,
                                                          const int64_t* __restrict__ slot, int t, int heads, int rep, int dv,
                                                          const float* __restrict__ k, const float* __restrict__ v,
                                                          const float* __restrict__ g, const float* __restrict__ beta,
                                                          const int64_t* __restrict__ path, const int64_t* __restrict__ lengths,
                                                          int rule_blocks, PathWindow win) {
  if ((int)blockIdx.x >= rule_blocks) {  // uniform over the one-wave workgroup
    path_window(win, (int)blockIdx.x - rule_blocks, threadIdx.x);
    return;
  }
  delta_rule_kg_body<4, false, true>((int)blockIdx.x, state, slots_total, slot, t, heads, rep, dv, k, k, v, g, beta, nullptr,
                                     DnStepsOnPath{path, lengths});
}

template <int DK>
__global__ __launch_bounds__(kWave) void k_path_commit_any(float* __restrict__ state, int64_t slots_total,
                                                           const int64_t* __restrict__ slot, int t, int heads, int rep, int dv,
                                                           const float* __restrict__ k, const float* __restrict__ v,
                                                           const float* __restrict__ g, const float* __restrict__ beta,
                                                           const int64_t* __restrict__ path, const int64_t* __restrict__ lengths,
                                                           int rule_blocks, PathWindow win) {
  if ((int)blockIdx.x >= rule_blocks) {
    path_window(win, (int)blockIdx.x - rule_blocks, threadIdx.x);
    return;
  }
  delta_rule_body<DK, false, true>((int)blockIdx.x, state, slots_total, slot, t, heads, rep, dv, k, k, v, g, beta, nullptr,
                                   DnStepsOnPath{path, lengths});
}

namespace {

bool tree_rule_shape(int64_t rows, int64_t t, int64_t heads, int64_t qk_heads, int64_t k_dim, int64_t v_dim, int64_t slots_total) {
  return rows >= 0 && t >= 1 && t <= kTreeNodes && heads > 0 && qk_heads > 0 && heads % qk_heads == 0 &&
         (k_dim == 16 || k_dim == 32 || k_dim == 64 || k_dim == 128) && v_dim > 0 && v_dim <= 4096 && slots_total > 0 &&
         heads <= (1 << 20) && slots_total < (int64_t(1) << 40) / (heads * k_dim * v_dim) && rows <= INT32_MAX / heads;
}

template <int DK, int NT, int W>
int tree_rule_waves(const TreeRuleArgs& a, int64_t rows, hipStream_t st) {
  const int64_t grid = rows * a.qk_heads * ((a.rep * a.slabs + W - 1) / W);
  if (grid > 4 * kMaxGroups / W) return MTPK_EINVAL;  // of 64 W threads: fewer than 2^32 in all
  hipLaunchKernelGGL((k_tree_rule<DK, NT, W>), dim3((unsigned)grid), dim3(W * kWave), 0, st, a);
  return status_of(hipGetLastError());
}

// Four waves a workgroup: two lanes of 7 nodes 10.0 us, with eight 13.1; 48 of 16 53.1 / 55.4; 24 of 32 47.5 / 49.5. Above 32 nodes
// LDS holds one workgroup a compute unit, and one of eight waves takes five thirds of the time of one of four (8 lanes of
// 61: 256 of four 30.1, 128 of eight 41.6; 12: 384 of four 55.5, 192 of eight 46.5; 24 of 48: 768 of four 82.9, 384 of eight 94.7).
template <int DK, int NT>
int tree_rule_tiles(const TreeRuleArgs& a, int64_t rows, hipStream_t st) {
  if constexpr (NT > 2) {
    const int64_t units = (int64_t)a.rep * a.slabs, shared = rows * a.qk_heads, cus = device_cu_count();
    auto rounds = [&](int64_t waves) { return (shared * ((units + waves - 1) / waves) + cus - 1) / cus; };
    if (units >= 8 && 5 * rounds(8) < 3 * rounds(4)) return tree_rule_waves<DK, NT, 8>(a, rows, st);
  }
  return tree_rule_waves<DK, NT, 4>(a, rows, st);
}

template <int DK>
int tree_rule_launch(const TreeRuleArgs& a, int64_t rows, hipStream_t st) {
  if (a.t <= 16) return tree_rule_tiles<DK, 1>(a, rows, st);
  if (a.t <= 32) return tree_rule_tiles<DK, 2>(a, rows, st);
  if (a.t <= 48) return tree_rule_tiles<DK, 3>(a, rows, st);
  return tree_rule_tiles<DK, 4>(a, rows, st);
}

}  // namespace
}  // namespace mtpk

using namespace mtpk;

extern "C" {

int mtpk_deltanet_prep_tree(const void* proj, int dtype, int64_t proj_stride, const void* conv_state, const int64_t* slot,
                            int64_t slots_total, const void* conv_w, const float* a_log, const float* dt_bias, const void* parents,
                            int parents_dtype, const int64_t* parents_strides, int64_t batch, int64_t t, int64_t k_heads,
                            int64_t k_dim, int64_t v_heads, int64_t v_dim, int64_t conv_k, float eps, float q_scale, float* q,
                            float* k, float* v, float* g, float* beta, void* stream) {
  if (dtype != MTPK_F32 && dtype != MTPK_BF16) return MTPK_EINVAL;
  if (parents_dtype != MTPK_I32 && parents_dtype != MTPK_I64) return MTPK_EINVAL;
  if (batch < 0 || batch > INT32_MAX || t < 1 || t > kTreeNodes || k_heads < 1 || v_heads < 1 || k_heads > 65535 || v_heads > 65535 ||
      conv_k < 2 || conv_k > kTreeConvMost + 1 || slots_total < 1)
    return MTPK_EINVAL;
  if (k_dim < 1 || k_dim > kTreeHeadMost || v_dim < 1 || v_dim > kTreeHeadMost) return MTPK_EINVAL;
  const int64_t C = 2 * k_heads * k_dim + v_heads * v_dim;
  // a lane's rows are one buffer of less than 2^31 bytes
  if (proj_stride < C + v_heads * v_dim + 2 * v_heads || proj_stride >= (int64_t(1) << 31) / (4 * kTreeNodes)) return MTPK_EINVAL;
  if (batch == 0) return 0;
  if (!proj || !conv_state || !slot || !conv_w || !a_log || !dt_bias || !parents || !parents_strides || !q || !k || !v || !g || !beta)
    return MTPK_EINVAL;
  const TreePrepArgs a{proj, proj_stride, conv_state, slot, slots_total, conv_w, a_log, dt_bias,
                       {parents, parents_dtype, parents_strides[0], parents_strides[1]}, (int)batch, (int)t, (int)k_heads, (int)k_dim,
                       (int)v_heads, (int)v_dim, (int)conv_k, eps, q_scale, q, k, v, g, beta};
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == MTPK_F32) return launch_tree_prep<float, 0, false>(a, st);
  auto at = [](const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
  const bool pair = conv_k == 4 && proj_stride % 2 == 0 && k_dim % 2 == 0 && v_dim % 2 == 0 && at(proj, 4) && at(conv_state, 4) &&
                    at(conv_w, 16) && at(q, 8) && at(k, 8) && at(v, 8);
  return pair ? launch_tree_prep<uint16_t, 4, true>(a, st) : launch_tree_prep<uint16_t, 0, false>(a, st);
}

int mtpk_delta_rule_tree(const float* state, int64_t slots_total, const int64_t* slot, int64_t rows, int64_t t, int64_t heads,
                         int64_t qk_heads, int64_t k_dim, int64_t v_dim, const float* q, const float* k, const float* v,
                         const float* g, const float* beta, const void* parents, int parents_dtype, const int64_t* parents_strides,
                         float* out, void* stream) {
  if (!tree_rule_shape(rows, t, heads, qk_heads, k_dim, v_dim, slots_total) || (!slot && slots_total < rows)) return MTPK_EINVAL;
  if (parents_dtype != MTPK_I32 && parents_dtype != MTPK_I64) return MTPK_EINVAL;
  if (rows == 0) return 0;
  if (!state || !q || !k || !v || !g || !beta || !parents || !parents_strides || !out) return MTPK_EINVAL;
  const TreeParents tree{parents, parents_dtype, parents_strides[0], parents_strides[1]};
  const hipStream_t st = (hipStream_t)stream;
  const int rep = (int)(heads / qk_heads);
  const int64_t slabs = (v_dim + kWave - 1) / kWave, grid = rows * heads * slabs;
  if (grid > 4 * kMaxGroups) return MTPK_EINVAL;  // workgroups of one wave, step by step; all at once they are counted again
  if (v_dim % 4 == 0 && aligned16(state) && aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out)) {
    const TreeRuleArgs a{state, slots_total, slot, (int)t, (int)heads, (int)qk_heads, rep, (int)v_dim, (int)slabs, q, k, v, g, beta, tree, out};
    switch (k_dim) {
      case 16: return tree_rule_launch<16>(a, rows, st);
      case 32: return tree_rule_launch<32>(a, rows, st);
      case 64: return tree_rule_launch<64>(a, rows, st);
      default: return tree_rule_launch<128>(a, rows, st);
    }
  }
#define MTPK_DNT(DK_)                                                                                                       \
  hipLaunchKernelGGL((k_tree_rule_steps<DK_>), dim3((unsigned)grid), dim3(kWave), 0, st, state, slots_total, slot, (int)t,  \
                     (int)heads, rep, (int)v_dim, q, k, v, g, beta, tree, out)
  switch (k_dim) {
    case 16: MTPK_DNT(16); break;
    case 32: MTPK_DNT(32); break;
    case 64: MTPK_DNT(64); break;
    default: MTPK_DNT(128); break;
  }
#undef MTPK_DNT
  return status_of(hipGetLastError());
}

int mtpk_deltanet_commit_path(float* state, int64_t slots_total, const int64_t* slot, int64_t rows, int64_t t, int64_t heads,
                              int64_t qk_heads, int64_t k_dim, int64_t v_dim, const float* k, const float* v, const float* g,
                              const float* beta, const int64_t* path, const int64_t* lengths, void* conv_state, int conv_dtype,
                              int64_t conv_slots_total, const void* proj, int64_t proj_stride, int64_t channels, int64_t k1,
                              void* stream) {
  if (!tree_rule_shape(rows, t, heads, qk_heads, k_dim, v_dim, slots_total)) return MTPK_EINVAL;
  if (conv_dtype != MTPK_F32 && conv_dtype != MTPK_BF16) return MTPK_EINVAL;
  if (channels < 1 || channels > INT32_MAX / 2 || k1 < 1 || k1 > kTreeConvMost || proj_stride < channels || conv_slots_total < 1)
    return MTPK_EINVAL;
  if (rows == 0) return 0;
  if (!state || !slot || !k || !v || !g || !beta || !path || !lengths || !conv_state || !proj) return MTPK_EINVAL;
  const PathWindow win{conv_state, conv_dtype, slot, conv_slots_total, proj, proj_stride, path, lengths, (int)channels, (int)k1,
                       (int)t, (int)((channels + kWave - 1) / kWave)};
  const hipStream_t st = (hipStream_t)stream;
  const int rep = (int)(heads / qk_heads);
  const bool quads = k_dim == 128 && v_dim % kWave == 0 && aligned16(state) && aligned16(v);
  const int64_t rule = rows * heads * ((v_dim + kWave - 1) / kWave), grid = rule + rows * win.per_row;
  if (grid > 4 * kMaxGroups) return MTPK_EINVAL;
#define MTPK_DNP(KERNEL_)                                                                                                    \
  hipLaunchKernelGGL(KERNEL_, dim3((unsigned)grid), dim3(kWave), 0, st, state, slots_total, slot, (int)t, (int)heads, rep,   \
                     (int)v_dim, k, v, g, beta, path, lengths, (int)rule, win)
  if (quads) {
    MTPK_DNP(k_path_commit);
  } else {
    switch (k_dim) {
      case 16: MTPK_DNP(k_path_commit_any<16>); break;
      case 32: MTPK_DNP(k_path_commit_any<32>); break;
      case 64: MTPK_DNP(k_path_commit_any<64>); break;
      default: MTPK_DNP(k_path_commit_any<128>); break;
    }
  }
#undef MTPK_DNP
  return status_of(hipGetLastError());
}

}  // extern "C"
