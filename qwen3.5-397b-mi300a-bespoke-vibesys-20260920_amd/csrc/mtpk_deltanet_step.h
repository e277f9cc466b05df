// The gated delta rule step by step (mtpk_deltanet.hip), as a body of its launches over a call's rows and along
// paths of a tree (mtpk_deltanet_tree.hip). `Steps` says which steps a row runs and where their inputs lie.
#pragma once

#include "mtpk_deltanet_chunk.h"
#include "mtpk_device.h"

namespace mtpk {

// The first steps of the row, all of them without `lengths`.
struct DnStepsInOrder {
  const int64_t* lengths;
  int t0;  // of a piece's first step
  __device__ inline int begin(int row, int t) const { return dn_steps(lengths, row, t, t0); }
  __device__ inline int64_t row(int r, int t, int st) const { return (int64_t)r * t + st; }
};

template <int DK, bool OUT, bool COMMIT, typename Steps>
__device__ __forceinline__ void delta_rule_body(
    int bid, float* __restrict__ state, int64_t slots_total, const int64_t* __restrict__ slot, int t,
    int heads, int rep, int dv, const float* __restrict__ q, const float* __restrict__ k, const float* __restrict__ v,
    const float* __restrict__ g, const float* __restrict__ beta, float* __restrict__ out, Steps steps) {
  static_assert(DK % 4 == 0, "k and q are read back four values at a time");
  // Workgroup (bh, c) is id `bid` = bh * nblk + c: the column blocks of one matrix are dispatched
  // together, so the matrix's rows are read whole (its 64-column blocks interleave every
  // 256 bytes) while they are still open in the memory's row buffers.
  const int nblk = (dv + kWave - 1) / kWave;
  const int bh = bid / nblk;  // row * heads + head
  const int row = bh / heads, head = bh - row * heads;
  const int col = (bid - bh * nblk) * kWave + threadIdx.x;
  const bool live = col < dv;
  const int64_t s_idx = slot ? slot[row] : row;
  if (s_idx < 0 || s_idx >= slots_total) {  // no such slot: zero outputs, no state access
    if (OUT && live)
      for (int st = 0; st < t; ++st) out[((int64_t)row * t + st) * heads * dv + (int64_t)head * dv + col] = 0.f;
    return;  // uniform over the one-wave workgroup
  }
  // the (slot, head) matrix as one buffer: element (i, col) at byte 4 col + 4 dv i, the
  // per-lane part in voffset (out of range for lanes past dv) and the row offset in soffset
  const rsrc_t rsm = make_rsrc(state + ((s_idx * heads + head) * DK) * (int64_t)dv,
                               (uint32_t)(DK * dv * 4));
  const uint32_t vcol = live ? (uint32_t)col * 4u : kOutOfRange, drow = (uint32_t)dv * 4u;
  float s[DK];
#pragma unroll
  for (int i = 0; i < DK; ++i)
    s[i] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rsm, (int)vcol, (int)(drow * i), 0));
  const int n = steps.begin(row, t);
  const int qk_heads = heads / rep, kh = head / rep;
  // A step's k and q (the same for the whole wave) pass through LDS: each lane loads one or two
  // of their values, and the product loops read them back four at a time as broadcasts. Step
  // st + 1's k, q, v, g and beta are loaded while step st runs, so no step waits for its
  // inputs after the first.
  constexpr int kPer = (DK + kWave - 1) / kWave;
  __shared__ __attribute__((aligned(16))) float kq[2][2][DK];
  const int lane = threadIdx.x;
  float nk[kPer], nq[kPer], nv = 0.f, ng = 0.f, nbt = 0.f;
  auto step_load = [&](int st) {
    const int64_t rs = steps.row(row, t, st < n ? st : 0);
    const int64_t qk_off = (rs * qk_heads + kh) * DK, hv = rs * heads + head;
#pragma unroll
    for (int p = 0; p < kPer; ++p) {
      const int i = p * kWave + lane;
      nk[p] = i < DK ? k[qk_off + i] : 0.f;
      nq[p] = OUT && i < DK ? q[qk_off + i] : 0.f;
    }
    nv = live ? v[hv * dv + col] : 0.f;
    ng = g[hv];
    nbt = beta[hv];
  };
  if (n > 0) step_load(0);
  for (int st = 0; st < n; ++st) {
    const int b = st & 1;
#pragma unroll
    for (int p = 0; p < kPer; ++p) {
      const int i = p * kWave + lane;
      if (i < DK) {
        kq[b][0][i] = nk[p];
        if (OUT) kq[b][1][i] = nq[p];
      }
    }
    const float decay = __expf(ng), bt = nbt, vv = nv;
    __syncthreads();  // this step's k and q are in LDS (a one-wave workgroup)
    if (st + 1 < n) step_load(st + 1);
    const float4* kk = reinterpret_cast<const float4*>(kq[b][0]);
    const float4* qq = reinterpret_cast<const float4*>(kq[b][1]);
    float mem = 0.f;
#pragma unroll
    for (int i4 = 0; i4 < DK / 4; ++i4) {
      const float4 kv = kk[i4];
      s[4 * i4] *= decay;
      s[4 * i4 + 1] *= decay;
      s[4 * i4 + 2] *= decay;
      s[4 * i4 + 3] *= decay;
      mem = fmaf(s[4 * i4], kv.x, mem);
      mem = fmaf(s[4 * i4 + 1], kv.y, mem);
      mem = fmaf(s[4 * i4 + 2], kv.z, mem);
      mem = fmaf(s[4 * i4 + 3], kv.w, mem);
    }
    const float delta = (vv - mem) * bt;
    // read k again rather than keep all DK values live across both loops: the state already
    // takes DK registers
    asm volatile("" ::: "memory");
    float o = 0.f;
#pragma unroll
    for (int i4 = 0; i4 < DK / 4; ++i4) {
      const float4 kv = kk[i4];
      s[4 * i4] = fmaf(kv.x, delta, s[4 * i4]);
      s[4 * i4 + 1] = fmaf(kv.y, delta, s[4 * i4 + 1]);
      s[4 * i4 + 2] = fmaf(kv.z, delta, s[4 * i4 + 2]);
      s[4 * i4 + 3] = fmaf(kv.w, delta, s[4 * i4 + 3]);
      if (OUT) {
        const float4 qv = qq[i4];
        o = fmaf(s[4 * i4], qv.x, o);
        o = fmaf(s[4 * i4 + 1], qv.y, o);
        o = fmaf(s[4 * i4 + 2], qv.z, o);
        o = fmaf(s[4 * i4 + 3], qv.w, o);
      }
    }
    if (OUT && live) out[((int64_t)row * t + st) * heads * dv + (int64_t)head * dv + col] = o;
  }
  if (COMMIT) {
#pragma unroll
    for (int i = 0; i < DK; ++i)
      __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, s[i]), rsm, (int)vcol,
                                            (int)(drow * i), 0);
  }
}

// The k_dim = 128 form (dv a multiple of 64): the rows of a matrix are cut into KG groups of
// 128 / KG and lane (cg = l / KG, kg = l % KG) owns the 4 adjacent columns 4 cg .. 4 cg + 3 of
// its block (64 4 / KG columns) over row group kg, so the state comes in with 16-byte loads
// (128 / KG per lane; every wave instruction reads KG row segments of 16 columns each) instead
// of 128 dword loads, and each step reads only its row group of k and q back from LDS. A
// column's sums over the row groups (S^T k and S^T q) are DPP butterfly adds inside the KG
// adjacent lanes, which leave the same bits in all of them, so every lane applies the same
// delta to its rows. The first 4 lanes of each group write the group's 4 output columns.
template <int CTRL>
__device__ inline float dn_dpp(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CTRL, 0xf, 0xf, false));
}
template <int KG>
__device__ inline float group_sum(float x) {
  x += dn_dpp<0xB1>(x);  // quad_perm [1, 0, 3, 2]
  x += dn_dpp<0x4E>(x);  // quad_perm [2, 3, 0, 1]
  if (KG == 8) x += dn_dpp<0x141>(x);  // row_half_mirror: the other quad of the 8 lanes
  return x;
}

// `left`, where not null, has a word for each 32 columns of the (row, head) matrices: only those with
// a nonzero one are written.
template <int KG, bool OUT, bool COMMIT, typename Steps>
__device__ __forceinline__ void delta_rule_kg_body(
    int bid, float* __restrict__ state, int64_t slots_total, const int64_t* __restrict__ slot, int t,
    int heads, int rep, int dv, const float* __restrict__ q, const float* __restrict__ k,
    const float* __restrict__ v, const float* __restrict__ g, const float* __restrict__ beta,
    float* __restrict__ out, Steps steps, DnPiece piece = {0, nullptr},
    const int32_t* left = nullptr) {
  static_assert(KG == 4 || KG == 8, "row groups of 32 or 16");
  constexpr int DK = 128, QR = DK / KG, CW = 4 * kWave / KG;  // rows per group, columns per wave
  const int nblk = dv / CW;
  const int bh = bid / nblk;  // row * heads + head; a matrix's blocks are adjacent ids
  const int row = bh / heads, head = bh - row * heads;
  const int lane = threadIdx.x, cg = lane / KG, kg = lane % KG;
  const int base = (bid - bh * nblk) * CW;  // the block's first column
  const int col4 = base + 4 * cg;                   // this lane's first state column
  const int64_t s_idx = slot ? slot[row] : row;
  const int64_t o_row = (int64_t)head * dv + col4 + kg;  // kg < 4: the output column it writes
  const bool writes = !left || left[(int64_t)bh * (dv / kDnScanCols) + col4 / kDnScanCols] != 0;
  if (s_idx < 0 || s_idx >= slots_total) {  // no such slot: zero outputs, no state access
    if (OUT && kg < 4)
      for (int st = 0; st < t; ++st) out[((int64_t)row * t + st) * heads * dv + o_row] = 0.f;
    return;  // uniform over the one-wave workgroup
  }
  float* const pool = state + ((s_idx * heads + head) * DK) * (int64_t)dv;
  float* const kept = piece.carry ? piece.carry + (int64_t)head * DK * dv : pool;  // one row
  const rsrc_t rsm = make_rsrc(kept, (uint32_t)(DK * dv * 4));
  const rsrc_t rsi = make_rsrc(piece.t0 > 0 ? kept : pool, (uint32_t)(DK * dv * 4));
  const uint32_t voff = ((uint32_t)(QR * kg) * (uint32_t)dv + (uint32_t)col4) * 4u, drow = (uint32_t)dv * 4u;
  f32x4_t s[QR];  // s[i] = row QR kg + i, columns col4 .. col4 + 3
#pragma unroll
  for (int i = 0; i < QR; ++i) s[i] = __builtin_bit_cast(f32x4_t, buf16(rsi, voff, drow * (uint32_t)i));
  const int n = steps.begin(row, t);
  const int qk_heads = heads / rep, kh = head / rep;
  // k and q pass through LDS as in the general form; step st + 1's inputs load while step st runs
  __shared__ __attribute__((aligned(16))) float kq[2][2][DK];
  float nk[2], nq[2], ng = 0.f, nbt = 0.f;
  f32x4_t nv = {0.f, 0.f, 0.f, 0.f};
  auto step_load = [&](int st) {
    const int64_t rs = steps.row(row, t, st < n ? st : 0);
    const int64_t qk_off = (rs * qk_heads + kh) * DK, hv = rs * heads + head;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      nk[p] = k[qk_off + p * kWave + lane];
      nq[p] = OUT ? q[qk_off + p * kWave + lane] : 0.f;
    }
    nv = *reinterpret_cast<const f32x4_t*>(v + hv * dv + col4);
    ng = g[hv];
    nbt = beta[hv];
  };
  if (n > 0) step_load(0);
  for (int st = 0; st < n; ++st) {
    const int b = st & 1;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      kq[b][0][p * kWave + lane] = nk[p];
      if (OUT) kq[b][1][p * kWave + lane] = nq[p];
    }
    const float decay = __expf(ng), bt = nbt;
    const f32x4_t vv = nv;
    __syncthreads();  // this step's k and q are in LDS (a one-wave workgroup)
    if (st + 1 < n) step_load(st + 1);
    const float4* kk = reinterpret_cast<const float4*>(&kq[b][0][QR * kg]);
    const float4* qq = reinterpret_cast<const float4*>(&kq[b][1][QR * kg]);
    float m[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i4 = 0; i4 < QR / 4; ++i4) {
      const float4 kv = kk[i4];
      const float kr[4] = {kv.x, kv.y, kv.z, kv.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = 4 * i4 + e;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          s[i][c] *= decay;
          m[c] = fmaf(s[i][c], kr[e], m[c]);
        }
      }
    }
    float delta[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) delta[c] = (vv[c] - group_sum<KG>(m[c])) * bt;
    asm volatile("" ::: "memory");
    float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i4 = 0; i4 < QR / 4; ++i4) {
      const float4 kv = kk[i4];
      const float kr[4] = {kv.x, kv.y, kv.z, kv.w};
      float qr[4] = {0.f, 0.f, 0.f, 0.f};
      if (OUT) {
        const float4 qv = qq[i4];
        qr[0] = qv.x;
        qr[1] = qv.y;
        qr[2] = qv.z;
        qr[3] = qv.w;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = 4 * i4 + e;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          s[i][c] = fmaf(kr[e], delta[c], s[i][c]);
          if (OUT) o[c] = fmaf(s[i][c], qr[e], o[c]);
        }
      }
    }
    if (OUT) {
      float mine = 0.f;  // column col4 + kg (kg < 4), by selects (no indexed registers)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float sum = group_sum<KG>(o[c]);
        if (kg == c) mine = sum;
      }
      if (kg < 4 && writes) out[((int64_t)row * t + st) * heads * dv + o_row] = mine;
    }
  }
  if (COMMIT && writes) {
#pragma unroll
    for (int i = 0; i < QR; ++i)
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, s[i]), rsm, (int)voff,
                                             (int)(drow * (uint32_t)i), 0);
  }
}

}  // namespace mtpk
