// The merge of split-KV partials, shared by the decode over contiguous caches
// and the one over pages.
#pragma once
#include "kf_common.hpp"

namespace kf {

// Merge of the split partials: one wave per output row, no LDS and no
// barrier. Lane l = (q = l % QL, sl = l / QL) owns the 4 head-dim columns
// 4q .. 4q + 3 (QL = 16 or 32 lanes cover D / 4 <= QL) of splits sl, sl + SW,
// sl + 2 SW, ... (SW = 64 / QL). Its loads are buffer loads whose
// out-of-range lanes read zero, so no branch separates them and all kMergeU
// of a chunk (O and LSE) are in flight before the first is used: the common
// case (nsplit <= kMergeU * SW) costs one memory round trip. The SW lanes of
// a column then combine with lane swaps (v_permlane16/32_swap).
constexpr int kMergeU = 16;

// A lane's part of a merge: 4 columns and the denominator, in units of
// 2^M, M the largest LSE (log2) it has seen.
struct MergeState {
  f32x4 acc;
  float den, M;
};

// Splits [first, last) of one output row: orr / lrr address split s's O row at
// s * ostride floats and its LSE at s * lstride floats; every offset must fit
// 32 bits (checked by the callers' hosts). All SW lanes of a column end with
// the same state; U of a lane's splits are in flight at once.
template <int QL, int U = kMergeU>
__device__ inline MergeState merge_splits(__amdgpu_buffer_rsrc_t orr, __amdgpu_buffer_rsrc_t lrr,
                                          uint32_t ostride, uint32_t lstride, int first, int last, int D) {
  constexpr int SW = 64 / QL;
  const int lane = threadIdx.x & 63;
  const int q = lane % QL, sl = lane / QL;
  const bool col = 4 * q < D;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  float den = 0.f, mrun = kNegInf;  // running reference max of this lane's chunks (log2 units)
  for (int c0 = first; c0 < last; c0 += U * SW) {
    u32x4 v[U];
    float w[U];
    uint32_t lw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s2 = c0 + sl + SW * u;
      lw[u] = __builtin_amdgcn_raw_buffer_load_b32(lrr, s2 < last ? (uint32_t)s2 * lstride * 4u : kOOB, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s2 = c0 + sl + SW * u;
      v[u] = buf_load16(orr, s2 < last && col ? ((uint32_t)s2 * ostride + 4u * q) * 4u : kOOB);
    }
    // Keep every load of the chunk ahead of the first use: left alone, the
    // scheduler recycles early result registers and waits for them mid-batch.
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < U; ++u)
      w[u] = c0 + sl + SW * u < last ? __uint_as_float(lw[u]) * kLog2e : kNegInf;
    float mx = kNegInf;
#pragma unroll
    for (int u = 0; u < U; ++u) mx = fmaxf(mx, w[u]);
    // Lane-local online rescale across chunks (one chunk in the common case).
    const float mnew = fmaxf(mrun, mx);
    const float ms = mnew == kNegInf ? 0.f : mnew;
    const float alpha = fast_exp2(mrun - ms);
    acc *= alpha;
    den *= alpha;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float wt = fast_exp2(w[u] - ms);
      den += wt;
      acc[0] += wt * __uint_as_float(v[u][0]); acc[1] += wt * __uint_as_float(v[u][1]);
      acc[2] += wt * __uint_as_float(v[u][2]); acc[3] += wt * __uint_as_float(v[u][3]);
    }
    mrun = mnew;
  }
  // Combine the SW split lanes of each column: common reference max, then sums.
  const float M = QL == 16 ? wave_group16_max(mrun) : wave_xor32_max(mrun);
  const float Ms = M == kNegInf ? 0.f : M;
  const float sc = fast_exp2(mrun - Ms);
  float dtot = den * sc;
  dtot = QL == 16 ? wave_group16_sum(dtot) : wave_xor32_sum(dtot);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float x = acc[e] * sc;
    acc[e] = QL == 16 ? wave_group16_sum(x) : wave_xor32_sum(x);
  }
  return {acc, dtot, M};
}

// O and LSE of the row, from the lanes of the first SW. A part whose LSE is NaN
// has a NaN weight (the maximum leaves it out), and so makes den, O and LSE NaN.
template <typename T, int QL>
__device__ inline void merge_store(const MergeState& m, int D, uint16_t* out_row, float* lse_out) {
  const int lane = threadIdx.x & 63;
  const int q = lane % QL;
  if (lane < QL && 4 * q < D) {
    const float inv = m.den == 0.f ? 0.f : 1.f / m.den;
    u32x2 wv;
    wv[0] = pack2<T>(m.acc[0] * inv, m.acc[1] * inv);
    wv[1] = pack2<T>(m.acc[2] * inv, m.acc[3] * inv);
    *reinterpret_cast<u32x2*>(out_row + 4 * q) = wv;
    if (q == 0 && lse_out) *lse_out = m.den == 0.f ? kNegInf : (m.M + fast_log2(m.den)) * kLn2;
  }
}

template <typename T, int QL, int U = kMergeU>
__device__ inline void merge_row(__amdgpu_buffer_rsrc_t orr, __amdgpu_buffer_rsrc_t lrr,
                                 uint32_t ostride, uint32_t lstride, int nsplit, int D,
                                 uint16_t* out_row, float* lse_out) {
  merge_store<T, QL>(merge_splits<QL, U>(orr, lrr, ostride, lstride, 0, nsplit, D), D, out_row, lse_out);
}

}  // namespace kf
