// Rotary positions: queries and keys turned pair by pair, gfx950. No
// counterpart in the reference, whose models bring none.
//
// Pair i of the first R dims of a head, (x, y), at the token's position n:
//   (x cos a - y sin a, x sin a + y cos a) amplitude,  a = n f_i,
// pairs (i, i + R/2), or (2i, 2i + 1) when interleaved; the other dims pass
// as they are. `inverse` turns by -a: with the same amplitude that is the
// transpose, so the gradient's kernel too.
//
// Angles. f_i / 2 pi comes as a 64-bit fraction of a turn, F_i / 2^64, rounded
// to the nearest. n F_i mod 2^64 is then the angle's fraction of a turn with an
// error of n / 2^65, negative n too; its top 32 bits are kept (2^-32 of a turn;
// the table's error reaches that at n = 2^33, and 2^-22 rad at 2^40).
// In fp32 the product n f_i alone would be off by 0.03 rad at n = 10^6. The
// nearest quarter turn leaves |x| <= pi / 4 for Taylor polynomials in fp32:
// sin to x^9 (next term 2e-9), cos to x^8 (3e-8).
//
// HBM-bound: every element is read and written once. What the angles cost, about
// 35 vector instructions per pair, is shared by all heads of a token that a
// wave takes. 671 MB (40 heads of 128, 32768 tokens, bf16) 119 us, 5.6 TB/s; a large
// copy reaches 5.1 to 5.5. Loads or stores marked as read once: level.
#include "kf_common.hpp"
#include "kf_host.hpp"

namespace kf {

struct RotaryTensor {
  const uint16_t* x;
  uint16_t* y;
  int64_t x_sb, x_sh, x_ss, x_sd;
  int64_t y_sb, y_sh, y_ss, y_sd;
};

struct RotaryParams {
  RotaryTensor t[2];         // queries, keys
  const uint64_t* turns;     // [R / 2]
  const void* positions;     // null: `first`
  int64_t first, p_sb, p_ss;
  int wide;                  // positions are 64-bit
  int step;                  // 1: a position is that of the request's first token
  int64_t S;
  int64_t tokens;            // B * S
  int Hq, H;                 // query heads, all heads
  int D, R;
  int lanes;                 // of a row: each takes two 16-byte pieces
  int rows;                  // rows (heads) that a wave takes at once
  int groups;                // waves of a token
  float amplitude, sign;
};

__device__ inline int64_t rotary_position(const RotaryParams& p, int64_t b, int64_t s) {
  int64_t n = p.first;
  if (p.positions) {
    const int64_t at = b * p.p_sb + s * p.p_ss;
    n = p.wide ? ((const int64_t*)p.positions)[at] : ((const int32_t*)p.positions)[at];
  }
  return p.step ? n + s : n;
}

// sin and cos of n F / 2^64 turns.
__device__ inline void turn_sincos(int64_t n, uint64_t F, float& s, float& c) {
  const uint32_t phase = (uint32_t)(((uint64_t)n * F) >> 32);
  const uint32_t quarter = (phase + 0x20000000u) >> 30;
  const float x = (float)(int32_t)(phase - (quarter << 30)) * 1.46291807926715968e-9f;  // 2 pi / 2^32
  const float z = x * x;
  float ps = 2.7557319223985893e-6f, pc = 2.4801587301587302e-5f;  // 1/9!, 1/8!
  ps = fmaf(ps, z, -1.9841269841269841e-4f);
  pc = fmaf(pc, z, -1.3888888888888889e-3f);
  ps = fmaf(ps, z, 8.3333333333333333e-3f);
  pc = fmaf(pc, z, 4.1666666666666667e-2f);
  ps = fmaf(ps, z, -1.6666666666666667e-1f);
  pc = fmaf(pc, z, -0.5f);
  const float si = fmaf(ps * z, x, x), co = fmaf(pc, z, 1.f);
  const float a = quarter & 1 ? co : si, b = quarter & 1 ? si : co;
  s = quarter & 2 ? -a : a;
  c = (quarter + 1) & 2 ? -b : b;
}

// A wave per token and group of PASSES * rows heads. A lane holds two pieces of
// eight elements of a row: of the halves' places (x of eight pairs, y of the
// same), of 16 neighbours when interleaved, or of 16 that pass.
template <typename T, bool INTERLEAVED, int PASSES>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t w = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 4 + wave_index();
  const int64_t token = w / p.groups;
  if (token >= p.tokens) return;
  const int group = (int)(w - token * p.groups);
  const int64_t b = token / p.S, s = token - b * p.S;
  const int row = lane / p.lanes, j = lane - row * p.lanes;
  const int turning = p.R / 16;
  const bool turns = j < turning;
  int d0, d1;
  if (turns) {
    d0 = INTERLEAVED ? 16 * j : 8 * j;
    d1 = INTERLEAVED ? 16 * j + 8 : p.R / 2 + 8 * j;
  } else {
    d0 = p.R + 16 * (j - turning);
    d1 = d0 + 8;
  }
  const bool second = d1 < p.D;

  u32x4 x0[PASSES], x1[PASSES];
  uint16_t* to[PASSES];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int h = (group * PASSES + i) * p.rows + row;
    to[i] = nullptr;
    if (row < p.rows && h < p.H) {
      const RotaryTensor& t = p.t[h >= p.Hq];
      const int hh = h >= p.Hq ? h - p.Hq : h;
      const uint16_t* from = t.x + b * t.x_sb + hh * t.x_sh + s * t.x_ss;
      to[i] = t.y + b * t.y_sb + hh * t.y_sh + s * t.y_ss;
      x0[i] = ldg16(from + d0);
      if (second) x1[i] = ldg16(from + d1);
    }
  }
  float sn[8], cs[8];
  if (turns) {
    const int64_t n = rotary_position(p, b, s);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      turn_sincos(n, p.turns[8 * j + e], sn[e], cs[e]);
      sn[e] *= p.amplitude * p.sign;
      cs[e] *= p.amplitude;
    }
  }
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    if (!to[i]) continue;
    if (turns) {
      uint32_t* a = (uint32_t*)&x0[i];
      uint32_t* c = (uint32_t*)&x1[i];
      auto low = [](uint32_t v) { return Elem<T>::to_f32((uint16_t)v); };
      auto high = [](uint32_t v) { return Elem<T>::to_f32((uint16_t)(v >> 16)); };
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (INTERLEAVED) {
          uint32_t& v = e < 4 ? a[e] : c[e - 4];
          const float x = low(v), y = high(v);
          v = pack2<T>(x * cs[e] - y * sn[e], x * sn[e] + y * cs[e]);
        } else if (e % 2 == 0) {
          const uint32_t vx = a[e / 2], vy = c[e / 2];
          const float xl = low(vx), yl = low(vy), xh = high(vx), yh = high(vy);
          a[e / 2] = pack2<T>(xl * cs[e] - yl * sn[e], xh * cs[e + 1] - yh * sn[e + 1]);
          c[e / 2] = pack2<T>(xl * sn[e] + yl * cs[e], xh * sn[e + 1] + yh * cs[e + 1]);
        }
      }
    }
    stg16(to[i] + d0, x0[i]);
    if (second) stg16(to[i] + d1, x1[i]);
  }
}

// Any strides and any even R: a thread per pair, or element that passes. Bound
// by instructions (64-bit divisions, an angle per head) and 2-byte accesses, at a
// quarter to a seventh of a copy's rate: 40 heads, 32768 tokens, D = R = 72 285
// us (a copy 71), 40 166 (40), R = 56 of D = 112 665 (109).
template <typename T>
__global__ __launch_bounds__(256) void rotary_plain_kernel(const RotaryParams p, int interleaved) {
  const int half = p.R / 2, items = half + p.D - p.R;
  const int64_t all = p.tokens * p.H * items;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / items;
    const int j = (int)(i - r * items);
    const int64_t token = r / p.H, b = token / p.S, s = token - b * p.S;
    const int h = (int)(r - token * p.H);
    const RotaryTensor& t = p.t[h >= p.Hq];
    const int hh = h >= p.Hq ? h - p.Hq : h;
    const uint16_t* from = t.x + b * t.x_sb + hh * t.x_sh + s * t.x_ss;
    uint16_t* to = t.y + b * t.y_sb + hh * t.y_sh + s * t.y_ss;
    if (j >= half) {
      const int d = p.R + j - half;
      to[d * t.y_sd] = from[d * t.x_sd];
      continue;
    }
    const int d0 = interleaved ? 2 * j : j, d1 = interleaved ? 2 * j + 1 : j + half;
    float sn, cs;
    turn_sincos(rotary_position(p, b, s), p.turns[j], sn, cs);
    sn *= p.amplitude * p.sign;
    cs *= p.amplitude;
    const float x = Elem<T>::to_f32(from[d0 * t.x_sd]), y = Elem<T>::to_f32(from[d1 * t.x_sd]);
    to[d0 * t.y_sd] = Elem<T>::bits(x * cs - y * sn);
    to[d1 * t.y_sd] = Elem<T>::bits(x * sn + y * cs);
  }
}

// Waves, with one pass of heads each, from which a wave takes up to four passes
// and shares the token's angles among them; fewer waves are better spread out.
// 40 heads of 128 (five passes), us with one pass and with three: 256 tokens 3.7
// and 4.1, 512 4.6 and 4.5, 1024 6.6 and 5.9, 4096 16.7 and 15.4.
constexpr int64_t kRotaryWaves = 2048;

template <typename T, bool INTERLEAVED>
static void launch_rotary(RotaryParams& p, hipStream_t stream) {
  const int passes = cdiv(p.H, p.rows);
  int each = 1;
  if (p.tokens * passes >= kRotaryWaves) {
    p.groups = cdiv(passes, 4);
    each = cdiv(passes, p.groups);
  } else {
    p.groups = passes;
  }
  // HIP counts the threads of one dimension of a grid in 32 bits.
  const int64_t blocks = (p.tokens * p.groups + 3) / 4, wide = 1 << 23;
  const dim3 grid((unsigned)(blocks < wide ? blocks : wide), (unsigned)((blocks + wide - 1) / wide)), block(256);
  switch (each) {
    case 1: hipLaunchKernelGGL((rotary_kernel<T, INTERLEAVED, 1>), grid, block, 0, stream, p); break;
    case 2: hipLaunchKernelGGL((rotary_kernel<T, INTERLEAVED, 2>), grid, block, 0, stream, p); break;
    case 3: hipLaunchKernelGGL((rotary_kernel<T, INTERLEAVED, 3>), grid, block, 0, stream, p); break;
    default: hipLaunchKernelGGL((rotary_kernel<T, INTERLEAVED, 4>), grid, block, 0, stream, p); break;
  }
}

}  // namespace kf

using namespace kf;

extern "C" int kf_rotary(const void* q, const void* k, void* q_out, void* k_out, const int64_t* turns,
                         const void* positions, int wide, int64_t first, int step, int64_t B, int64_t Hq,
                         int64_t Hk, int64_t S, int64_t D, int64_t R, const int64_t* q_strides4,
                         const int64_t* k_strides4, const int64_t* q_out_strides4, const int64_t* k_out_strides4,
                         const int64_t* position_strides2, float amplitude, int interleaved, int inverse, int dtype,
                         void* stream) {
  const char* what = "kf_rotary";
  if (!q || !q_out || !turns || (Hk > 0 && (!k || !k_out))) return set_error(KF_EINVAL, "%s: null pointer", what);
  if (!q_strides4 || !q_out_strides4 || (Hk > 0 && (!k_strides4 || !k_out_strides4)) || (positions && !position_strides2))
    return set_error(KF_EINVAL, "%s: null strides", what);
  if (B <= 0 || Hq <= 0 || Hk < 0 || S <= 0 || D <= 0) return set_error(KF_EINVAL, "%s: all sizes must be positive", what);
  if (R <= 0 || R > D || R % 2) return set_error(KF_EINVAL, "%s: the dims that turn must be even and at most D", what);
  if (dtype != KF_F16 && dtype != KF_BF16) return set_error(KF_EINVAL, "%s: dtype must be KF_F16 or KF_BF16", what);
  if (!(amplitude - amplitude == 0.f)) return set_error(KF_EINVAL, "%s: amplitude must be finite", what);
  if (D > 65536 || Hq > (1 << 20) || Hk > (1 << 20) || S > 0x7fffffff || B > 0x7fffffff / S ||
      B * S > 0x7fffffff / (Hq + Hk))
    return set_error(KF_EUNSUPPORTED, "%s: dimension too large", what);
  RotaryParams p{};
  const void* x[2] = {q, k};
  void* y[2] = {q_out, k_out};
  const int64_t *xs[2] = {q_strides4, k_strides4}, *ys[2] = {q_out_strides4, k_out_strides4};
  bool vec = R % 16 == 0 && D % 8 == 0 && D <= 1024;
  for (int i = 0; i < (Hk > 0 ? 2 : 1); ++i) {
    p.t[i] = {(const uint16_t*)x[i], (uint16_t*)y[i], xs[i][0], xs[i][1], xs[i][2], xs[i][3],
              ys[i][0], ys[i][1], ys[i][2], ys[i][3]};
    vec = vec && aligned16(x[i]) && aligned16(y[i]) && xs[i][3] == 1 && ys[i][3] == 1;
    for (int j = 0; j < 3; ++j) vec = vec && xs[i][j] % 8 == 0 && ys[i][j] % 8 == 0;
  }
  p.turns = (const uint64_t*)turns;
  p.positions = positions;
  p.wide = wide != 0;
  p.step = step != 0;
  p.first = first;
  if (positions) { p.p_sb = position_strides2[0]; p.p_ss = position_strides2[1]; }
  p.S = S; p.tokens = B * S;
  p.Hq = (int)Hq; p.H = (int)(Hq + Hk); p.D = (int)D; p.R = (int)R;
  p.amplitude = amplitude;
  p.sign = inverse ? -1.f : 1.f;
  hipStream_t st = (hipStream_t)stream;
  if (vec) {
    p.lanes = (int)(R / 16 + (D - R + 15) / 16);
    p.rows = 64 / p.lanes;
    if (dtype == KF_F16) interleaved ? launch_rotary<_Float16, true>(p, st) : launch_rotary<_Float16, false>(p, st);
    else interleaved ? launch_rotary<__bf16, true>(p, st) : launch_rotary<__bf16, false>(p, st);
    return check_launch(what);
  }
  const int64_t all = p.tokens * p.H * (R / 2 + D - R), blocks = (all + 255) / 256;
  const dim3 grid((unsigned)(blocks < 65536 ? blocks : 65536));
  if (dtype == KF_F16) hipLaunchKernelGGL(rotary_plain_kernel<_Float16>, grid, dim3(256), 0, st, p, interleaved);
  else hipLaunchKernelGGL(rotary_plain_kernel<__bf16>, grid, dim3(256), 0, st, p, interleaved);
  return check_launch(what);
}
