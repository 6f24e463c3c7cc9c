// Rows of a paged K/V cache in 8 bits: the store, which quantises, and the
// read back into 16 bits. gfx950. No counterpart in the reference, whose cache
// holds what it is given (kotflash/cache.py:91-290).
//
// Pools of e4m3 codes (4 significant bits, largest 448, smallest step 2^-9),
// laid out as the 16-bit ones. 16 positions of a page, one head, are a block;
// scales [pages, H, page / 16, 2] holds its scale for K and for V, and a value is
// code * scale. Scales are powers of two: x / scale and code * scale are exact,
// so a value is rounded once, and a block whose scale grows loses nothing but
// below its smallest normal code.
//
// store: s = least power of two >= 2^-126 with |x| <= 448 s for all finite x of
// the rows that come into a block. Rows of a request follow one another, so the
// block is new if its row 0 is among them: its scale is s. Else it is max(s, the
// scale it has), and where that is more the block's other rows are divided by
// the ratio. Infinities become NaN, which is all that e4m3 has; a code that
// would stand for 2^16 in fp16 (2^128 in bf16) is one step smaller.
#include "fp8.hpp"
#include "kf_host.hpp"

namespace kf {

struct Fp8StoreParams {
  uint8_t* kp;
  uint8_t* vp;
  float* scales;
  const uint16_t* nk;
  const uint16_t* nv;
  const int64_t* slots;
  int64_t s_sb;
  int64_t kp_sp, kp_sh, kp_ss;
  int64_t vp_sp, vp_sh, vp_ss;
  int64_t sc_sp, sc_sh;
  int64_t nk_sb, nk_sh, nk_ss;
  int64_t nv_sb, nv_sh, nv_ss;
  int64_t places;   // slots of the pool
  int waves;
  int n;
  Divisor heads, windows, blocks;  // windows of 16 new tokens of a request; blocks of a page
  int lanes, rows;                 // lanes of a row, rows that a wave loads at once
};

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

__device__ inline uint32_t pk_max(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
// Both 16-bit halves' maxima over the wave, in every lane.
__device__ inline uint32_t wave_pk_max(uint32_t x) {
  x = pk_max(x, __builtin_amdgcn_update_dpp(0, x, 0x128, 0xf, 0xf, false));  // rotations in rows of 16
  x = pk_max(x, __builtin_amdgcn_update_dpp(0, x, 0x124, 0xf, 0xf, false));
  x = pk_max(x, __builtin_amdgcn_update_dpp(0, x, 0x122, 0xf, 0xf, false));
  x = pk_max(x, __builtin_amdgcn_update_dpp(0, x, 0x121, 0xf, 0xf, false));
  auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = pk_max(r[0], r[1]);
  r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return pk_max(r[0], r[1]);
}

template <typename T> struct HalfBits;
template <> struct HalfBits<_Float16> { static constexpr uint32_t exp = 0x7c00u; static constexpr int top = 16; };
template <> struct HalfBits<__bf16> { static constexpr uint32_t exp = 0x7f80u; static constexpr int top = 128; };

// Biased exponent of the scale for magnitudes up to a: with a = m 2^e, 448 =
// 1.75 2^8, that is e - 8, or e - 7 for m > 1.75.
__device__ inline int scale_exponent(float a) {
  const int e = (int)((__float_as_uint(a) + 0x1fffffu) >> 23) - 8;
  return e < 1 ? 1 : e;
}
__device__ inline float power(int biased) { return __uint_as_float((uint32_t)biased << 23); }

// Eight elements over a scale (by its inverse) as codes. `special`: some may
// not be finite, or reach the largest that the type holds of this scale.
template <typename T>
__device__ inline u32x2 quantise(u32x4 x, float inv, float limit, bool special) {
  float y[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    y[2 * j] = Elem<T>::to_f32((uint16_t)x[j]) * inv;
    y[2 * j + 1] = Elem<T>::to_f32((uint16_t)(x[j] >> 16)) * inv;
  }
  if (special) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t bits = j & 1 ? x[j / 2] >> 16 : x[j / 2];
      const float c = fminf(fmaxf(y[j], -limit), limit);
      y[j] = (bits & HalfBits<T>::exp) == HalfBits<T>::exp ? __builtin_nanf("") : c;
    }
  }
  u32x2 out;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * j], y[4 * j + 1], 0, false);
    out[j] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * j + 2], y[4 * j + 3], w, true);
  }
  return out;
}

// Eight codes times a power of two.
__device__ inline u32x2 rescale(u32x2 x, float ratio) {
  u32x2 out;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)x[j], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)x[j], true);
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(a[0] * ratio, a[1] * ratio, 0, false);
    out[j] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(b[0] * ratio, b[1] * ratio, w, true);
  }
  return out;
}

// Bytes of new keys and values from which the codes' stores are marked as not
// read again soon (us, plain and marked: 17 MB of them 6.5 and 6.1, 33 MB 8.9
// and 7.9, 134 MB 21.3 and 19.9, 268 MB 45.1 and 39.2; marked loads 40.4, both
// 42.1). A step's rows are read next.
constexpr int64_t kStreamRows = 16 << 20;

// One run: the rows kx and vx of a wave (lane's piece at element d of each), to
// places place[] of block blk, head h; -1: none. begins: row 0 is among them.
// written: gives the mask of these places.
template <typename T, int PASSES, bool STREAM, typename Written>
__device__ inline void store_run(const Fp8StoreParams& p, int blk, int h, int row, int d, const u32x4 (&kx)[PASSES],
                                 const u32x4 (&vx)[PASSES], const int (&place)[PASSES], bool begins, Written written) {
  const int page = quotient(blk, p.blocks), group = blk - page * (int)p.blocks.d;
  uint8_t* kb = p.kp + page * p.kp_sp + h * p.kp_sh + (int64_t)group * 16 * p.kp_ss;
  uint8_t* vb = p.vp + page * p.vp_sp + h * p.vp_sh + (int64_t)group * 16 * p.vp_ss;
  float* sc = p.scales + page * p.sc_sp + h * p.sc_sh + group * 2;
  const f32x2 old = *(const f32x2*)sc;

  uint32_t km = 0, vm = 0;
#pragma unroll
  for (int i = 0; i < PASSES; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      km = pk_max(km, kx[i][j] & 0x7fff7fffu);
      vm = pk_max(vm, vx[i][j] & 0x7fff7fffu);
    }
  // Magnitudes as 16-bit numbers: those of K in the low half, of V in the high.
  auto both = [](uint32_t k, uint32_t v) {
    return pk_max((k & 0xffffu) | v << 16, k >> 16 | (v & 0xffff0000u));
  };
  uint32_t most = wave_pk_max(both(km, vm));
  constexpr uint32_t kExp = HalfBits<T>::exp;
  const bool odd = (most & 0xffffu) >= kExp || (most >> 16) >= kExp;
  if (odd) {  // the largest finite ones
    auto finite = [](uint32_t x) {
      const uint32_t lo = x & 0x7fffu, hi = x >> 16 & 0x7fffu;
      return (lo >= kExp ? 0u : lo) | (hi >= kExp ? 0u : hi << 16);
    };
    km = vm = 0;
#pragma unroll
    for (int i = 0; i < PASSES; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        km = pk_max(km, finite(kx[i][j]));
        vm = pk_max(vm, finite(vx[i][j]));
      }
    most = wave_pk_max(both(km, vm));
  }
  most = __builtin_amdgcn_readfirstlane(most);
  int ek = scale_exponent(Elem<T>::to_f32((uint16_t)most)), ev = scale_exponent(Elem<T>::to_f32((uint16_t)(most >> 16)));
  const uint32_t ok = __builtin_amdgcn_readfirstlane(__float_as_uint(old[0]));
  const uint32_t ov = __builtin_amdgcn_readfirstlane(__float_as_uint(old[1]));
  bool grown = false;
  if (!begins) {
    const int bk = (int)(ok >> 23 & 0xff), bv = (int)(ov >> 23 & 0xff);
    grown = ek > bk || ev > bv;
    ek = max(ek, bk);
    ev = max(ev, bv);
  }
  // 240 for the scale whose 256 is 2^top, the largest code before it for those behind.
  auto limit_of = [](int e) {
    const int room = HalfBits<T>::top - (e - 127);
    return room < 9 ? ldexpf(0.9375f, room) : 448.f;
  };
  const float klimit = limit_of(ek), vlimit = limit_of(ev);
  const bool special = odd || klimit < 448.f || vlimit < 448.f;
  const float kinv = power(254 - ek), vinv = power(254 - ev);
  if (grown) {
    const uint32_t mine = written();
    // A block of scale 0 holds nothing.
    const float kr = ok ? __uint_as_float(ok) * kinv : 0.f, vr = ov ? __uint_as_float(ov) * vinv : 0.f;
#pragma unroll 1
    for (int r = row; r < 16; r += p.rows) {
      if (row >= p.rows || (mine >> r & 1)) continue;
      u32x2* ka = (u32x2*)(kb + r * p.kp_ss + d);
      u32x2* va = (u32x2*)(vb + r * p.vp_ss + d);
      const u32x2 k8 = *ka, v8 = *va;
      *ka = rescale(k8, kr);
      *va = rescale(v8, vr);
    }
  }
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    if (place[i] < 0) continue;
    const u32x2 k8 = quantise<T>(kx[i], kinv, klimit, special), v8 = quantise<T>(vx[i], vinv, vlimit, special);
    u32x2* ka = (u32x2*)(kb + place[i] * p.kp_ss + d);
    u32x2* va = (u32x2*)(vb + place[i] * p.vp_ss + d);
    if constexpr (STREAM) {
      __builtin_nontemporal_store(k8, ka);
      __builtin_nontemporal_store(v8, va);
    } else {
      *ka = k8;
      *va = v8;
    }
  }
  if ((threadIdx.x & 63) == 0) *(f32x2*)sc = f32x2{power(ek), power(ev)};
}

// One token per request: a wave per request and head. Its row is on its way
// while the slot is (64 tokens, 8 heads of 128, in a graph: 3.75 us by the kernel
// below, 3.19 by this one).
template <typename T>
__global__ __launch_bounds__(256) void fp8_store_one_kernel(const Fp8StoreParams p) {
  const int lane = threadIdx.x & 63;
  const int w = blockIdx.x * 4 + wave_index();
  if (w >= p.waves) return;
  const int64_t b = quotient(w, p.heads);
  const int h = w - (int)b * (int)p.heads.d;
  const int row = lane / p.lanes, d = (lane - row * p.lanes) * 8;
  const int64_t slot = p.slots[b * p.s_sb];
  u32x4 kx[1] = {zero_u4()}, vx[1] = {zero_u4()};
  if (row == 0) {
    kx[0] = ldg16(p.nk + b * p.nk_sb + h * p.nk_sh + d);
    vx[0] = ldg16(p.nv + b * p.nv_sb + h * p.nv_sh + d);
  }
  if (slot < 0 || slot >= p.places) return;
  const int blk = __builtin_amdgcn_readfirstlane((int)(slot >> 4)), at = __builtin_amdgcn_readfirstlane((int)slot & 15);
  const int place[1] = {row == 0 ? at : -1};
  store_run<T, 1, false>(p, blk, h, row, d, kx, vx, place, at == 0, [&] { return 1u << at; });
}

// A wave per request, window of 16 new tokens and head: it stores the runs of
// tokens of one block that begin in its window (one, in a prompt), so that
// every block has one wave. `lanes` lanes hold a row, eight elements each.
template <typename T, int PASSES, bool STREAM>
__global__ __launch_bounds__(256) void fp8_store_kernel(const Fp8StoreParams p) {
  const int lane = threadIdx.x & 63;
  const int w = blockIdx.x * 4 + wave_index();
  if (w >= p.waves) return;
  const int bw = quotient(w, p.heads), h = w - bw * (int)p.heads.d;
  const int64_t b = quotient(bw, p.windows);
  const int t0 = (bw - (int)b * (int)p.windows.d) * 16;

  // Lane l: the slot of token t0 - 1 + l, and its block, -1 if there is none.
  const int t = t0 - 1 + lane;
  int64_t slot = -1;
  if (t >= 0 && t < p.n && lane <= 32) slot = p.slots[b * p.s_sb + t];
  const int block = slot >= 0 && slot < p.places ? (int)(slot >> 4) : -1;
  const int before = __builtin_amdgcn_update_dpp(-1, block, 0x138, 0xf, 0xf, false);  // of lane - 1
  uint64_t starts = __builtin_amdgcn_ballot_w64(lane >= 1 && lane <= 16 && block >= 0 && block != before);
  const int row = lane / p.lanes, d = (lane - row * p.lanes) * 8;

  while (starts) {
    const int first = __builtin_ctzll(starts);
    starts &= starts - 1;
    const int blk = __builtin_amdgcn_readlane(block, first);
    const uint64_t same = __builtin_amdgcn_ballot_w64(block == blk) >> first;
    const int count = min(__builtin_ctzll(~same), 16);
    u32x4 kx[PASSES], vx[PASSES];
    int place[PASSES];
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int r = i * p.rows + row;
      const int at = __builtin_amdgcn_ds_bpermute((first + r) * 4, (int)slot & 15);
      place[i] = row < p.rows && r < count ? at : -1;
      kx[i] = vx[i] = zero_u4();
      if (place[i] >= 0) {
        const int64_t from = t0 - 1 + first + r;
        kx[i] = ldg16(p.nk + b * p.nk_sb + h * p.nk_sh + from * p.nk_ss + d);
        vx[i] = ldg16(p.nv + b * p.nv_sb + h * p.nv_sh + from * p.nv_ss + d);
      }
    }
    const bool mine = block == blk && lane >= first && lane < first + count;
    const bool begins = __builtin_amdgcn_ballot_w64(mine && (slot & 15) == 0) != 0;
    store_run<T, PASSES, STREAM>(p, blk, h, row, d, kx, vx, place, begins, [&] {
      uint32_t mask = 0;
      for (int i = 0; i < 16; ++i)
        if (__builtin_amdgcn_ballot_w64(mine && ((int)slot & 15) == i)) mask |= 1u << i;
      return mask;
    });
  }
}

struct Fp8ReadParams {
  const uint8_t* kp;
  const uint8_t* vp;
  const float* scales;
  uint16_t* ko;
  uint16_t* vo;
  const int32_t* tables;
  const int32_t* lengths;
  const int32_t* starts;  // null: `start`
  int64_t start;
  int64_t t_sb;
  int64_t kp_sp, kp_sh, kp_ss;
  int64_t vp_sp, vp_sh, vp_ss;
  int64_t sc_sp, sc_sh;
  int64_t ko_sb, ko_sh, ko_ss;
  int64_t vo_sb, vo_sh, vo_ss;
  int64_t cap;            // tokens that a table has columns for
  int items;              // 8-element pieces of a request and head
  Divisor blocks;         // workgroups of a request and head
  Divisor heads, pieces;  // pieces of a row
  Divisor page;
  int pages;
};

// Eight codes times their block's scale.
template <typename T>
__device__ inline u32x4 dequantise(u32x2 codes, float scale) {
  return {dequantise2<T, false>(codes[0], scale), dequantise2<T, true>(codes[0], scale),
          dequantise2<T, false>(codes[1], scale), dequantise2<T, true>(codes[1], scale)};
}

// A thread per 8 elements of a row of K and of V: a wave's stores are whole
// kilobytes. HBM-bound: 459 MB written and 229 read 117 us, 5.9 TB/s; 16
// elements per thread 143, two or four rows per thread 121 and 127.
template <typename T, bool STREAM>
__global__ __launch_bounds__(256) void fp8_read_kernel(const Fp8ReadParams p) {
  const int bh = quotient(blockIdx.x, p.blocks);
  const int item = ((int)blockIdx.x - bh * (int)p.blocks.d) * 256 + threadIdx.x;
  if (item >= p.items) return;
  const int64_t b = quotient(bh, p.heads);
  const int h = bh - (int)b * (int)p.heads.d;
  const int t = quotient(item, p.pieces);
  const int d = (item - t * (int)p.pieces.d) * 8;
  int64_t first = p.starts ? p.starts[b] : p.start;
  first = first < 0 ? 0 : first;
  const int64_t held = p.lengths[b], at = first + t;
  u32x4 k = zero_u4(), v = zero_u4();
  if (at < held && at < p.cap) {
    const int column = quotient((int)at, p.page), row = (int)at - column * (int)p.page.d;
    const int id = p.tables[b * p.t_sb + column];
    if (id >= 0 && id < p.pages) {
      const u32x2 k8 = *(const u32x2*)(p.kp + id * p.kp_sp + h * p.kp_sh + row * p.kp_ss + d);
      const u32x2 v8 = *(const u32x2*)(p.vp + id * p.vp_sp + h * p.vp_sh + row * p.vp_ss + d);
      const f32x2 s = *(const f32x2*)(p.scales + id * p.sc_sp + h * p.sc_sh + (row >> 4) * 2);
      k = dequantise<T>(k8, s[0]);
      v = dequantise<T>(v8, s[1]);
    }
  }
  u32x4* ko = (u32x4*)(p.ko + b * p.ko_sb + h * p.ko_sh + t * p.ko_ss + d);
  u32x4* vo = (u32x4*)(p.vo + b * p.vo_sb + h * p.vo_sh + t * p.vo_ss + d);
  if constexpr (STREAM) {
    __builtin_nontemporal_store(k, ko);
    __builtin_nontemporal_store(v, vo);
  } else {
    *ko = k;
    *vo = v;
  }
}

// Bytes of K and V from which the read's stores are marked as not read again
// soon (us, plain and marked: 67 MB 14.0 and 13.8, 134 MB 24.9 and 24.6, 268 MB 67
// and 46, beyond what the memory-side cache takes; 459 MB 128 and 117).
constexpr int64_t kStreamReads = 128 << 20;

int check_fp8_pools(const char* what, const void* k_pages, const void* v_pages, const void* scales, int64_t H,
                    int64_t D, int64_t num_pages, int64_t page_size, const int64_t* k_strides,
                    const int64_t* v_strides, const int64_t* scale_strides) {
  if (!k_pages || !v_pages || !scales) return set_error(KF_EINVAL, "%s: null pointer", what);
  if (!k_strides || !v_strides || !scale_strides) return set_error(KF_EINVAL, "%s: null strides", what);
  if (H <= 0 || D <= 0 || num_pages <= 0 || page_size <= 0)
    return set_error(KF_EINVAL, "%s: all sizes must be positive", what);
  if (D % 8 || D > 128) return set_error(KF_EUNSUPPORTED, "%s: head_dim must be a multiple of 8 up to 128", what);
  if (page_size % 16) return set_error(KF_EUNSUPPORTED, "%s: page_size must be a multiple of 16, got %lld", what, (long long)page_size);
  if (num_pages > 0x7fffffff || page_size > 0x3fffffff || H > 0x7fffffff || num_pages > (1ll << 35) / page_size)
    return set_error(KF_EUNSUPPORTED, "%s: dimension too large", what);
  if (!aligned16(k_pages) || !aligned16(v_pages) || !aligned8(scales))
    return set_error(KF_EINVAL, "%s: pools must be 16-byte aligned, scales 8-byte", what);
  for (const int64_t* s : {k_strides, v_strides})
    if (s[0] % 16 || s[1] % 16 || s[2] % 16)
      return set_error(KF_EINVAL, "%s: pool strides must be multiples of 16 bytes", what);
  if (scale_strides[0] % 2 || scale_strides[1] % 2)
    return set_error(KF_EINVAL, "%s: scale strides must be multiples of a pair", what);
  return KF_OK;
}

int check_tensor(const char* what, const char* name, const void* ptr, const int64_t* strides);

}  // namespace kf

using namespace kf;

extern "C" int kf_fp8_append(void* k_pages, void* v_pages, float* scales, const void* new_k, const void* new_v,
                             const int64_t* slots, int64_t B, int64_t H, int64_t Snew, int64_t D, int64_t num_pages,
                             int64_t page_size, int64_t slots_stride, const int64_t* k_strides,
                             const int64_t* v_strides, const int64_t* scale_strides, const int64_t* new_k_strides,
                             const int64_t* new_v_strides, int dtype, void* stream) {
  const char* what = "kf_fp8_append";
  int rc = check_fp8_pools(what, k_pages, v_pages, scales, H, D, num_pages, page_size, k_strides, v_strides, scale_strides);
  if (rc) return rc;
  if (!slots) return set_error(KF_EINVAL, "%s: slots is null", what);
  if (B <= 0 || Snew <= 0) return set_error(KF_EINVAL, "%s: all sizes must be positive", what);
  if ((rc = check_tensor(what, "new_k", new_k, new_k_strides)) || (rc = check_tensor(what, "new_v", new_v, new_v_strides)))
    return rc;
  if (dtype != KF_F16 && dtype != KF_BF16) return set_error(KF_EINVAL, "%s: dtype must be KF_F16 or KF_BF16", what);
  const int64_t windows = (Snew + 15) / 16;
  if (Snew > 0x3fffffff || B > 0x7fffffff / windows || B * windows > ((1ll << 26) - 4) / H)
    return set_error(KF_EUNSUPPORTED, "%s: grid too large", what);
  Fp8StoreParams p{};
  p.kp = (uint8_t*)k_pages; p.vp = (uint8_t*)v_pages; p.scales = scales;
  p.nk = (const uint16_t*)new_k; p.nv = (const uint16_t*)new_v;
  p.slots = slots; p.s_sb = slots_stride;
  p.kp_sp = k_strides[0]; p.kp_sh = k_strides[1]; p.kp_ss = k_strides[2];
  p.vp_sp = v_strides[0]; p.vp_sh = v_strides[1]; p.vp_ss = v_strides[2];
  p.sc_sp = scale_strides[0]; p.sc_sh = scale_strides[1];
  p.nk_sb = new_k_strides[0]; p.nk_sh = new_k_strides[1]; p.nk_ss = new_k_strides[2];
  p.nv_sb = new_v_strides[0]; p.nv_sh = new_v_strides[1]; p.nv_ss = new_v_strides[2];
  p.places = num_pages * page_size;
  p.n = (int)Snew;
  p.heads = divisor((uint32_t)H);
  p.windows = divisor((uint32_t)windows);
  p.blocks = divisor((uint32_t)(page_size / 16));
  p.waves = (int)(B * windows * H);
  p.lanes = (int)(D / 8);
  p.rows = 64 / p.lanes;
  const dim3 grid((unsigned)((p.waves + 3) / 4)), block(256);
  hipStream_t st = (hipStream_t)stream;
  auto launch = [&](auto type, auto once) {
    using T = decltype(type);
    constexpr bool S = decltype(once)::value;
    switch (cdiv(16, p.rows)) {
      case 1: hipLaunchKernelGGL((fp8_store_kernel<T, 1, S>), grid, block, 0, st, p); break;
      case 2: hipLaunchKernelGGL((fp8_store_kernel<T, 2, S>), grid, block, 0, st, p); break;
      case 3: hipLaunchKernelGGL((fp8_store_kernel<T, 3, S>), grid, block, 0, st, p); break;
      default: hipLaunchKernelGGL((fp8_store_kernel<T, 4, S>), grid, block, 0, st, p); break;
    }
  };
  const bool once = B * H * Snew * D * 4 >= kStreamRows;
  if (Snew == 1) {
    if (dtype == KF_F16) hipLaunchKernelGGL(fp8_store_one_kernel<_Float16>, grid, block, 0, st, p);
    else hipLaunchKernelGGL(fp8_store_one_kernel<__bf16>, grid, block, 0, st, p);
    return check_launch(what);
  }
  if (dtype == KF_F16) once ? launch(_Float16{}, std::true_type{}) : launch(_Float16{}, std::false_type{});
  else once ? launch(__bf16{}, std::true_type{}) : launch(__bf16{}, std::false_type{});
  return check_launch(what);
}

extern "C" int kf_fp8_read(const void* k_pages, const void* v_pages, const float* scales, void* k_out, void* v_out,
                           const int32_t* tables, const int32_t* lengths, const int32_t* starts, int64_t start,
                           int64_t B, int64_t H, int64_t width, int64_t D, int64_t num_pages, int64_t page_size,
                           int64_t columns, int64_t table_stride, const int64_t* k_strides, const int64_t* v_strides,
                           const int64_t* scale_strides, const int64_t* k_out_strides, const int64_t* v_out_strides,
                           int dtype, void* stream) {
  const char* what = "kf_fp8_read";
  int rc = check_fp8_pools(what, k_pages, v_pages, scales, H, D, num_pages, page_size, k_strides, v_strides, scale_strides);
  if (rc) return rc;
  if (!tables || !lengths) return set_error(KF_EINVAL, "%s: tables and lengths must be non-null", what);
  if (B <= 0 || width <= 0 || columns <= 0) return set_error(KF_EINVAL, "%s: all sizes must be positive", what);
  if (columns > 1 && table_stride < 0) return set_error(KF_EINVAL, "%s: negative table stride", what);
  if (!starts && start < 0) return set_error(KF_EINVAL, "%s: start must not be negative", what);
  if ((rc = check_tensor(what, "k_out", k_out, k_out_strides)) || (rc = check_tensor(what, "v_out", v_out, v_out_strides)))
    return rc;
  if (dtype != KF_F16 && dtype != KF_BF16) return set_error(KF_EINVAL, "%s: dtype must be KF_F16 or KF_BF16", what);
  if (page_size > 0x3fffffff / columns)
    return set_error(KF_EUNSUPPORTED, "%s: a table of %lld pages of %lld tokens is beyond 32-bit positions", what,
                     (long long)columns, (long long)page_size);
  Fp8ReadParams p{};
  const int64_t pieces = D / 8, blocks = (width * pieces + 255) / 256;
  if (width > 0x3fffffff / pieces || start > 0x3fffffff)
    return set_error(KF_EUNSUPPORTED, "%s: width or start too large", what);
  if (B > 0x7fffffff / H || B * H > ((1ll << 24) - 1) / blocks) return set_error(KF_EUNSUPPORTED, "%s: grid too large", what);
  p.items = (int)(width * pieces);
  p.pieces = divisor((uint32_t)pieces);
  p.blocks = divisor((uint32_t)blocks);
  p.heads = divisor((uint32_t)H);
  p.kp = (const uint8_t*)k_pages; p.vp = (const uint8_t*)v_pages; p.scales = scales;
  p.ko = (uint16_t*)k_out; p.vo = (uint16_t*)v_out;
  p.tables = tables; p.lengths = lengths; p.starts = starts; p.start = start; p.t_sb = table_stride;
  p.kp_sp = k_strides[0]; p.kp_sh = k_strides[1]; p.kp_ss = k_strides[2];
  p.vp_sp = v_strides[0]; p.vp_sh = v_strides[1]; p.vp_ss = v_strides[2];
  p.sc_sp = scale_strides[0]; p.sc_sh = scale_strides[1];
  p.ko_sb = k_out_strides[0]; p.ko_sh = k_out_strides[1]; p.ko_ss = k_out_strides[2];
  p.vo_sb = v_out_strides[0]; p.vo_sh = v_out_strides[1]; p.vo_ss = v_out_strides[2];
  p.cap = columns * page_size;
  p.page = divisor((uint32_t)page_size); p.pages = (int)num_pages;
  const dim3 grid((unsigned)(B * H * blocks));
  const bool once = B * H * width * D * 4 >= kStreamReads;
  hipStream_t st = (hipStream_t)stream;
  auto launch = [&](auto type) {
    using T = decltype(type);
    if (once) hipLaunchKernelGGL((fp8_read_kernel<T, true>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((fp8_read_kernel<T, false>), grid, dim3(256), 0, st, p);
  };
  if (dtype == KF_F16) launch(_Float16{});
  else launch(__bf16{});
  return check_launch(what);
}
