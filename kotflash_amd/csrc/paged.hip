// Attention over a paged K/V cache: the merge, launches and entry points. The
// workers' kernel, and how the work is cut, are in paged_attn.hpp.
#include "paged_attn.hpp"

namespace kf {

int check_attn_common(const char* what, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t Sk,
                      int64_t D, int dtype);
int check_tensor(const char* what, const char* name, const void* ptr, const int64_t* strides);

// One workgroup of W waves per output row: merges the row's partials, writes
// zeros where the request holds nothing, and leaves rows that one worker wrote
// whole. Bound by its chain of loads: which partials, then all of them. The
// first wave alone takes what one round trip brings; more partials the waves
// share, and combine through LDS in their order.
// Half the partials in flight of the contiguous decode's merge (half the
// registers, twice the rows at once: 8192 rows of two or three partials 7.3 us
// with 16, 5.7 with 8, 5.3 with 4; 131072 keys of one request and one KV head,
// about 1000 partials a row, want them).
constexpr int kPartsU = 8;
// With W = 1, four rows share a workgroup.
template <typename T, int QL, int W>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void paged_merge_kernel(const PagedParams p) {
  const int lane = threadIdx.x & 63, wave = wave_index();
  const int row = W == 1 ? blockIdx.x * 4 + wave : blockIdx.x;
  const int r = row % p.rows;
  const int bh = row / p.rows;
  if (W == 1 && bh >= p.B * p.heads) return;
  const int hh = bh % p.heads, b = bh / p.heads;
  const int kvh = hh / p.nrb, rho = (hh % p.nrb) * p.rows + r;
  // What the workers wrote is not there for a request without keys.
  const int len = ((const_i32)(uintptr_t)p.lengths)[b];
  const int w0 = ((const_i32)(uintptr_t)p.parts)[2 * bh], parts = ((const_i32)(uintptr_t)p.parts)[2 * bh + 1];
  if (rho >= p.G * p.Sq) return;
  const bool alone = W == 1 || len <= 0 || parts <= kPartsU * (64 / QL);
  if (W > 1 && alone && wave > 0) return;
  const int h = kvh * p.G + rho / p.Sq, i = rho % p.Sq;
  uint16_t* out = p.o + b * p.o_sb + h * p.o_sh + i * p.o_ss;
  float* lse = p.lse ? p.lse + ((int64_t)b * p.Hq + h) * p.Sq + i : nullptr;
  if (len <= 0) {
    if (4 * lane < p.D) *reinterpret_cast<u32x2*>(out + 4 * lane) = u32x2{0u, 0u};
    if (lane == 0 && lse) *lse = kNegInf;
    return;
  }
  if (parts == 1) return;
  const int64_t slot = (int64_t)(w0 + bh) * p.rows + r;
  const auto orr = make_rsrc(p.part_o + slot * p.D, (uint32_t)(((int64_t)(parts - 1) * p.rows * p.D + p.D) * 4));
  const auto lrr = make_rsrc(p.part_lse + slot, (uint32_t)(((int64_t)(parts - 1) * p.rows + 1) * 4));
  const uint32_t ostride = (uint32_t)(p.rows * p.D), lstride = (uint32_t)p.rows;
  if (alone) {
    merge_row<T, QL, kPartsU>(orr, lrr, ostride, lstride, parts, p.D, out, lse);
    return;
  }
  if constexpr (W > 1) {
    __shared__ float sums[W][QL][6];
    const int share = (parts + W - 1) / W;
    const MergeState mine = merge_splits<QL, kPartsU>(orr, lrr, ostride, lstride, min(wave * share, parts),
                                             min((wave + 1) * share, parts), p.D);
    if (lane < QL) {
      float* to = sums[wave][lane];
      to[0] = mine.M; to[1] = mine.den;
      for (int e = 0; e < 4; ++e) to[2 + e] = mine.acc[e];
    }
    __syncthreads();
    if (wave > 0) return;
    MergeState all = {{0.f, 0.f, 0.f, 0.f}, 0.f, kNegInf};
    for (int w = 0; w < W; ++w) all.M = fmaxf(all.M, sums[w][lane % QL][0]);
    const float Ms = all.M == kNegInf ? 0.f : all.M;
    for (int w = 0; w < W; ++w) {
      const float* from = sums[w][lane % QL];
      const float sc = fast_exp2(from[0] - Ms);
      all.den += sc * from[1];
      for (int e = 0; e < 4; ++e) all.acc[e] += sc * from[2 + e];
    }
    merge_store<T, QL>(all, p.D, out, lse);
  }
}

// Workers: what 256 CUs hold of them at once.
template <int NW>
static int workers_of(int DT, bool kv8) {
  return 256 * (DT == 32 ? workers_per_cu(32, NW, kv8) : DT == 64 ? workers_per_cu(64, NW, kv8)
                : DT == 96 ? workers_per_cu(96, NW, kv8) : workers_per_cu(128, NW, kv8));
}
static int paged_workers(int64_t D, int64_t R, bool kv8) {
  const int DT = paged_tile(D, kv8), NW = paged_waves(R);
  return NW == 1 ? workers_of<1>(DT, kv8) : NW == 2 ? workers_of<2>(DT, kv8) : workers_of<4>(DT, kv8);
}

static int64_t paged_slots(int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t D, bool kv8) {
  const int64_t R = Hq / Hkv * Sq;
  return paged_workers(D, R, kv8) + B * Hkv * ((R + paged_rows(R) - 1) / paged_rows(R));
}

// Waves per row of the merge, from the most partials a row group can have: a
// head's share of the workers (all of them on one request), cut at both ends.
// More waves cost launch time where they are not needed and save round trips
// where one row has many partials. Measured, us with one, four and sixteen
// waves: 8192 rows of two or three partials 5.7, 9.8 and 30, 2048 of them 4.6,
// 4.7 and 10; 32 rows of 128 partials 7.6, 4.7 and 5.0; 16 rows of about 1000
// 37, 11.8 and 9.5.
template <typename T, int QL>
static void launch_merge(const PagedParams& p, hipStream_t stream) {
  constexpr int kTrip = kPartsU * (64 / QL);  // partials that a wave takes at once
  const int64_t rows = (int64_t)p.B * p.heads * p.rows;
  const int share = p.workers / p.heads + 2, steps = p.cap / (p.scales ? kStepOf<true> : kStepOf<false>) + 1;
  const int most = share < steps ? share : steps;
  const dim3 grid((unsigned)rows);
  if (most > 16 * kTrip && rows <= 256)
    hipLaunchKernelGGL((paged_merge_kernel<T, QL, 16>), grid, dim3(1024), 0, stream, p);
  else if (most > kTrip && (rows <= 256 || (most > 8 * kTrip && rows <= 2048) || (most > 32 * kTrip && rows < 1 << 24)))
    hipLaunchKernelGGL((paged_merge_kernel<T, QL, 4>), grid, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((paged_merge_kernel<T, QL, 1>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream, p);
}

template <typename T, int DT, int NW>
static void launch_workers(const PagedParams& p, hipStream_t stream) {
  const dim3 grid((unsigned)p.workers), block(64 * NW);
  if (p.nnew > 0) hipLaunchKernelGGL((paged_kernel<T, DT, NW, true, kPool16>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((paged_kernel<T, DT, NW, false, kPool16>), grid, block, 0, stream, p);
}

template <typename T, int DT>
static void launch_paged(const PagedParams& p, hipStream_t stream) {
  switch (paged_waves(p.rows)) {
    case 1: launch_workers<T, DT, 1>(p, stream); break;
    case 2: launch_workers<T, DT, 2>(p, stream); break;
    default: launch_workers<T, DT, 4>(p, stream); break;
  }
}

template <typename T>
static int dispatch_paged(const char* what, const PagedParams& p, hipStream_t stream) {
  if (p.scales) {
    launch_workers_fp8(p, std::is_same_v<T, _Float16> ? KF_F16 : KF_BF16, stream);
  } else {
    switch (head_tile(p.D)) {
      case 32: launch_paged<T, 32>(p, stream); break;
      case 64: launch_paged<T, 64>(p, stream); break;
      case 96: launch_paged<T, 96>(p, stream); break;
      default: launch_paged<T, 128>(p, stream); break;
    }
  }
  const int rc = check_launch(what);
  if (rc) return rc;
  if (p.D <= 64) launch_merge<T, 16>(p, stream);
  else launch_merge<T, 32>(p, stream);
  return check_launch(what);
}

}  // namespace kf

using namespace kf;

static size_t workspace_bytes_of(int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t D, bool kv8) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Sq <= 0 || D <= 0 || D > 128 || Hq % Hkv) return 0;
  const int64_t R = Hq / Hkv * Sq;
  const size_t rows = (size_t)paged_slots(B, Hq, Hkv, Sq, D, kv8) * paged_rows(R);
  const size_t groups = (size_t)(B * Hkv * ((R + paged_rows(R) - 1) / paged_rows(R)));
  return (rows * (size_t)D * sizeof(float) + 255) / 256 * 256 + (rows * sizeof(float) + 255) / 256 * 256 +
         groups * 2 * sizeof(int32_t);
}

extern "C" size_t kf_paged_decode_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t D) {
  return workspace_bytes_of(B, Hq, Hkv, Sq, D, false);
}

extern "C" size_t kf_fp8_decode_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t D) {
  return workspace_bytes_of(B, Hq, Hkv, Sq, D, true);
}

// Scales of 8-bit pools; null for 16-bit ones.
struct Scales {
  const float* at;
  const int64_t* strides;
};

// New rows of kf_paged_append_decode; n = 0 without.
struct NewRows {
  const void *k, *v;
  const int64_t* slots;
  int64_t n, slots_stride;
  const int64_t *k_strides, *v_strides;
};

// Rows that the merge's launch takes at one wave each: HIP counts a grid's threads
// in 32 bits.
constexpr int64_t kMergeRows = (1ll << 32) / 64 - 4;

// Extent of one KV head's queries or outputs.
static int64_t group_bytes(int64_t Hq, int64_t Hkv, int64_t Sq, int64_t D, const int64_t* strides) {
  return ((Hq / Hkv - 1) * strides[1] + (Sq - 1) * strides[2] + D) * 2;
}

// The sizes and strides that the kernels address.
static int check_paged_sizes(const char* what, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t D,
                             int64_t num_pages, int64_t page_size, int64_t columns, const int64_t* q_strides,
                             const int64_t* k_strides, const int64_t* v_strides, const int64_t* o_strides) {
  if (num_pages <= 0 || columns <= 0 || num_pages > 0x7fffffff)
    return set_error(KF_EINVAL, "%s: num_pages and table columns must be positive", what);
  if (page_size <= 0 || page_size % 16 != 0)
    return set_error(KF_EUNSUPPORTED, "%s: page_size must be a multiple of 16, got %lld", what, (long long)page_size);
  if (page_size > 0x3fffffff / columns)
    return set_error(KF_EUNSUPPORTED, "%s: a table of %lld pages of %lld tokens is beyond 32-bit positions", what,
                     (long long)columns, (long long)page_size);
  const int64_t R = Hq / Hkv * Sq;
  if (R > 0x3fffffff) return set_error(KF_EUNSUPPORTED, "%s: too many query rows", what);
  const int rows = paged_rows(R);
  const int64_t nrb = (R + rows - 1) / rows, heads = Hkv * nrb;
  const int64_t cap = columns * page_size;
  constexpr int kStep = kStepOf<false>;
  if (heads * ((cap + kStep - 1) / kStep) > 0x7f000000 / B)
    return set_error(KF_EUNSUPPORTED, "%s: %lld tables of %lld tokens are beyond 32-bit step numbers", what,
                     (long long)B, (long long)cap);
  if (B * heads * rows > kMergeRows) return set_error(KF_EUNSUPPORTED, "%s: grid too large", what);
  if (group_bytes(Hq, Hkv, Sq, D, q_strides) > 0x7fffffff || group_bytes(Hq, Hkv, Sq, D, o_strides) > 0x7fffffff)
    return set_error(KF_EUNSUPPORTED, "%s: one KV group of q or o spans more than 2 GiB", what);
  for (const int64_t* st : {k_strides, v_strides})
    if ((15 * st[2] + D) * 2 > 0x7fffffffLL || st[0] > 0x7fffffffLL)
      return set_error(KF_EUNSUPPORTED, "%s: 16 rows of a page span more than 2 GiB, or a page more than 4", what);
  return KF_OK;
}

static int paged_entry(const char* what, const void* q, const void* k_pages, const void* v_pages,
                       const Scales& scales, const NewRows& fresh, void* o, float* lse, const int32_t* tables, const int32_t* lengths,
                       int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t D, int64_t num_pages,
                       int64_t page_size, int64_t columns, int64_t table_stride, const int64_t* q_strides,
                       const int64_t* k_strides, const int64_t* v_strides, const int64_t* o_strides, float scale,
                       int causal, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_attn_common(what, B, Hq, Hkv, Sq, 1, D, dtype);
  if (rc) return rc;
  if ((rc = check_tensor(what, "q", q, q_strides)) || (rc = check_tensor(what, "k_pages", k_pages, k_strides)) ||
      (rc = check_tensor(what, "v_pages", v_pages, v_strides)) || (rc = check_tensor(what, "o", o, o_strides)))
    return rc;
  if (tables == nullptr || lengths == nullptr)
    return set_error(KF_EINVAL, "%s: tables and lengths must be non-null", what);
  if (!(scale == scale) || scale - scale != 0.f) return set_error(KF_EINVAL, "%s: scale must be finite", what);
  if (columns > 1 && table_stride < 0) return set_error(KF_EINVAL, "%s: negative table stride", what);
  if ((rc = check_paged_sizes(what, B, Hq, Hkv, Sq, D, num_pages, page_size, columns, q_strides, k_strides, v_strides,
                              o_strides)))
    return rc;
  const bool kv8 = scales.at != nullptr;
  const size_t need = workspace_bytes_of(B, Hq, Hkv, Sq, D, kv8);
  if (workspace == nullptr || workspace_bytes < need)
    return set_error(KF_EINVAL, "%s: workspace of %zu bytes required, got %zu", what, need,
                     workspace == nullptr ? (size_t)0 : workspace_bytes);
  if (!aligned16(workspace)) return set_error(KF_EINVAL, "%s: workspace must be 16-byte aligned", what);
  const int64_t R = Hq / Hkv * Sq, cap = columns * page_size;
  const int rows = paged_rows(R);
  const int64_t nrb = (R + rows - 1) / rows, heads = Hkv * nrb;
  const int64_t q_bytes = group_bytes(Hq, Hkv, Sq, D, q_strides), o_bytes = group_bytes(Hq, Hkv, Sq, D, o_strides);
  PagedParams p{};
  p.q = (const uint16_t*)q; p.k = (const uint16_t*)k_pages; p.v = (const uint16_t*)v_pages;
  p.o = (uint16_t*)o; p.lse = lse; p.tables = tables; p.lengths = lengths;
  const size_t slot_rows = (size_t)paged_slots(B, Hq, Hkv, Sq, D, kv8) * rows;
  p.part_o = (float*)workspace;
  p.part_lse = (float*)((char*)workspace + (slot_rows * (size_t)D * sizeof(float) + 255) / 256 * 256);
  p.parts = (int32_t*)((char*)p.part_lse + (slot_rows * sizeof(float) + 255) / 256 * 256);
  p.t_sb = table_stride;
  p.q_sb = q_strides[0]; p.q_sh = q_strides[1]; p.q_ss = q_strides[2];
  p.k_sh = k_strides[1]; p.v_sh = v_strides[1];
  const int eb = kv8 ? 1 : 2;
  p.k_page = (uint32_t)(eb * k_strides[0]); p.v_page = (uint32_t)(eb * v_strides[0]);
  p.k_row = (uint32_t)(eb * k_strides[2]); p.v_row = (uint32_t)(eb * v_strides[2]);
  if (kv8) {
    p.scales = scales.at;
    p.sc_page = (uint32_t)(4 * scales.strides[0]);
    p.sc_head = (uint32_t)(4 * scales.strides[1]);
    p.row_rest = (int)(k_strides[2] - (D + 15) / 16 * 16);
  }
  p.o_sb = o_strides[0]; p.o_sh = o_strides[1]; p.o_ss = o_strides[2];
  p.B = (int)B; p.Hq = (int)Hq; p.Hkv = (int)Hkv; p.Sq = (int)Sq; p.D = (int)D; p.G = (int)(Hq / Hkv);
  p.pages = (int)num_pages; p.gpp = (int)(page_size / 16);
  p.cap = (int)cap;
  p.rows = rows; p.nrb = (int)nrb; p.heads = (int)heads;
  p.workers = paged_workers(D, R, kv8);
  p.q_bytes = (uint32_t)q_bytes;
  p.o_bytes = (uint32_t)o_bytes;
  p.causal = causal != 0;
  p.scale_log2 = scale * kLog2e;
  p.page_size = (int)page_size;
  p.nnew = (int)fresh.n;
  p.nnew_inv = fresh.n > 0 ? (uint32_t)(65536 / fresh.n + 1) : 0;
  if (fresh.n > 0) {
    p.nk = (const uint16_t*)fresh.k; p.nv = (const uint16_t*)fresh.v;
    p.slots = fresh.slots; p.s_sb = fresh.slots_stride;
    p.nk_sb = fresh.k_strides[0]; p.nk_sh = fresh.k_strides[1]; p.nk_ss = fresh.k_strides[2];
    p.nv_sb = fresh.v_strides[0]; p.nv_sh = fresh.v_strides[1]; p.nv_ss = fresh.v_strides[2];
  }
  hipStream_t s = (hipStream_t)stream;
  return dtype == KF_F16 ? dispatch_paged<_Float16>(what, p, s) : dispatch_paged<__bf16>(what, p, s);
}

extern "C" int kf_paged_decode_check(int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t D, int64_t num_pages,
                                     int64_t page_size, int64_t columns, const int64_t* q_strides,
                                     const int64_t* k_strides, const int64_t* v_strides) {
  const char* what = "kf_paged_decode";
  const int rc = check_attn_common(what, B, Hq, Hkv, Sq, 1, D, KF_F16);
  if (rc) return rc;
  if (!q_strides || !k_strides || !v_strides) return set_error(KF_EINVAL, "%s: null strides", what);
  const int64_t o_strides[3] = {Hq * Sq * D, Sq * D, D};
  return check_paged_sizes(what, B, Hq, Hkv, Sq, D, num_pages, page_size, columns, q_strides, k_strides, v_strides,
                           o_strides);
}

extern "C" int kf_paged_decode(const void* q, const void* k_pages, const void* v_pages, void* o, float* lse,
                               const int32_t* tables, const int32_t* lengths, int64_t B, int64_t Hq, int64_t Hkv,
                               int64_t Sq, int64_t D, int64_t num_pages, int64_t page_size, int64_t columns,
                               int64_t table_stride, const int64_t* q_strides, const int64_t* k_strides,
                               const int64_t* v_strides, const int64_t* o_strides, float scale, int causal,
                               int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  return paged_entry("kf_paged_decode", q, k_pages, v_pages, Scales{}, NewRows{}, o, lse, tables, lengths, B, Hq, Hkv, Sq, D,
                     num_pages, page_size, columns, table_stride, q_strides, k_strides, v_strides, o_strides, scale,
                     causal, dtype, workspace, workspace_bytes, stream);
}

extern "C" int kf_paged_append_decode(const void* q, void* k_pages, void* v_pages, const void* new_k,
                                      const void* new_v, const int64_t* slots, void* o, float* lse,
                                      const int32_t* tables, const int32_t* lengths, int64_t B, int64_t Hq,
                                      int64_t Hkv, int64_t Sq, int64_t Snew, int64_t D, int64_t num_pages,
                                      int64_t page_size, int64_t columns, int64_t table_stride, int64_t slots_stride,
                                      const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                                      const int64_t* new_k_strides, const int64_t* new_v_strides,
                                      const int64_t* o_strides, float scale, int causal, int dtype, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  const char* what = "kf_paged_append_decode";
  int rc;
  if ((rc = check_tensor(what, "new_k", new_k, new_k_strides)) || (rc = check_tensor(what, "new_v", new_v, new_v_strides)))
    return rc;
  if (slots == nullptr) return set_error(KF_EINVAL, "%s: slots is null", what);
  if (Snew < 1 || Snew > KF_PAGED_STEP_TOKENS)
    return set_error(KF_EUNSUPPORTED, "%s: 1 to %d new tokens per request, got %lld", what, KF_PAGED_STEP_TOKENS,
                     (long long)Snew);
  if (B > KF_PAGED_STEP_SLOTS / Snew)
    return set_error(KF_EUNSUPPORTED, "%s: up to %d new tokens in all, got %lld", what, KF_PAGED_STEP_SLOTS,
                     (long long)(B * Snew));
  if (page_size > 0 && num_pages > 0x7fffffff / page_size)
    return set_error(KF_EUNSUPPORTED, "%s: a pool of 2^31 slots or more", what);
  const NewRows fresh = {new_k, new_v, slots, Snew, slots_stride, new_k_strides, new_v_strides};
  return paged_entry(what, q, k_pages, v_pages, Scales{}, fresh, o, lse, tables, lengths, B, Hq, Hkv, Sq, D, num_pages,
                     page_size, columns, table_stride, q_strides, k_strides, v_strides, o_strides, scale, causal,
                     dtype, workspace, workspace_bytes, stream);
}

// 8-bit pools: rows of whole 16-byte pieces, the last one perhaps half padding.
static int check_fp8_sizes(const char* what, int64_t D, int64_t num_pages, const int64_t* k_strides, const int64_t* v_strides,
                           const int64_t* scale_strides) {
  if (!scale_strides) return set_error(KF_EINVAL, "%s: null strides", what);
  if (D % 8 || D > 128) return set_error(KF_EUNSUPPORTED, "%s: head_dim must be a multiple of 8 up to 128", what);
  for (const int64_t* s : {k_strides, v_strides})
    if (s[0] % 16 || s[1] % 16 || s[2] % 16)
      return set_error(KF_EINVAL, "%s: pool strides must be multiples of 16 bytes", what);
  if (k_strides[0] != v_strides[0] || k_strides[1] != v_strides[1] || k_strides[2] != v_strides[2])
    return set_error(KF_EINVAL, "%s: K and V pools must have the same strides", what);
  if (k_strides[2] < (D + 15) / 16 * 16 || 16 * k_strides[2] > 0x7fffffff)
    return set_error(KF_EUNSUPPORTED, "%s: rows of a page overlap, or span more than 2 GiB", what);
  if (scale_strides[0] % 2 || scale_strides[1] % 2)
    return set_error(KF_EINVAL, "%s: scale strides must be multiples of a pair", what);
  // The scalar unit adds a page's offset to a head's in 32 bits.
  if (scale_strides[0] < 0 || scale_strides[1] < 0 || scale_strides[1] >= 1 << 30 ||
      scale_strides[0] > (1ll << 30) / (num_pages > 0 ? num_pages : 1) - 1)
    return set_error(KF_EUNSUPPORTED, "%s: scales of a head span more than 4 GiB", what);
  return KF_OK;
}

extern "C" int kf_fp8_decode_check(int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t D, int64_t num_pages,
                                   int64_t page_size, int64_t columns, const int64_t* q_strides,
                                   const int64_t* k_strides, const int64_t* v_strides, const int64_t* scale_strides) {
  const int rc = kf_paged_decode_check(B, Hq, Hkv, Sq, D, num_pages, page_size, columns, q_strides, k_strides, v_strides);
  return rc ? rc : check_fp8_sizes("kf_fp8_decode", D, num_pages, k_strides, v_strides, scale_strides);
}

extern "C" int kf_fp8_decode(const void* q, const void* k_pages, const void* v_pages, const float* scales, void* o,
                             float* lse, const int32_t* tables, const int32_t* lengths, int64_t B, int64_t Hq,
                             int64_t Hkv, int64_t Sq, int64_t D, int64_t num_pages, int64_t page_size,
                             int64_t columns, int64_t table_stride, const int64_t* q_strides,
                             const int64_t* k_strides, const int64_t* v_strides, const int64_t* scale_strides,
                             const int64_t* o_strides, float scale, int causal, int dtype, void* workspace,
                             size_t workspace_bytes, void* stream) {
  const char* what = "kf_fp8_decode";
  if (!scales || !aligned8(scales)) return set_error(KF_EINVAL, "%s: scales must be non-null and 8-byte aligned", what);
  if (!k_strides || !v_strides) return set_error(KF_EINVAL, "%s: null strides", what);
  const int rc = check_fp8_sizes(what, D, num_pages, k_strides, v_strides, scale_strides);
  if (rc) return rc;
  return paged_entry(what, q, k_pages, v_pages, Scales{scales, scale_strides}, NewRows{}, o, lse, tables, lengths, B,
                     Hq, Hkv, Sq, D, num_pages, page_size, columns, table_stride, q_strides, k_strides, v_strides,
                     o_strides, scale, causal, dtype, workspace, workspace_bytes, stream);
}
