// The pages of a paged K/V cache, on the GPU: block tables and slots from the
// requests' lengths, and the store of new K/V rows by slot. No counterpart in
// the reference, whose cache is one contiguous buffer (kotflash/cache.py:91).
//
// State of a page table (int32): tables [B, columns], the pages of every
// request in order, -1 where it has none; lengths [B], its tokens; free_pages
// [num_pages], a stack of the pages that belong to nobody; counters [4]: the
// stack's height, the requests that the last reserve refused, two spare.
//
// reserve, with p_b = ceil(L_b / page), need_b = ceil((L_b + c_b) / page) - p_b
// and C_b = need_0 + .. + need_b: request b is served iff its count and table
// allow it and need_b = 0 or C_b <= F (the height). C does not fall, so the
// requests in front of a served one that needs pages are served too, and what
// they took is C_b - need_b: one sum decides who is served and which pages
// they get, free_pages[F - 1 - (C_b - need_b) - i] for i < need_b.
// trim is its inverse: the pages behind ceil(min(L_b, n_b) / page) go back so
// that the reserve that took them would take the same ones again.
//
// Both are bound by latency: one workgroup, one sum over the batch.
#include "kf_common.hpp"
#include "kf_host.hpp"

namespace kf {

constexpr int kTableThreads = 1024;
constexpr int kTableWaves = kTableThreads / 64;

struct TableParams {
  int32_t* tables;
  int32_t* lengths;
  int32_t* free_pages;
  int32_t* counters;
  const int32_t* counts;  // reserve: per request, or null: `count` each; trim: new lengths, likewise
  int64_t* slots;         // [B, width]
  int64_t count, width;
  int64_t t_sb;
  int B, columns, page, pages;
};

// Inclusive sum over the workgroup; `sums` holds one value per wave. Ends with
// all waves past their reads of it.
__device__ inline int group_scan(int x, int* sums) {
  const int wave = wave_index();
  int s = wave_scan(x);
  if ((threadIdx.x & 63) == 63) sums[wave] = s;
  __syncthreads();
  for (int w = 0; w < wave; ++w) s += sums[w];
  __syncthreads();
  return s;
}

__device__ inline int pages_for(int tokens, int page) { return (tokens + page - 1) / page; }

__device__ inline int length_of(const TableParams& p, int b) {
  return min(max(p.lengths[b], 0), p.columns * p.page);
}

// The stack's height as far as it can be true.
__device__ inline int height(const TableParams& p) { return min(max(p.counters[0], 0), p.pages); }

__global__ __launch_bounds__(kTableThreads) void reserve_kernel(const TableParams p) {
  __shared__ int sums[kTableWaves];
  // Of the requests b0 + i of a turn: tokens before, tokens asked for (-1:
  // refused) and the place on the stack of their first new page.
  __shared__ int len_s[kTableThreads], add_s[kTableThreads], top_s[kTableThreads];
  __shared__ int taken_s, refused_s;
  const int tid = threadIdx.x;
  const int F = height(p);
  if (tid == 0) taken_s = refused_s = 0;
  int asked = 0;  // pages asked for by the requests of the turns before
  for (int b0 = 0; b0 < p.B; b0 += kTableThreads) {
    const int b = b0 + tid;
    const bool here = b < p.B;
    const int len = here ? length_of(p, b) : 0;
    const int64_t c = here ? (p.counts ? (int64_t)p.counts[b] : p.count) : 0;
    const bool fits = c >= 0 && c <= p.width && len + c <= (int64_t)p.columns * p.page;
    const int need = fits ? pages_for(len + (int)c, p.page) - pages_for(len, p.page) : 0;
    const int upto = asked + group_scan(need, sums);
    const bool served = here && fits && (need == 0 || upto <= F);
    len_s[tid] = len;
    add_s[tid] = served ? (int)c : -1;
    top_s[tid] = F - 1 - (upto - need);
    if (served && need > 0) atomicMax(&taken_s, upto);
    if (here && !served) atomicAdd(&refused_s, 1);
    __syncthreads();
    const int m = min(kTableThreads, p.B - b0);
    // New table entries: a wave per request.
    for (int i = wave_index(); i < m; i += kTableWaves) {
      if (add_s[i] < 0) continue;
      const int first = pages_for(len_s[i], p.page), end = pages_for(len_s[i] + add_s[i], p.page);
      for (int col = first + (tid & 63); col < end; col += 64)
        p.tables[(b0 + i) * p.t_sb + col] = p.free_pages[top_s[i] - (col - first)];
    }
    // Slots.
    const int64_t all = m * p.width;
    for (int64_t e = tid; e < all; e += kTableThreads) {
      const int i = (int)(e / p.width), t = (int)(e - i * p.width);
      int64_t slot = -1;
      if (t < add_s[i]) {
        const int pos = len_s[i] + t, col = pos / p.page, first = pages_for(len_s[i], p.page);
        const int id = col < first ? p.tables[(b0 + i) * p.t_sb + col] : p.free_pages[top_s[i] - (col - first)];
        slot = id < 0 ? -1 : (int64_t)id * p.page + (pos - col * p.page);
      }
      p.slots[(b0 + i) * p.width + t] = slot;
    }
    if (served) p.lengths[b] = len + (int)c;
    // Everybody's sum so far, from the last thread.
    __syncthreads();
    if (tid == kTableThreads - 1) sums[0] = upto;
    __syncthreads();
    asked = sums[0];
    __syncthreads();
  }
  if (tid == 0) {
    p.counters[0] = F - taken_s;
    p.counters[1] = refused_s;
  }
}

__global__ __launch_bounds__(kTableThreads) void trim_kernel(const TableParams p) {
  __shared__ int sums[kTableWaves];
  __shared__ int from_s[kTableThreads], end_s[kTableThreads], rank_s[kTableThreads];
  __shared__ int total_s;
  const int tid = threadIdx.x;
  const int F = height(p);
  auto kept = [&](int b, int len) {
    const int64_t to = p.counts ? (int64_t)p.counts[b] : p.count;
    return (int)min((int64_t)len, max(to, (int64_t)0));
  };
  if (tid == 0) total_s = 0;
  __syncthreads();
  // Pages that come back in all: the first of them in the requests' order
  // ends on top of the stack.
  int freed = 0;
  for (int b = tid; b < p.B; b += kTableThreads) {
    const int len = length_of(p, b);
    freed += pages_for(len, p.page) - pages_for(kept(b, len), p.page);
  }
  atomicAdd(&total_s, freed);
  __syncthreads();
  const int top = F + total_s - 1;
  int before = 0;
  for (int b0 = 0; b0 < p.B; b0 += kTableThreads) {
    const int b = b0 + tid;
    const bool here = b < p.B;
    const int len = here ? length_of(p, b) : 0;
    const int keep = here ? kept(b, len) : 0;
    const int from = pages_for(keep, p.page), end = pages_for(len, p.page);
    const int upto = before + group_scan(end - from, sums);
    from_s[tid] = from;
    end_s[tid] = end;
    rank_s[tid] = upto - (end - from);
    __syncthreads();
    const int m = min(kTableThreads, p.B - b0);
    for (int i = wave_index(); i < m; i += kTableWaves) {
      for (int col = from_s[i] + (tid & 63); col < end_s[i]; col += 64) {
        int32_t* entry = p.tables + (b0 + i) * p.t_sb + col;
        const int place = top - rank_s[i] - (col - from_s[i]);
        if (place >= 0 && place < p.pages) p.free_pages[place] = *entry;
        *entry = -1;
      }
    }
    if (here) p.lengths[b] = keep;
    __syncthreads();
    if (tid == kTableThreads - 1) sums[0] = upto;
    __syncthreads();
    before = sums[0];
    __syncthreads();
  }
  if (tid == 0) p.counters[0] = min(F + total_s, p.pages);
}

// Store of new K/V rows: pool[slot / page, h, slot % page] = new[b, h, t] for
// slot = slots[b, t], K and V, bit-exact; slots outside the pool are skipped.
// HBM-bound: each row is read once and written once. A thread moves 16 bytes
// of K and of V (one element where a layout does not allow it).
struct StoreParams {
  uint16_t* kp;
  uint16_t* vp;
  const uint16_t* nk;
  const uint16_t* nv;
  const int64_t* slots;
  int64_t s_sb;
  int64_t kp_sp, kp_sh, kp_ss;
  int64_t vp_sp, vp_sh, vp_ss;
  int64_t nk_sb, nk_sh, nk_ss, nk_sd;
  int64_t nv_sb, nv_sh, nv_ss, nv_sd;
  int64_t total, places;  // work items; slots of the pool
  int H, S, D, page;
};

template <bool VEC>
__global__ __launch_bounds__(256) void store_kernel(const StoreParams p) {
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (idx >= p.total) return;
  const int per_row = VEC ? p.D / 8 : p.D;
  const int c = (int)(idx % per_row);
  int64_t rest = idx / per_row;
  const int h = (int)(rest % p.H);
  rest /= p.H;
  const int t = (int)(rest % p.S);
  const int64_t b = rest / p.S;
  const int64_t slot = p.slots[b * p.s_sb + t];
  if (slot < 0 || slot >= p.places) return;
  const int64_t page = slot / p.page, at = slot - page * p.page;
  if (VEC) {
    const int d = c * 8;
    const u32x4 kk = ldg16(p.nk + b * p.nk_sb + h * p.nk_sh + t * p.nk_ss + d);
    const u32x4 vv = ldg16(p.nv + b * p.nv_sb + h * p.nv_sh + t * p.nv_ss + d);
    stg16(p.kp + page * p.kp_sp + h * p.kp_sh + at * p.kp_ss + d, kk);
    stg16(p.vp + page * p.vp_sp + h * p.vp_sh + at * p.vp_ss + d, vv);
  } else {
    p.kp[page * p.kp_sp + h * p.kp_sh + at * p.kp_ss + c] =
        p.nk[b * p.nk_sb + h * p.nk_sh + t * p.nk_ss + c * p.nk_sd];
    p.vp[page * p.vp_sp + h * p.vp_sh + at * p.vp_ss + c] =
        p.nv[b * p.nv_sb + h * p.nv_sh + t * p.nv_ss + c * p.nv_sd];
  }
}

// Sizes and pointers that reserve and trim have in common.
static int check_table(const char* what, const void* tables, const void* lengths, const void* free_pages,
                       const void* counters, int64_t B, int64_t columns, int64_t table_stride,
                       int64_t page_size, int64_t num_pages) {
  if (!tables || !lengths || !free_pages || !counters)
    return set_error(KF_EINVAL, "%s: null pointer", what);
  if (B <= 0 || columns <= 0 || page_size <= 0 || num_pages <= 0)
    return set_error(KF_EINVAL, "%s: all sizes must be positive", what);
  if (B > 1 && table_stride < columns)
    return set_error(KF_EINVAL, "%s: table rows of %lld entries overlap (stride %lld)", what, (long long)columns,
                     (long long)table_stride);
  if (page_size > 0x3fffffff / columns || B > 0x7fffffff / columns || num_pages > 0x3fffffff)
    return set_error(KF_EUNSUPPORTED, "%s: tables beyond 32-bit positions or page counts", what);
  return KF_OK;
}

static TableParams table_params(int32_t* tables, int32_t* lengths, int32_t* free_pages, int32_t* counters,
                                const int32_t* counts, int64_t count, int64_t B, int64_t columns,
                                int64_t table_stride, int64_t page_size, int64_t num_pages) {
  TableParams p{};
  p.tables = tables; p.lengths = lengths; p.free_pages = free_pages; p.counters = counters;
  p.counts = counts; p.count = count; p.t_sb = table_stride;
  p.B = (int)B; p.columns = (int)columns; p.page = (int)page_size; p.pages = (int)num_pages;
  return p;
}

}  // namespace kf

using namespace kf;

extern "C" int kf_page_reserve(int32_t* tables, int32_t* lengths, int32_t* free_pages, int32_t* counters,
                               const int32_t* counts, int64_t count, int64_t* slots, int64_t width, int64_t B,
                               int64_t columns, int64_t table_stride, int64_t page_size, int64_t num_pages,
                               void* stream) {
  const char* what = "kf_page_reserve";
  int rc = check_table(what, tables, lengths, free_pages, counters, B, columns, table_stride, page_size, num_pages);
  if (rc) return rc;
  if (slots == nullptr) return set_error(KF_EINVAL, "%s: slots is null", what);
  if (width <= 0 || width > 0x3fffffff) return set_error(KF_EINVAL, "%s: width must be positive", what);
  if (counts == nullptr && (count < 0 || count > width))
    return set_error(KF_EINVAL, "%s: %lld new tokens do not fit %lld slots a request", what, (long long)count,
                     (long long)width);
  TableParams p = table_params(tables, lengths, free_pages, counters, counts, count, B, columns, table_stride,
                               page_size, num_pages);
  p.slots = slots;
  p.width = width;
  hipLaunchKernelGGL(reserve_kernel, dim3(1), dim3(kTableThreads), 0, (hipStream_t)stream, p);
  return check_launch(what);
}

extern "C" int kf_page_trim(int32_t* tables, int32_t* lengths, int32_t* free_pages, int32_t* counters,
                            const int32_t* new_lengths, int64_t new_length, int64_t B, int64_t columns,
                            int64_t table_stride, int64_t page_size, int64_t num_pages, void* stream) {
  const char* what = "kf_page_trim";
  int rc = check_table(what, tables, lengths, free_pages, counters, B, columns, table_stride, page_size, num_pages);
  if (rc) return rc;
  if (new_lengths == nullptr && new_length < 0)
    return set_error(KF_EINVAL, "%s: the new length must not be negative", what);
  const TableParams p = table_params(tables, lengths, free_pages, counters, new_lengths, new_length, B, columns,
                                     table_stride, page_size, num_pages);
  hipLaunchKernelGGL(trim_kernel, dim3(1), dim3(kTableThreads), 0, (hipStream_t)stream, p);
  return check_launch(what);
}

extern "C" int kf_paged_append(void* k_pages, void* v_pages, const void* new_k, const void* new_v,
                               const int64_t* slots, int64_t B, int64_t H, int64_t Snew, int64_t D,
                               int64_t num_pages, int64_t page_size, int64_t slots_stride,
                               const int64_t* k_strides, const int64_t* v_strides, const int64_t* new_k_strides4,
                               const int64_t* new_v_strides4, int dtype, void* stream) {
  const char* what = "kf_paged_append";
  if (!k_pages || !v_pages || !new_k || !new_v || !slots) return set_error(KF_EINVAL, "%s: null pointer", what);
  if (!k_strides || !v_strides || !new_k_strides4 || !new_v_strides4)
    return set_error(KF_EINVAL, "%s: null strides", what);
  if (B <= 0 || H <= 0 || Snew <= 0 || D <= 0 || num_pages <= 0 || page_size <= 0)
    return set_error(KF_EINVAL, "%s: all sizes must be positive", what);
  if (dtype != KF_F16 && dtype != KF_BF16)
    return set_error(KF_EINVAL, "%s: dtype must be KF_F16 or KF_BF16", what);
  if (H > 0x7fffffff || Snew > 0x7fffffff || D > 0x7fffffff || page_size > 0x7fffffff || num_pages > 0x7fffffff)
    return set_error(KF_EUNSUPPORTED, "%s: dimension too large", what);
  StoreParams p{};
  p.kp = (uint16_t*)k_pages; p.vp = (uint16_t*)v_pages;
  p.nk = (const uint16_t*)new_k; p.nv = (const uint16_t*)new_v;
  p.slots = slots; p.s_sb = slots_stride;
  p.kp_sp = k_strides[0]; p.kp_sh = k_strides[1]; p.kp_ss = k_strides[2];
  p.vp_sp = v_strides[0]; p.vp_sh = v_strides[1]; p.vp_ss = v_strides[2];
  p.nk_sb = new_k_strides4[0]; p.nk_sh = new_k_strides4[1]; p.nk_ss = new_k_strides4[2]; p.nk_sd = new_k_strides4[3];
  p.nv_sb = new_v_strides4[0]; p.nv_sh = new_v_strides4[1]; p.nv_ss = new_v_strides4[2]; p.nv_sd = new_v_strides4[3];
  p.H = (int)H; p.S = (int)Snew; p.D = (int)D; p.page = (int)page_size;
  p.places = num_pages * page_size;
  bool vec = D % 8 == 0 && p.nk_sd == 1 && p.nv_sd == 1 && aligned16(k_pages) && aligned16(v_pages) &&
             aligned16(new_k) && aligned16(new_v);
  const int64_t s12[] = {p.kp_sp, p.kp_sh, p.kp_ss, p.vp_sp, p.vp_sh, p.vp_ss,
                         p.nk_sb, p.nk_sh, p.nk_ss, p.nv_sb, p.nv_sh, p.nv_ss};
  for (int64_t s : s12) vec = vec && (s % 8 == 0);
  p.total = B * H * Snew * (vec ? D / 8 : D);
  const int64_t blocks = (p.total + 255) / 256;
  if (blocks > 0x7fffffff) return set_error(KF_EUNSUPPORTED, "%s: grid too large", what);
  if (vec)
    hipLaunchKernelGGL((store_kernel<true>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, p);
  else
    hipLaunchKernelGGL((store_kernel<false>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, p);
  return check_launch(what);
}
