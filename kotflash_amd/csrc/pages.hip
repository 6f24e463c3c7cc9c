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
// Both are bound by latency: a step's call is a chain of two loads (lengths and
// counts, then pages) in one workgroup with one sum over the batch. Slots of
// whole prompts are megabytes of stores and get a workgroup per request first.
#include "kf_common.hpp"
#include "kf_host.hpp"

namespace kf {

// n / d for n < 2^31 by a multiplication (Granlund and Montgomery 1994): with
// 2^(s-1) < d <= 2^s, m = ceil(2^(31+s) / d) is exact for 31-bit n.
struct Divisor {
  uint32_t d, m;
  int shift;
};
static Divisor divisor(uint32_t d) {
  int s = 0;
  while ((1ull << s) < d) ++s;
  return {d, (uint32_t)(((1ull << (31 + s)) + d - 1) / d), 31 + s};
}
__device__ inline int quotient(int n, const Divisor& v) { return (int)(((uint64_t)(uint32_t)n * v.m) >> v.shift); }

struct TableParams {
  int32_t* tables;
  int32_t* lengths;
  int32_t* free_pages;
  int32_t* counters;
  const int32_t* counts;  // reserve: per request, or null: `count` each; trim: new lengths, likewise
  int64_t* slots;         // [B, width]; null: tables and slots have been written, only the state is left
  int count, width;
  int64_t t_sb;
  int B, columns, pages;
  Divisor page;
  Divisor row;            // width
};

// Inclusive sum over the TH threads, and their total. `sums` holds a value per
// wave; a turn's array must not be the one of the turn before.
struct Sums {
  int upto, total;
};
template <int TH>
__device__ inline Sums group_scan(int x, int* sums) {
  const int wave = wave_index();
  int s = wave_scan(x), total = 0;
  if ((threadIdx.x & 63) == 63) sums[wave] = s;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < TH / 64; ++w) {
    const int v = sums[w];
    s += w < wave ? v : 0;
    total += v;
  }
  return {s, total};
}

__device__ inline int pages_for(int tokens, const TableParams& p) { return quotient(tokens + (int)p.page.d - 1, p.page); }

__device__ inline int length_of(const TableParams& p, int raw) { return min(max(raw, 0), p.columns * (int)p.page.d); }

// The stack's height as far as it can be true.
__device__ inline int height(const TableParams& p) { return min(max(p.counters[0], 0), p.pages); }

// One request of a reserve: tokens before, tokens asked for, pages.
struct Demand {
  int len, count, first, need;
  bool fits;
};
__device__ inline Demand demand(const TableParams& p, int b) {
  Demand d;
  const int raw = p.lengths[b];
  d.count = p.counts ? p.counts[b] : p.count;
  d.len = length_of(p, raw);
  d.fits = d.count >= 0 && d.count <= p.width && d.len + (int64_t)d.count <= (int64_t)p.columns * p.page.d;
  d.first = pages_for(d.len, p);
  d.need = d.fits ? pages_for(d.len + d.count, p) - d.first : 0;
  return d;
}

// Slot of position pos of a request whose pages from `first` on lie on the
// stack from `top` down; -1 for a page outside the pool, which only a state that
// was written from outside can name.
__device__ inline int64_t slot_of(const TableParams& p, const int32_t* table, int pos, int first, int top) {
  const int col = quotient(pos, p.page);
  const int id = col < first ? table[col] : p.free_pages[top - (col - first)];
  return (uint32_t)id >= (uint32_t)p.pages ? -1 : (int64_t)id * p.page.d + (pos - col * (int)p.page.d);
}

// The request, of m, that item k belongs to: the last whose first item is not
// behind it. (Requests without items have their successor's first.)
__device__ inline int owner(const int* first, int m, int k) {
  int i = 0;
  for (int step = 1 << (31 - __builtin_clz(m)); step > 0; step >>= 1)
    if (i + step < m && first[i + step] <= k) i += step;
  return i;
}

constexpr int kOwnPages = 2;  // new (or returned) pages that a request's own thread handles

template <int TH>
__global__ __launch_bounds__(TH) void reserve_kernel(const TableParams p) {
  __shared__ int sums[2][TH / 64];
  __shared__ int len_s[TH], add_s[TH], first_s[TH], top_s[TH], rank_s[TH];
  __shared__ int taken_s, refused_s;
  const int tid = threadIdx.x;
  const int F = height(p);
  if (tid == 0) taken_s = refused_s = 0;
  int asked = 0;  // pages asked for by the requests of the turns before
  for (int b0 = 0, turn = 0; b0 < p.B; b0 += TH, ++turn) {
    const int b = b0 + tid;
    Demand d = {0, 0, 0, 0, false};
    if (b < p.B) d = demand(p, b);
    const Sums sum = group_scan<TH>(d.need, sums[turn & 1]);
    const int upto = asked + sum.upto;
    asked += sum.total;
    const bool served = d.fits && (d.need == 0 || upto <= F);
    const int top = F - 1 - (upto - d.need);  // place on the stack of its first new page
    if (served && d.need > 0) atomicMax(&taken_s, upto);
    if (b < p.B && !served) atomicAdd(&refused_s, 1);
    if (served) p.lengths[b] = d.len + d.count;
    if (p.slots == nullptr) continue;
    int32_t* table = p.tables + b * p.t_sb;
    if (served) {
#pragma unroll
      for (int i = 0; i < kOwnPages; ++i)
        if (i < d.need) table[d.first + i] = p.free_pages[top - i];
    }
    const int m = min(TH, p.B - b0);
    if (p.width == 1) {
      if (b < p.B) p.slots[b] = served && d.count ? slot_of(p, table, d.len, d.first, top) : -1;
      continue;
    }
    len_s[tid] = d.len;
    add_s[tid] = served ? d.count : -1;
    first_s[tid] = d.first;
    top_s[tid] = top;
    // More new pages: by their number in the turn, whichever request's.
    if (__syncthreads_or(served && d.need > kOwnPages)) {
      rank_s[tid] = sum.upto - d.need;
      __syncthreads();
      for (int k = tid; k < sum.total; k += TH) {
        const int i = owner(rank_s, m, k);
        if (add_s[i] >= 0) p.tables[(b0 + i) * p.t_sb + first_s[i] + k - rank_s[i]] = p.free_pages[top_s[i] - (k - rank_s[i])];
      }
    }
    for (int e = tid; e < m * p.width; e += TH) {
      const int i = quotient(e, p.row), t = e - i * p.width;
      p.slots[(int64_t)b0 * p.width + e] =
          t < add_s[i] ? slot_of(p, p.tables + (b0 + i) * p.t_sb, len_s[i] + t, first_s[i], top_s[i]) : -1;
    }
    __syncthreads();
  }
  __syncthreads();
  if (tid == 0) {
    p.counters[0] = F - taken_s;
    p.counters[1] = refused_s;
  }
}

// Tables and slots of request blockIdx.x before the state moves on: part
// blockIdx.y of its slots. Each workgroup sums the demand in front of it anew.
constexpr int kFillSlots = 2048;
__global__ __launch_bounds__(256) void fill_kernel(const TableParams p) {
  __shared__ int sums[4];
  const int tid = threadIdx.x, b = blockIdx.x;
  const int F = height(p);
  int before = 0;
  for (int i = tid; i < b; i += 256) before += demand(p, i).need;
  const Demand d = demand(p, b);
  before = group_scan<256>(before, sums).total;
  const bool served = d.fits && (d.need == 0 || before + d.need <= F);
  const int top = F - 1 - before;
  int32_t* table = p.tables + b * p.t_sb;
  if (served && blockIdx.y == 0)
    for (int i = tid; i < d.need; i += 256) table[d.first + i] = p.free_pages[top - i];
  int64_t* out = p.slots + (int64_t)b * p.width;
  const int t0 = blockIdx.y * kFillSlots, t1 = min(t0 + kFillSlots, p.width);
  for (int t = t0 + tid; t < t1; t += 256)
    out[t] = served && t < d.count ? slot_of(p, table, d.len + t, d.first, top) : -1;
}

template <int TH>
__global__ __launch_bounds__(TH) void trim_kernel(const TableParams p) {
  __shared__ int sums[2][TH / 64], all_s[TH / 64];
  __shared__ int from_s[TH], end_s[TH], rank_s[TH];
  const int tid = threadIdx.x;
  const int F = height(p);
  struct Cut {
    int keep, from, end;
  };
  auto cut = [&](int b) {
    const int raw = p.lengths[b], to = p.counts ? p.counts[b] : p.count;
    const int len = length_of(p, raw), keep = min(len, max(to, 0));
    return Cut{keep, pages_for(keep, p), pages_for(len, p)};
  };
  // Pages that come back in all: the first of them in the requests' order
  // ends on top of the stack. A batch of one turn learns it from the turn.
  int all = 0;
  if (p.B > TH) {
    for (int b = tid; b < p.B; b += TH) {
      const Cut c = cut(b);
      all += c.end - c.from;
    }
    all = group_scan<TH>(all, all_s).total;
  }
  int before = 0;
  for (int b0 = 0, turn = 0; b0 < p.B; b0 += TH, ++turn) {
    const int b = b0 + tid;
    Cut c = {0, 0, 0};
    if (b < p.B) c = cut(b);
    const Sums sum = group_scan<TH>(c.end - c.from, sums[turn & 1]);
    if (p.B <= TH) all = sum.total;
    const int top = F + all - 1;
    const int rank = before + sum.upto - (c.end - c.from);
    before += sum.total;
    auto give_back = [&](int32_t* entry, int32_t id, int place) {
      if (place >= 0 && place < p.pages) p.free_pages[place] = id;
      *entry = -1;
    };
    int32_t* table = p.tables + b * p.t_sb;
    if (b < p.B) p.lengths[b] = c.keep;
    from_s[tid] = c.from;
    end_s[tid] = c.end;
    rank_s[tid] = rank;
    const int m = min(TH, p.B - b0), base = before - sum.total;
    if (!__syncthreads_or(c.end - c.from > kOwnPages)) {
#pragma unroll
      for (int i = 0; i < kOwnPages; ++i)
        if (i < c.end - c.from) give_back(table + c.from + i, table[c.from + i], top - rank - i);
    } else if (sum.total <= 32 * m) {
      // By their number in the turn, whichever request's, four loads in flight.
      for (int k0 = tid; k0 < sum.total; k0 += 4 * TH) {
        int32_t* entry[4];
        int32_t id[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int k = min(k0 + j * TH, sum.total - 1);
          const int i = owner(rank_s, m, base + k);
          entry[j] = p.tables + (b0 + i) * p.t_sb + from_s[i] + base + k - rank_s[i];
          id[j] = *entry[j];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (k0 + j * TH < sum.total) give_back(entry[j], id[j], top - base - (k0 + j * TH));
      }
    } else {
      // Long rows: a wave per request, eight loads of a lane in flight.
      for (int i = wave_index(); i < m; i += TH / 64) {
        int32_t* row = p.tables + (b0 + i) * p.t_sb;
        const int from = from_s[i], end = end_s[i];
        for (int c0 = from + (tid & 63); c0 < end; c0 += 8 * 64) {
          int32_t id[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) id[k] = c0 + 64 * k < end ? row[c0 + 64 * k] : 0;
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (c0 + 64 * k < end) give_back(row + c0 + 64 * k, id[k], top - rank_s[i] - (c0 + 64 * k - from));
        }
      }
    }
    __syncthreads();
  }
  if (tid == 0) p.counters[0] = min(F + all, p.pages);
}

// Store of new K/V rows: pool[slot / page, h, slot % page] = new[b, h, t] for
// slot = slots[b, t], K and V, bit-exact; slots outside the pool are skipped.
// HBM-bound: each row is read once and written once. A thread moves 16 bytes
// of K and of V (one element where a layout does not allow it); more of them
// per thread measured slower (286 MB of prompts: 57.8 us with one, 65.4 with
// four, at a copy's rate 58). A workgroup's work items lie in one request.
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
  int64_t places;  // slots of the pool
  int items;       // work items of a request
  int blocks;      // workgroups of a request
  int H, page;
  Divisor per_row, heads;
};

// From this many bytes of new keys and values on, the stores are marked as not
// read again soon (a prompt's rows: 72 MB of them 33 us plain and 26 marked,
// 143 MB 58 and 56, 268 MB 104 and 105). A step's rows are read next.
constexpr int64_t kStreamStores = 64 << 20;

template <bool VEC, bool STREAM>
__global__ __launch_bounds__(256) void store_kernel(const StoreParams p) {
  const uint32_t b = blockIdx.x / (uint32_t)p.blocks;
  const int item = (int)(blockIdx.x - b * (uint32_t)p.blocks) * 256 + threadIdx.x;
  if (item >= p.items) return;
  const int row = quotient(item, p.per_row), c = item - row * (int)p.per_row.d;
  const int t = quotient(row, p.heads), h = row - t * p.H;
  const int64_t slot = p.slots[b * p.s_sb + t];
  if (slot < 0 || slot >= p.places) return;
  const int64_t page = slot / p.page, at = slot - page * p.page;
  if constexpr (VEC) {
    const int d = c * 8;
    const u32x4 kk = ldg16(p.nk + b * p.nk_sb + h * p.nk_sh + t * p.nk_ss + d);
    const u32x4 vv = ldg16(p.nv + b * p.nv_sb + h * p.nv_sh + t * p.nv_ss + d);
    u32x4* ko = reinterpret_cast<u32x4*>(p.kp + page * p.kp_sp + h * p.kp_sh + at * p.kp_ss + d);
    u32x4* vo = reinterpret_cast<u32x4*>(p.vp + page * p.vp_sp + h * p.vp_sh + at * p.vp_ss + d);
    if constexpr (STREAM) {
      __builtin_nontemporal_store(kk, ko);
      __builtin_nontemporal_store(vv, vo);
    } else {
      *ko = kk;
      *vo = vv;
    }
  } else {
    p.kp[page * p.kp_sp + h * p.kp_sh + at * p.kp_ss + c] =
        p.nk[b * p.nk_sb + h * p.nk_sh + t * p.nk_ss + c * p.nk_sd];
    p.vp[page * p.vp_sp + h * p.vp_sh + at * p.vp_ss + c] =
        p.nv[b * p.nv_sb + h * p.nv_sh + t * p.nv_ss + c * p.nv_sd];
  }
}

constexpr int64_t kOneGroupSlots = 2048, kSmallTables = 2048;

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
  p.row = divisor(1);
  p.tables = tables; p.lengths = lengths; p.free_pages = free_pages; p.counters = counters;
  p.counts = counts; p.count = (int)count; p.t_sb = table_stride;
  p.B = (int)B; p.columns = (int)columns; p.page = divisor((uint32_t)page_size); p.pages = (int)num_pages;
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
  p.width = (int)width;
  p.row = divisor((uint32_t)width);
  hipStream_t st = (hipStream_t)stream;
  // Many slots are written by many workgroups before one moves the state.
  // Measured with a trim before each, us in one workgroup and in two launches:
  // 1024 slots 7.1 and 9.4, 1280 8.6 and 9.7, 4096 10.0 to 11.8 and 9.4 to 9.9,
  // 8192 14.6 and 9.5, 512000 574 and 17.
  if (B * width > kOneGroupSlots) {
    const int64_t parts = (width + kFillSlots - 1) / kFillSlots;
    if (parts > 65535) return set_error(KF_EUNSUPPORTED, "%s: width too large", what);
    hipLaunchKernelGGL(fill_kernel, dim3((unsigned)B, (unsigned)parts), dim3(256), 0, st, p);
    if ((rc = check_launch(what))) return rc;
    p.slots = nullptr;
  }
  if (B <= 256) hipLaunchKernelGGL(reserve_kernel<256>, dim3(1), dim3(256), 0, st, p);
  else hipLaunchKernelGGL(reserve_kernel<1024>, dim3(1), dim3(1024), 0, st, p);
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
  // No request is longer than 2^30, which check_table sees to.
  const int64_t keep = new_length < 0x3fffffff ? new_length : 0x3fffffff;
  const TableParams p = table_params(tables, lengths, free_pages, counters, new_lengths, keep, B, columns,
                                     table_stride, page_size, num_pages);
  // More threads for larger tables, which may give back many pages at once
  // (64 requests of 512 tokens 14.2 us with 256, 12.2 with 1024; 256 of 5 8.2
  // and 8.7).
  if (B * columns <= kSmallTables) hipLaunchKernelGGL(trim_kernel<256>, dim3(1), dim3(256), 0, (hipStream_t)stream, p);
  else hipLaunchKernelGGL(trim_kernel<1024>, dim3(1), dim3(1024), 0, (hipStream_t)stream, p);
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
  if (H > 0x7fffffff || Snew > 0x7fffffff || D > 0x7fffffff || page_size > 0x7fffffff || num_pages > 0x7fffffff ||
      H * Snew > 0x7fffff00 / D)
    return set_error(KF_EUNSUPPORTED, "%s: dimension too large", what);
  StoreParams p{};
  p.kp = (uint16_t*)k_pages; p.vp = (uint16_t*)v_pages;
  p.nk = (const uint16_t*)new_k; p.nv = (const uint16_t*)new_v;
  p.slots = slots; p.s_sb = slots_stride;
  p.kp_sp = k_strides[0]; p.kp_sh = k_strides[1]; p.kp_ss = k_strides[2];
  p.vp_sp = v_strides[0]; p.vp_sh = v_strides[1]; p.vp_ss = v_strides[2];
  p.nk_sb = new_k_strides4[0]; p.nk_sh = new_k_strides4[1]; p.nk_ss = new_k_strides4[2]; p.nk_sd = new_k_strides4[3];
  p.nv_sb = new_v_strides4[0]; p.nv_sh = new_v_strides4[1]; p.nv_ss = new_v_strides4[2]; p.nv_sd = new_v_strides4[3];
  p.H = (int)H; p.page = (int)page_size;
  p.places = num_pages * page_size;
  bool vec = D % 8 == 0 && p.nk_sd == 1 && p.nv_sd == 1 && aligned16(k_pages) && aligned16(v_pages) &&
             aligned16(new_k) && aligned16(new_v);
  const int64_t s12[] = {p.kp_sp, p.kp_sh, p.kp_ss, p.vp_sp, p.vp_sh, p.vp_ss,
                         p.nk_sb, p.nk_sh, p.nk_ss, p.nv_sb, p.nv_sh, p.nv_ss};
  for (int64_t s : s12) vec = vec && (s % 8 == 0);
  const int64_t per_row = vec ? D / 8 : D;
  p.per_row = divisor((uint32_t)per_row);
  p.heads = divisor((uint32_t)H);
  p.items = (int)(H * Snew * per_row);
  p.blocks = (p.items + 255) / 256;
  const int64_t blocks = B * p.blocks;
  if (B > 0x7fffffff || blocks > 0x7fffffff) return set_error(KF_EUNSUPPORTED, "%s: grid too large", what);
  const dim3 grid((unsigned)blocks);
  hipStream_t st = (hipStream_t)stream;
  if (!vec) hipLaunchKernelGGL((store_kernel<false, false>), grid, dim3(256), 0, st, p);
  else if (B * H * Snew * D * 4 < kStreamStores) hipLaunchKernelGGL((store_kernel<true, false>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((store_kernel<true, true>), grid, dim3(256), 0, st, p);
  return check_launch(what);
}
