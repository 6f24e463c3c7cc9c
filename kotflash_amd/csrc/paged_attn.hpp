// Attention of a few new tokens per request over a paged K/V cache, gfx950.
//
//   O[b, h, i] = sum_j softmax_j(scale q[b, h, i] . K_b[j]) V_b[j],
//
// K_b[j] being row j % page of page tables[b, j / page] of the pool, j < L_b =
// lengths[b] (with `causal`, j < L_b - Sq + 1 + i: the Sq query tokens are the
// request's last). HBM-bound: every visible key and value is read once for all
// Hq / Hkv * Sq query rows that use it (about 2 FLOP per byte and row).
//
// How the work is cut. The lengths are known on the GPU only (a captured graph
// replays with others), so the launch cannot be planned on the host. All
// requests' keys are numbered in steps of 32 (64 in 8 bits): unit u = (request, KV head and
// row group of up to 64 packed query rows, step). A fixed number of workers, as
// many as the GPU holds at once, take equal runs of consecutive units, wherever
// requests begin and end in them: every worker streams the same number of bytes
// however the lengths differ, which a grid of (request, head, split) does not
// give.
//  * A worker finds its run from the lengths: a sum over the batch, and the
//    request in which the run begins.
//  * Within a run the part in one (request, row group) is a segment: S^T =
//    K Q^T, online softmax, O^T += V^T P^T on 16x16x32 MFMAs, as in the
//    contiguous decode. Two units are in flight in an LDS ring that
//    direct-to-LDS loads fill, across the ends of segments: short requests
//    stream like long ones.
//  * A worker is one wave per 16 packed rows (one, two or four). One wave needs
//    no barrier; more share the ring with two per unit.
//  * A segment that is a whole request writes O; others write an fp32 partial
//    (O, LSE) to slot worker + row group. Both numbers grow along the units
//    and one of them at every segment, so the slots are distinct, and those of
//    one row group are consecutive. The second launch merges them in order
//    (no atomics, same bits every time) and zeroes the rows that see nothing.
//  * A decoding step's new rows may be stored by the same launch (FUSED).
//
// What it reaches on MI355X (16 packed rows or fewer): 6.3 to 6.6 TB/s behind
// the first 8 us, which are two dependent launches and, in the first, a chain
// of loads; reading the same 4 KB pieces in random order without any of the
// work reaches 6.7 to 6.8.
//
// Pages: 16 rows of one page at a time have a buffer resource of their own,
// from a page number read by the scalar unit, with 64-bit bases (a pool may be
// larger than 4 GiB) and an extent that ends at the last visible row: rows
// behind it load as zeros, whatever the page holds there (NaN included), and a
// page number outside the pool reads nothing and its keys are masked.
//
// Pools in 8 bits (KV8) hold e4m3 codes, and a scale per 16 rows and head, a power
// of two. The codes stay codes through the LDS; a conversion that multiplies by
// the scale makes two 16-bit elements of them in front of the matrix units,
// exactly, so that the products, and what is rounded, are those of the 16-bit
// cache. A step has 64 keys, for the same bytes in flight. Half the bytes per
// key leave the scalar unit, which builds a resource per 16 rows and reads pages
// and scales, and the vector unit half the time for each key: 64 requests of 512
// to 8192 tokens (Hq=32 Hkv=8), 16-bit and 8-bit, D=128 185 and 103 us, D=64 99
// and 59: 6.2, 5.6, 5.8 and 5.0 TB/s. What is left at D=64 is the tail: equal runs
// end after 40 to 50 us, by where on the chip they are.
#pragma once
#include "decode_merge.hpp"
#include "fp8.hpp"
#include "kf_common.hpp"
#include "kf_host.hpp"

namespace kf {

// Read by the scalar unit: uniform addresses, never written by the launch.
#define KF_CONST __attribute__((address_space(4)))
typedef const int32_t KF_CONST* const_i32;

struct PagedParams {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* o;
  float* lse;
  float* part_o;    // [slots][rows][D]
  float* part_lse;  // [slots][rows]
  int32_t* parts;   // [B * heads][2]: first worker of a row group, its number of partials
  const int32_t* tables;
  const int32_t* lengths;
  int64_t t_sb;
  int64_t q_sb, q_sh, q_ss;
  int64_t k_sh, v_sh;            // per KV head
  uint32_t k_page, v_page;       // bytes of a page
  uint32_t k_row, v_row;         // bytes of a row
  int64_t o_sb, o_sh, o_ss;
  int B, Hq, Hkv, Sq, D, G;
  int pages, gpp;  // pages of the pool; 16-row groups per page
  int cap;         // tokens that a table has columns for
  int rows, nrb;   // packed rows per row group, row groups per KV head
  int heads;       // Hkv * nrb
  int workers;
  uint32_t q_bytes, o_bytes;  // extents of a KV head's queries and outputs
  int causal;
  float scale_log2;
  // Fused store (nnew > 0): the new rows [B, Hkv, nnew, D], B * nnew <=
  // KF_PAGED_STEP_SLOTS, and their slots.
  const uint16_t* nk;
  const uint16_t* nv;
  const int64_t* slots;
  int64_t s_sb;
  int64_t nk_sb, nk_sh, nk_ss;
  int64_t nv_sb, nv_sh, nv_ss;
  int nnew, page_size;
  uint32_t nnew_inv;  // 2^16 / nnew + 1
  // 8-bit pools: the blocks' scales, in pairs (K, V); bytes per page and head.
  const float* scales;
  uint32_t sc_page, sc_head;
  int row_rest;  // k_row without the row's own 16-byte pieces
};

// Direct-to-LDS loads (kf_common.hpp) of whole tiles: N loads of 1 KB, one
// per lane offset, to consecutive places from LDS address `to` on. A resource
// may have been written by the vector unit just before (a spilled scalar comes
// back by v_readlane), and a vector-memory instruction may read such a register
// five wait states later: hence the first, longer s_nop. The others separate
// the write of M0 from its use.
// STREAM: marked as read once (nt).
#define KF_FIRST(off, rsrc, nt) "s_nop 4\n\tbuffer_load_dwordx4 " off ", " rsrc ", 0 offen" nt " lds\n\t"
#define KF_NEXT(off, rsrc, nt) \
  "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tbuffer_load_dwordx4 " off ", " rsrc ", 0 offen" nt " lds\n\t"
#define KF_TILE1(nt) "s_mov_b32 m0, %0\n\t" KF_FIRST("%2", "%1", nt)
#define KF_TILE2(nt) KF_TILE1(nt) KF_NEXT("%3", "%1", nt)
#define KF_TILE3(nt) KF_TILE2(nt) KF_NEXT("%4", "%1", nt)
#define KF_TILE4(nt) KF_TILE3(nt) KF_NEXT("%5", "%1", nt)
template <int N, bool STREAM>
__device__ inline void dma_tile(__amdgpu_buffer_rsrc_t r, uint32_t to, const uint32_t* off) {
  static_assert(N >= 1 && N <= 4);
  const uint32_t m0 = __builtin_amdgcn_readfirstlane(to);
#define KF_EMIT(text, ...)                                                                        \
  do {                                                                                            \
    if constexpr (STREAM) asm volatile(text(" nt") : : "s"(m0), "s"(r), __VA_ARGS__ : "memory", "m0", "scc"); \
    else asm volatile(text("") : : "s"(m0), "s"(r), __VA_ARGS__ : "memory", "m0", "scc");         \
  } while (0)
  if constexpr (N == 1) KF_EMIT(KF_TILE1, "v"(off[0]));
  else if constexpr (N == 2) KF_EMIT(KF_TILE2, "v"(off[0]), "v"(off[1]));
  else if constexpr (N == 3) KF_EMIT(KF_TILE3, "v"(off[0]), "v"(off[1]), "v"(off[2]));
  else KF_EMIT(KF_TILE4, "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]));
#undef KF_EMIT
}

// Keys per unit: 16 KB of K and V at D = 128 either way.
template <bool KV8>
constexpr int kStepOf = KV8 ? 64 : 32;

// K/V bytes of a call from which its loads are marked as read once. Such loads
// do not go through the 256 MB memory-side cache, which costs the others a
// tenth of their rate (us, plain and marked, three sets of inputs in turn: 1158
// MB 205 and 185, 537 MB 99 and 89, 300 MB 65 and 59, 294 MB 60 and 54); but a
// call of which the cache still holds a part from the last time is faster plain
// (59 MB 19.9 and 20.8). The kernel counts what all row groups load: measured
// with one, where nothing is read twice.
constexpr int64_t kStreamBytes = 128 << 20;

__device__ inline int wave_sum(int x) { return __builtin_amdgcn_readlane(wave_scan(x), 63); }

__device__ inline int visible(const PagedParams& p, int len) { return min(max(len, 0), p.cap); }
template <int STEP>
__device__ inline int lane_steps(const PagedParams& p, int b) {
  return b < p.B ? (visible(p, p.lengths[b]) + STEP - 1) / STEP : 0;
}
// Steps (of one head) of the requests from b0 on.
template <int STEP>
__device__ inline int steps_from(const PagedParams& p, int b0, int lane) {
  int n = 0;
  for (; b0 < p.B; b0 += 64) n += lane_steps<STEP>(p, b0 + lane);
  return wave_sum(n);
}
// Units per worker.
__device__ inline int run_length(const PagedParams& p, int total) {
  return (total * p.heads + p.workers - 1) / p.workers;
}

// A unit: a step of row group hh of request b, with `rem` keys of the request
// from its first on. begin: 1 if a segment begins with it, 2 if that is the
// row group's first step.
struct Unit {
  int b, hh, rem, begin;
};

// Whether any of eight elements is infinite or NaN (all exponent bits set).
template <typename T>
__device__ inline bool any_nonfinite(u32x4 x) {
  constexpr uint32_t kExp = std::is_same_v<T, _Float16> ? 0x7c00u : 0x7f80u;
  bool bad = false;
#pragma unroll
  for (int j = 0; j < 4; ++j) bad |= (x[j] & kExp) == kExp || (x[j] >> 16 & kExp) == kExp;
  return bad;
}

// i / nnew of a new row's number: exact, as i < 2^8 and nnew <= 2^4.
template <typename P>
__device__ inline int new_row_request(const P& c, int i) { return (int)((uint32_t)i * c.nnew_inv >> 16); }

template <typename T> struct PBias;  // P = 2^(s - m + bias), see paged_kernel
template <> struct PBias<_Float16> { static constexpr float v = 7.f; };
template <> struct PBias<__bf16> { static constexpr float v = 0.f; };

// 1 KB loads of the Q tile of 16 rows.
constexpr int q_loads(int DT) { return 16 * (DT / 8) / 64; }
// LDS of a worker: two steps of K and V, and every wave's Q tiles of two
// segments.
constexpr int worker_lds(int DT, int NW) { return 2 * (2 * 64 * DT + NW * q_loads(DT) * 1024); }
// Workers that a CU holds: by its 160 KB of LDS, given out in pieces of 1280
// bytes, and by waves (two per SIMD, four of four-wave workers: 16 requests up
// to 16384 tokens, 8 KV heads, D=64, us with 8, 12 and 16 waves: 32 rows 58.2,
// 61.6 and 61.4, 64 rows 89.4, 77.1 and 72.6; D=128 is bound by the LDS).
// In 8 bits the two-wave ones up to three per SIMD (32 rows 52.0 and 48.7; D=128 is
// bound by the LDS there too).
constexpr int workers_per_cu(int DT, int NW, bool kv8) {
  const int by_lds = 160 * 1024 / ((worker_lds(DT, NW) + 1279) / 1280 * 1280);
  const int by_waves = NW == 4 ? 4 : NW == 2 && kv8 ? 6 : 8 / NW;
  return by_lds < by_waves ? by_lds : by_waves;
}

// All waves of a worker are here, and what they have written or read in LDS is
// behind them. (Each waits for its own loads and reads before.)
template <int NW>
__device__ inline void worker_barrier() {
  if constexpr (NW > 1) asm volatile("s_barrier" ::: "memory");
}

// NW waves per worker, 16 packed rows each: they share the ring, every wave
// loading a part of each step, and read all of it. FUSED: with the store of new
// rows (in one kernel it costs calls without any up to 0.2 us, for scalars that
// no longer fit the registers).
enum PoolKind { kPool16, kPool8, kPool8Padded };  // 16 bits; e4m3 codes; rows with padding
template <typename T, int DT, int NW, bool FUSED, PoolKind POOL>
__global__ __launch_bounds__(64 * NW, (workers_per_cu(DT, NW, POOL != kPool16) * NW + 3) / 4) void paged_kernel(const PagedParams p) {
  constexpr bool KV8 = POOL != kPool16;
  constexpr int STEP = kStepOf<KV8>;
  constexpr int GROUPS = STEP / 16;   // 16-row groups of a step
  constexpr int EB = KV8 ? 1 : 2;     // bytes of an element of K and V
  constexpr int QCPR = DT / 8;        // 16-byte chunks per row of Q
  constexpr int CPR = DT * EB / 16;   // and of K and V
  constexpr int NDC = DT / 32;        // 32-wide head-dim chunks (S contraction)
  constexpr int NDB = DT / 16;        // 16-wide head-dim blocks of O^T
  constexpr int VT = STEP * DT * EB / 2;  // half-words of one K (or V) step tile
  constexpr int NGI = 16 * CPR / 64;  // 1 KB loads per 16-row group of K (or V)
  constexpr int NL = 2 * GROUPS * NGI / NW;  // a wave's loads per step
  constexpr int NQ = q_loads(DT);
  using Tile = SwizzledTile<CPR>;
  using QTile = SwizzledTile<QCPR>;
  using Store = std::conditional_t<KV8, uint8_t, uint16_t>;
  static_assert(NW == 1 || NW == 2 || NW == 4);
  static_assert(!KV8 || (!FUSED && DT % 64 == 0));
  // Two ring slots of a step's K and V tiles; per slot and wave, the Q tile of
  // the segment that begins with it.
  __shared__ __attribute__((aligned(16))) uint16_t smem[worker_lds(DT, NW) / 2];

  const int lane = threadIdx.x & 63, wave = NW > 1 ? wave_index() : 0;
  const int l16 = lane & 15, g16 = lane >> 4;
  const const_i32 lengths = (const_i32)(uintptr_t)p.lengths;

  // The first 64 requests' lengths. What does not depend on them is computed
  // while they are on their way: a short call is one chain of loads (lengths,
  // pages, keys), 5 us of it in this kernel.
  const int raw0 = p.lengths[min(lane, p.B - 1)];

  // The parameters that only the ends of segments need are read again there:
  // the scalar registers do not hold them all, and spilled ones cost vector
  // instructions in every step. (The empty asm keeps the compiler from reading
  // them once.)
  auto cold = [&]() -> const PagedParams KF_CONST& {
    auto ptr = (const PagedParams KF_CONST*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(ptr));
    return *ptr;
  };
  // The fused store. A new row may be read by any request whose table leads to
  // its slot, at any position, and no order between the workers says who is
  // first. So every worker that reads 16 rows of a page first writes the new rows
  // among them itself (store_hits), all of them the same bytes, and none waits
  // for another. For that each wave keeps the 16-row groups of the call's slots:
  // slot i's in lane i % 64 of register i / 64, -1 where it is outside the pool.
  // Rows that nobody reads are stored by the loop below, which has every row
  // once, shared out from the last wave, idle in a short call, to the first.
  int fresh[KF_PAGED_STEP_SLOTS / 64] = {-1, -1, -1, -1};
  static_assert(KF_PAGED_STEP_SLOTS == 4 * 64);
  auto put_row = [&](const auto& c, int i, int kvh, uint64_t kbase, uint64_t vbase) {  // by 16 lanes
    const int ch = lane & 15;
    if (ch * 8 >= c.D) return;
    const int b = new_row_request(c, i), t = i - b * c.nnew;
    const int64_t slot = c.slots[b * c.s_sb + t];
    const u32x4 kk = ldg16(c.nk + b * c.nk_sb + kvh * c.nk_sh + t * c.nk_ss + ch * 8);
    const u32x4 vv = ldg16(c.nv + b * c.nv_sb + kvh * c.nv_sh + t * c.nv_ss + ch * 8);
    if (slot < 0 || slot >= (int64_t)c.pages * c.page_size) return;
    const uint32_t id = (uint32_t)slot / (uint32_t)c.page_size, at = (uint32_t)slot - id * (uint32_t)c.page_size;
    stg16((char*)(uintptr_t)kbase + (uint64_t)id * c.k_page + (uint64_t)at * c.k_row + ch * 16, kk);
    stg16((char*)(uintptr_t)vbase + (uint64_t)id * c.v_page + (uint64_t)at * c.v_row + ch * 16, vv);
  };
  if constexpr (FUSED) {
    const auto& c = cold();
    const int rows = c.B * c.nnew;
    int64_t slot[4];  // all on their way at once
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = min(64 * k + lane, rows - 1), b = new_row_request(c, i);
      slot[k] = c.slots[b * c.s_sb + i - b * c.nnew];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      fresh[k] = 64 * k + lane < rows && slot[k] >= 0 && slot[k] < (int64_t)c.pages * c.page_size ? (int)slot[k] >> 4 : -1;
    const uint32_t all = (uint32_t)rows * (uint32_t)c.Hkv;  // at most 2^30: B Hkv <= kMergeRows
    for (uint32_t e = ((uint32_t)(c.workers - 1 - (int)blockIdx.x) * NW + wave) * 4 + (lane >> 4); e < all;
         e += (uint32_t)c.workers * NW * 4) {
      const int kvh = (int)(e / (uint32_t)rows);
      put_row(c, (int)(e - (uint32_t)kvh * rows), kvh, (uint64_t)(uintptr_t)(c.k + kvh * c.k_sh),
              (uint64_t)(uintptr_t)(c.v + kvh * c.v_sh));
    }
  }

  // Per-lane plan of a group's loads: this lane's 16-byte chunk within the 16
  // rows (kOOB for head-dim padding). The swizzle key has a period of 16 rows,
  // so both groups of a step share it.
  uint32_t koff[NGI], voff[NGI];
#pragma unroll
  for (int k = 0; k < NGI; ++k) {
    const int pc = k * 64 + lane;
    const int r = pc / CPR;
    const int c = (pc % CPR) ^ Tile::key(r);
    const bool ok = c * 16 < EB * p.D;
    koff[k] = ok ? (uint32_t)r * p.k_row + c * 16u : kOOB;
    voff[k] = ok ? (uint32_t)r * p.v_row + c * 16u : kOOB;
  }
  // The wave's Q loads and its lane's row, for the first row group of a
  // KV head (of most, the only one).
  auto query_offset = [&](const auto& c, int k, int rb) -> uint32_t {
    const int pc = k * 64 + lane;
    const int r = wave * 16 + pc / QCPR;
    const int ch = (pc % QCPR) ^ QTile::key(pc / QCPR);
    const int rho = rb * c.rows + r;
    const int g = rho / c.Sq, i = rho - g * c.Sq;
    const bool ok = r < c.rows && rho < c.G * c.Sq && ch * 8 < c.D;
    return ok ? (uint32_t)(g * c.q_sh + i * c.q_ss + ch * 8) * 2u : kOOB;
  };
  struct Row {
    uint32_t out;  // byte offset of the row within its KV head's outputs, kOOB if there is none
    int lag;       // keys that it sees fewer than the last query token does
  };
  auto output_row = [&](const auto& c, int rb) -> Row {
    const int r = wave * 16 + l16, rho = rb * c.rows + r;
    const int g = rho / c.Sq, i = rho - g * c.Sq;
    return {r < c.rows && rho < c.G * c.Sq ? (uint32_t)(g * c.o_sh + i * c.o_ss) * 2u : kOOB,
            c.causal ? c.Sq - 1 - i : 0};
  };
  uint32_t qoff[NQ];
#pragma unroll
  for (int k = 0; k < NQ; ++k) qoff[k] = query_offset(p, k, 0);
  const Row row0 = output_row(p, 0);

  // This worker's run of units, and where it begins: request b, whose first
  // unit is `start`.
  const int worker = blockIdx.x;
  const int len0 = lane < p.B ? visible(p, raw0) : 0;
  const int mine0 = (len0 + STEP - 1) / STEP;
  const int sum0 = wave_scan(mine0);
  int total = __builtin_amdgcn_readlane(sum0, 63);
  if (p.B > 64) total += steps_from<STEP>(p, 64, lane);
  const int run = run_length(p, total);
  const int u = worker * run;
  if (u >= total * p.heads) return;  // more workers than runs
  const int count = min(run, total * p.heads - u);
  Unit at;  // the next one to load
  int len, start;
  uint64_t past = __builtin_amdgcn_ballot_w64(sum0 * p.heads > u);
  if (past) {
    at.b = __builtin_ctzll(past);
    len = __builtin_amdgcn_readlane(len0, at.b);
    start = (__builtin_amdgcn_readlane(sum0, at.b) - __builtin_amdgcn_readlane(mine0, at.b)) * p.heads;
  } else {
    start = __builtin_amdgcn_readlane(sum0, 63) * p.heads;
    for (at.b = 64;; at.b += 64) {
      const int mine = lane_steps<STEP>(p, at.b + lane) * p.heads;
      const int sum = wave_scan(mine);
      past = __builtin_amdgcn_ballot_w64(start + sum > u);
      if (past) {
        const int i = __builtin_ctzll(past);
        start += __builtin_amdgcn_readlane(sum, i) - __builtin_amdgcn_readlane(mine, i);
        at.b += i;
        break;
      }
      start += __builtin_amdgcn_readlane(sum, 63);
    }
    len = visible(p, lengths[at.b]);
  }
  const int n0 = (len + STEP - 1) / STEP;
  at.hh = (u - start) / n0;
  const int s0 = (u - start) - at.hh * n0;
  at.rem = len - STEP * s0;
  at.begin = s0 == 0 ? 2 : 1;
  // Its first 16-row group: column of the table, group of that page.
  int column = GROUPS * s0 / p.gpp, part = GROUPS * s0 - column * p.gpp;

  const uint32_t lds0 = lds_addr(smem);
  const bool stream = (int64_t)total * p.heads * (STEP * 2 * EB * p.D) > kStreamBytes;

  // Of the request and head under way at `at`.
  const_i32 table;
  uint64_t kh, vh, sh;
  auto head_base = [&](const auto& c) {
    const int kvh = at.hh / c.nrb;
    kh = (uint64_t)(uintptr_t)((const Store*)c.k + kvh * c.k_sh);
    vh = (uint64_t)(uintptr_t)((const Store*)c.v + kvh * c.v_sh);
    if constexpr (KV8) sh = (uint64_t)(uintptr_t)c.scales + (uint64_t)kvh * c.sc_head;
  };
  auto table_base = [&](const auto& c) {
    table = (const_i32)(uintptr_t)(c.tables + at.b * c.t_sb);
  };
  table_base(p);
  head_base(p);
  // Pages of the groups of unit `at`, the last visible one's where a group is
  // not visible. They are read by the scalar unit one unit before they are needed.
  int page[GROUPS], row1;
  auto look_up = [&] {
    if constexpr (KV8) {
      int col = column, q = part;
      page[0] = table[(uint32_t)col];
#pragma unroll
      for (int g = 1; g < GROUPS; ++g) {
        if (++q == p.gpp) q = 0, col += at.rem > 16 * g;
        page[g] = table[(uint32_t)col];
      }
      return;
    }
    const bool same = part + 1 < p.gpp;
    row1 = same ? (part + 1) * 16 : 0;
    page[0] = table[(uint32_t)column];
    page[1] = table[(uint32_t)(same || at.rem <= 16 ? column : column + 1)];
  };
  look_up();
  // `at` to the unit behind: next step, row group, or request that holds keys.
  auto advance = [&] {
    at.rem -= STEP;
    if (at.rem > 0) {
      at.begin = 0;
      part += GROUPS;
#pragma unroll
      for (int g = 0; g < GROUPS; ++g)
        if (part >= p.gpp) part -= p.gpp, ++column;
      return;
    }
    at.begin = 2;
    column = part = 0;
    const auto& c = cold();
    if (++at.hh == c.heads) {
      at.hh = 0;
      do {
        if (++at.b == c.B) return;  // behind the last unit
        len = min(max(((const_i32)(uintptr_t)c.lengths)[at.b], 0), c.cap);
      } while (len == 0);
      table_base(c);
    }
    at.rem = len;
    head_base(c);
  };

  // What is in the ring slots: the unit, and the visible rows of its groups (0
  // for a page outside the pool). KV8: whether each group's page is in the pool,
  // and its scales, which the scalar unit reads with the unit's loads.
  Unit held[2] = {at, at};
  int seen[2][2] = {{0, 0}, {0, 0}};
  int valid[2] = {0, 0};
  f32x2 scale8[2][GROUPS] = {};
  auto seen_of = [&](const Unit& w, int slot, int g) -> int {
    if constexpr (KV8) return valid[slot] >> g & 1 ? min(max(w.rem - 16 * g, 0), 16) : 0;
    else return seen[slot][g];
  };
  // The new rows in the two groups of unit `at`, to their slots before the
  // unit's loads, four at a time. Few units have any; those wait for their
  // stores. Against the store in a launch of its own, us for both: 1 to 8 short
  // requests 9.8 and 11.5, 64 of up to 500 tokens 10.8 and 12.4, but 294 MB over
  // 32 requests 57.1 and 56.1, 64 requests of 4 drafts 70.5 and 65.7, 16 of 16
  // 23.0 and 20.6.
  auto store_hits = [&] {
    const int g0 = (uint32_t)page[0] < (uint32_t)p.pages ? page[0] * p.gpp + part : -2;
    const int g1 = (uint32_t)page[1] < (uint32_t)p.pages ? page[1] * p.gpp + row1 / 16 : -2;
    uint32_t off = ~0u;
#pragma unroll
    for (int f : fresh) off = min(off, min((uint32_t)(f ^ g0), (uint32_t)(f ^ g1)));
    if (!wave_any(off == 0)) return;
    const auto& c = cold();
    const int kvh = at.hh / c.nrb;
#pragma unroll
    for (int k = 0; k < KF_PAGED_STEP_SLOTS / 64; ++k) {
      uint64_t hits = __builtin_amdgcn_ballot_w64(fresh[k] == g0 || fresh[k] == g1);
      while (hits) {
        int mine = -1;
        for (int s = 0; s < 4 && hits; ++s, hits &= hits - 1)
          if (lane >> 4 == s) mine = __builtin_ctzll(hits);
        if (mine >= 0) put_row(c, 64 * k + mine, kvh, kh, vh);
      }
    }
    KF_WAIT_VMCNT(0);
  };
  // Loads of unit `at` into a slot: the Q tile if a segment begins, then K and
  // V. All of the kernel's loads from here on are direct-to-LDS, so that the
  // explicit waits below are the only ones.
  auto issue = [&](bool more, auto slot_c) {
    constexpr int slot = decltype(slot_c)::value;
    const uint32_t kv0 = lds0 + slot * 2 * VT * 2;
    if constexpr (FUSED) store_hits();
    if (at.begin) {
      const auto& c = cold();
      const int kvh = at.hh / c.nrb;
      const int rb = at.hh - kvh * c.nrb;
      const auto qr = make_rsrc(c.q + at.b * c.q_sb + (int64_t)kvh * c.G * c.q_sh, c.q_bytes);
      const uint32_t q0 = lds0 + 4 * VT * 2 + (slot * NW + wave) * NQ * 1024u;
      if (rb == 0) {
        dma_tile<NQ, false>(qr, q0, qoff);
      } else {
        uint32_t off[NQ];
#pragma unroll
        for (int k = 0; k < NQ; ++k) off[k] = query_offset(c, k, rb);
        dma_tile<NQ, false>(qr, q0, off);
      }
    }
    if constexpr (KV8) {
      // K and V have the same strides, and the scalar unit, which has twice the
      // groups of a 16-bit step to look after, computes a group's offset once.
      uint32_t id[GROUPS], row[GROUPS];
      int left[GROUPS];  // visible rows from the group on
      int q = part, ok = 0;
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        id[g] = __builtin_amdgcn_readfirstlane(page[g]);
        const bool in = id[g] < (uint32_t)p.pages;
        ok |= (int)in << g;
        id[g] = in ? id[g] : 0;
        left[g] = in ? at.rem - 16 * g : 0;
        row[g] = q * 16;
        q = q + 1 == p.gpp ? 0 : q + 1;
        scale8[slot][g] = *(const f32x2 KF_CONST*)(sh + (uint64_t)(id[g] * p.sc_page + row[g] / 2));
      }
      valid[slot] = ok;
      // One wave loads all groups; of two, each every other; of four, K or V of
      // those. The extent ends with the last visible row; none of a page outside
      // the pool is.
      const int odd = wave & 1;
      auto send = [&](auto nt) {
#pragma unroll
        for (int j = 0; j < (NW > 1 ? GROUPS / 2 : GROUPS); ++j) {
          const int g = NW > 1 ? 2 * j : j, mine = NW > 1 ? g + odd : g;
          const uint32_t i = NW > 1 && odd ? id[g + 1] : id[g], r = NW > 1 && odd ? row[g + 1] : row[g];
          // A page's rows may be more than 4 GiB apart, where pages lie inside
          // a position's; 16 of them are less than 2.
          const uint64_t off = (uint64_t)i * p.k_page + (uint64_t)r * p.k_row;
          // (Not a clamp to 0 as well: that is a vector instruction, and a
          // resource is in scalar registers.)
          const int rows = min(NW > 1 && odd ? left[g + 1] : left[g], 16);
          const uint32_t extent = rows > 0 ? (uint32_t)rows * p.k_row - (uint32_t)p.row_rest : 0u;
          const uint32_t m0 = kv0 + mine * 16 * DT;
          if (NW < 4) {
            dma_tile<NGI, decltype(nt)::value>(make_rsrc((const void*)(uintptr_t)(kh + off), extent), m0, koff);
            dma_tile<NGI, decltype(nt)::value>(make_rsrc((const void*)(uintptr_t)(vh + off), extent), m0 + VT * 2, koff);
          } else {
            const uint64_t base = wave < 2 ? kh : vh;
            dma_tile<NGI, decltype(nt)::value>(make_rsrc((const void*)(uintptr_t)(base + off), extent),
                                               m0 + (wave < 2 ? 0 : VT * 2), koff);
          }
        }
      };
      if (stream) send(std::true_type{});
      else send(std::false_type{});
    }
#pragma unroll
    for (int g = 0; g < (KV8 ? 0 : GROUPS); ++g) {
      const uint32_t m0 = kv0 + g * 16 * DT * EB;
      const uint32_t id = __builtin_amdgcn_readfirstlane(page[g]);
      const int row = g == 0 ? part * 16 : row1;
      int rows = at.rem - 16 * g;
      rows = rows < 0 || id >= (uint32_t)p.pages ? 0 : rows < 16 ? rows : 16;
      seen[slot][g] = rows;
      // One wave loads both groups; of two, each a group; of four, K or V of one.
      if (NW > 1 && (wave & 1) != g) continue;
      // The extent ends with the last visible row.
      if (NW < 4 || wave < 2) {
        const uint64_t ka = kh + (rows ? (uint64_t)id * p.k_page + (uint32_t)row * (uint64_t)p.k_row : 0);
        const auto kr = make_rsrc((const void*)(uintptr_t)ka, rows ? (rows - 1) * p.k_row + EB * p.D : 0);
        if (stream) dma_tile<NGI, true>(kr, m0, koff);
        else dma_tile<NGI, false>(kr, m0, koff);
      }
      if (NW < 4 || wave >= 2) {
        const uint64_t va = vh + (rows ? (uint64_t)id * p.v_page + (uint32_t)row * (uint64_t)p.v_row : 0);
        const auto vr = make_rsrc((const void*)(uintptr_t)va, rows ? (rows - 1) * p.v_row + EB * p.D : 0);
        if (stream) dma_tile<NGI, true>(vr, m0 + VT * 2, voff);
        else dma_tile<NGI, false>(vr, m0 + VT * 2, voff);
      }
    }
    held[slot] = at;
    if (more) {
      advance();
      look_up();
    }
  };

  // The segment under way.
  u32x4 qf[NDC];    // Q rows as MFMA B operands: lane l = the wave's row l % 16
  f32x4 oacc[NDB];  // O^T: lane l, register r = head dim 16 db + 4 (l / 16) + r of row l % 16
  float m_i, l_i;
  Row row;          // this lane's
  const int most_lag = p.causal ? p.Sq - 1 : 0;
  bool from_start = false;  // whether it began with the row group's first step

  auto begin_segment = [&](const Unit& w, auto slot_c) {
    constexpr int slot = decltype(slot_c)::value;
    const uint16_t* qs = smem + 4 * VT + (slot * NW + wave) * NQ * 512;
    const auto& c = cold();
    const int rb = w.hh % c.nrb;
    from_start = w.begin == 2;
#pragma unroll
    for (int dc = 0; dc < NDC; ++dc) {
      // KV8: a 16-byte read of K holds two chunks' slots (below).
      const int ch = KV8 ? 8 * (dc / 2) + 2 * g16 + dc % 2 : 4 * dc + g16;
      qf[dc] = lds_read16(qs + QTile::chunk(l16, ch) * 8);
    }
    m_i = kNegInf;
    l_i = 0.f;
    row = row0;
    if (rb > 0) row = output_row(c, rb);
#pragma unroll
    for (int db = 0; db < NDB; ++db) oacc[db] = f32x4{0.f, 0.f, 0.f, 0.f};
  };

  auto step = [&](const Unit& w, auto slot_c) {
    constexpr int slot = decltype(slot_c)::value;
    const uint16_t* Ks = smem + slot * 2 * VT;
    const uint16_t* Vs = Ks + VT;
    // K rows as MFMA A operands: lane = key kb * 16 + l % 16, slots = head dims.
    // KV8: odd groups with their halves of eight rows exchanged, so that the
    // transposed reads of V below take their rows from eight different pairs of
    // both parities; 16 codes per read, the first eight for one product, the
    // others for the next.
    constexpr int NKA = KV8 ? NDC / 2 : NDC;
    u32x4 ka[GROUPS][NKA];
#pragma unroll
    for (int kb = 0; kb < GROUPS; ++kb)
#pragma unroll
      for (int dc = 0; dc < NKA; ++dc) {
        const int key = kb * 16 + (KV8 && kb % 2 ? l16 ^ 8 : l16);
        ka[kb][dc] = lds_read16(Ks + Tile::chunk(key, 4 * dc + g16) * 8);
        // The second half of a row's last piece: any codes, NaN among them,
        // which zeros of Q do not silence.
        if (POOL == kPool8Padded && 4 * dc + g16 == p.D / 16) ka[kb][dc][2] = ka[kb][dc][3] = 0;
      }
    bool masked;
    if constexpr (KV8) masked = valid[slot] != (1 << GROUPS) - 1 || w.rem - most_lag < STEP;
    else masked = seen[slot][0] + seen[slot][1] < STEP || w.rem - most_lag < STEP;
    // S^T: lane l, register r = key kb * 16 + key_of(kb) + r of row l % 16.
    auto key_of = [&](int kb) -> int { return KV8 && kb % 2 ? (4 * g16) ^ 8 : 4 * g16; };
    f32x4 sc[GROUPS];
#pragma unroll
    for (int kb = 0; kb < GROUPS; ++kb) {
      sc[kb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int dc = 0; dc < NDC; ++dc) {
        if constexpr (KV8) {
          const u32x4 codes = ka[kb][dc / 2];
          const uint32_t lo = codes[dc % 2 * 2], hi = codes[dc % 2 * 2 + 1];
          const float s = scale8[slot][kb][0];
          const u32x4 a = {dequantise2<T, false>(lo, s), dequantise2<T, true>(lo, s),
                           dequantise2<T, false>(hi, s), dequantise2<T, true>(hi, s)};
          sc[kb] = Elem<T>::mfma16(a, qf[dc], sc[kb]);
        } else {
          sc[kb] = Elem<T>::mfma16(ka[kb][dc], qf[dc], sc[kb]);
        }
      }
      sc[kb] *= p.scale_log2;
    }
    // Masked after the scale, so that a scale of zero leaves -inf.
    if (masked) {
      // A group without visible rows has codes of zero; its block's scale may be
      // anything (never written, or that of another request's page): 0 V.
      if constexpr (KV8) {
#pragma unroll
        for (int g = 0; g < GROUPS; ++g)
          if (seen_of(w, slot, g) == 0) scale8[slot][g][1] = 1.f;
      }
#pragma unroll
      for (int kb = 0; kb < GROUPS; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int c = key_of(kb) + r;
          const bool in = c < seen_of(w, slot, kb) && 16 * kb + c < w.rem - row.lag;
          sc[kb][r] = in ? sc[kb][r] : kNegInf;
        }
    }
    float mx = kNegInf;
#pragma unroll
    for (int kb = 0; kb < GROUPS; ++kb)
#pragma unroll
      for (int r = 0; r < 4; ++r) mx = fmaxf(mx, sc[kb][r]);
    mx = wave_group16_max(mx);
    if (m_i == kNegInf) {
      m_i = mx;
    } else {
      const bool grow = mx > m_i + kRescaleThreshold;
      if (wave_any(grow)) {
        const float alpha = grow ? fast_exp2(m_i - mx) : 1.f;
        l_i *= alpha;
#pragma unroll
        for (int db = 0; db < NDB; ++db) oacc[db] *= alpha;
        m_i = grow ? mx : m_i;
      }
    }
    // P in 16 bits for the second product, which takes its operands so: the
    // output's error is 1.2 to 1.4 times that of P in fp32 (fp16 2.9e-4, bf16
    // 2.3e-3 relative). With m up to 8 below the maximum and
    // the bias, P stays below 2^8 in bf16 and 2^15 in fp16, whose smallest value
    // 2^-24 is then 2^-31 of the maximum: a long tail of small P is not lost.
    const float msub = (m_i == kNegInf) ? 0.f : m_i - PBias<T>::v;
#pragma unroll
    for (int kb = 0; kb < GROUPS; ++kb)
#pragma unroll
      for (int r = 0; r < 4; ++r) sc[kb][r] = fast_exp2(sc[kb][r] - msub);
    // P^T as the B operand of O^T += V^T P^T, 32 keys at a time: slot t of lane
    // group g holds key key_of(kb) + t of the even group (t < 4), key_of(kb) + t
    // - 4 of the odd one behind it (t >= 4).
    u32x4 pk[GROUPS / 2];
#pragma unroll
    for (int kk = 0; kk < GROUPS / 2; ++kk) {
      const f32x4 a = sc[2 * kk], b = sc[2 * kk + 1];
      pk[kk] = {pack2<T>(a[0], a[1]), pack2<T>(a[2], a[3]), pack2<T>(b[0], b[1]), pack2<T>(b[2], b[3])};
      // The denominator sums the rounded P that the second product uses.
      l_i += sum2_acc<T>(pk[kk][0], sum2_acc<T>(pk[kk][1], 0.f)) + sum2_acc<T>(pk[kk][2], sum2_acc<T>(pk[kk][3], 0.f));
    }
    // V^T A operands by transposed reads: lane (g, i) receives V[key][16 db + i]
    // for the keys of slot t above.
    auto v_operand = [&](int db, int kk) -> u32x4 {
      if constexpr (KV8) {
        // Lanes 2 r and 2 r + 1 of 16 address row r of eight, 16 codes.
        const int r = l16 >> 1;
        const int key = 32 * kk + (r < 4 ? 4 * g16 + r : 16 + ((4 * g16) ^ 8) + r - 4);
        const u32x2 codes = lds_read_tr8((const uint8_t*)Vs + Tile::chunk(key, db) * 16 + 8 * (l16 & 1));
        const float s0 = scale8[slot][2 * kk][1], s1 = scale8[slot][2 * kk + 1][1];
        return {dequantise2<T, false>(codes[0], s0), dequantise2<T, true>(codes[0], s0),
                dequantise2<T, false>(codes[1], s1), dequantise2<T, true>(codes[1], s1)};
      }
      const int col = 16 * db + 4 * (l16 & 3);
      const u32x2 lo = lds_read_tr16(Vs + Tile::elem(4 * g16 + (l16 >> 2), col));
      const u32x2 hi = lds_read_tr16(Vs + Tile::elem(16 + 4 * g16 + (l16 >> 2), col));
      return {lo[0], lo[1], hi[0], hi[1]};
    };
    // Where the rows' limits differ within the step, a key that one row sees and
    // another does not may hold a V that is not finite: 0 V would reach both.
    bool apart = false;
    if (most_lag > 0 && w.rem - most_lag < STEP) {
      bool bad = false;
#pragma unroll
      for (int kk = 0; kk < GROUPS / 2; ++kk)
#pragma unroll
        for (int db = 0; db < NDB; ++db) bad |= any_nonfinite<T>(v_operand(db, kk));
      apart = wave_any(bad);
    }
    if (!apart) {
#pragma unroll
      for (int kk = 0; kk < GROUPS / 2; ++kk)
#pragma unroll
        for (int db = 0; db < NDB; ++db) oacc[db] = Elem<T>::mfma16(v_operand(db, kk), pk[kk], oacc[db]);
      return;
    }
    // Then the rows of each limit on their own, V behind it as zeros.
#pragma unroll 1
    for (int limit = 1; limit <= STEP; ++limit) {
      const bool mine = min(w.rem - row.lag, STEP) == limit;
      if (!wave_any(mine)) continue;
#pragma unroll
      for (int kk = 0; kk < GROUPS / 2; ++kk) {
        u32x4 keep;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = 32 * kk + (j < 2 ? key_of(0) : 16 + key_of(1)) + 2 * (j & 1);
          keep[j] = (key < limit ? 0xffffu : 0u) | (key + 1 < limit ? 0xffff0000u : 0u);
        }
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          const f32x4 sum = Elem<T>::mfma16(v_operand(db, kk) & keep, pk[kk], oacc[db]);
#pragma unroll
          for (int r = 0; r < 4; ++r) oacc[db][r] = mine ? sum[r] : oacc[db][r];
        }
      }
    }
  };

  // O and LSE of the row group, or this worker's partial of it: NS stores in
  // every case (lanes without an output, and whole stores where there is
  // nothing to say, lie outside their resource), so that the waits can count
  // them instead of waiting for them.
  constexpr int NS = NDB + 2;
  auto end_segment = [&](const Unit& w) {
    const bool whole = from_start && w.rem <= STEP;
    const auto& c = cold();
    const int kvh = w.hh / c.nrb, rb = w.hh - kvh * c.nrb;
    const int group = w.b * c.heads + w.hh;
    const int r = wave * 16 + l16;
    const float lt = wave_group16_sum(l_i);
    // A row without keys has lt = 0; one that sees a NaN score, or one of
    // +infinity, has a NaN lt, and passes it on to its O and LSE.
    const float inv = lt == 0.f ? 0.f : 1.f / lt;
    const float lse = lt == 0.f ? kNegInf : (m_i - PBias<T>::v + fast_log2(lt)) * kLn2;
    // kOOB is the top bit, which no offset inside a resource has.
    const uint32_t none = row.out & kOOB, one_lane = g16 == 0 ? none : kOOB;
    auto beyond = [&](int d) -> uint32_t { return (uint32_t)(c.D - 1 - d) & kOOB; };
    if (whole) {
      const auto orr = make_rsrc(c.o + w.b * c.o_sb + (int64_t)kvh * c.G * c.o_sh, c.o_bytes);
      const auto lrr = make_rsrc(c.lse + ((int64_t)w.b * c.Hq + kvh * c.G) * c.Sq, c.lse ? c.G * c.Sq * 4u : 0u);
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
        const int d = 16 * db + 4 * g16;
        const f32x4 ov = oacc[db] * inv;
        const u32x2 o2 = {pack2<T>(ov[0], ov[1]), pack2<T>(ov[2], ov[3])};
        __builtin_amdgcn_raw_buffer_store_b64(o2, orr, (row.out + d * 2u) | beyond(d), 0, 0);
      }
      __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(lse), lrr, (rb * c.rows + r) * 4u | one_lane, 0, 0);
    } else {
      const int64_t slot = (int64_t)(worker + group) * c.rows;
      const auto orr = make_rsrc(c.part_o + slot * c.D, (uint32_t)(c.rows * c.D * 4));
      const auto lrr = make_rsrc(c.part_lse + slot, c.rows * 4u);
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
        const int d = 16 * db + 4 * g16;
        const f32x4 ov = oacc[db] * inv;
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, ov), orr,
                                               (uint32_t)(r * c.D + d) * 4u | none | beyond(d), 0, 0);
      }
      __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(lse), lrr, r * 4u | one_lane, 0, 0);
    }
    // The row group's first worker says how many there are: the steps behind
    // its own fill whole runs.
    const u32x2 parts = {(uint32_t)worker, (uint32_t)(1 + ((w.rem - 1) / STEP + run - 1) / run)};
    __builtin_amdgcn_raw_buffer_store_b64(parts, make_rsrc(c.parts + 2 * (int64_t)group, 8u),
                                          from_start && threadIdx.x == 0 ? 0u : kOOB, 0, 0);
  };

  // Two units are in flight, whatever segments they belong to: a segment's
  // first steps load while the one before it is computed and written.
  // Waits until only what was issued behind a unit's loads is left: the
  // stores of the segment that ended before it, and the next unit's loads.
  auto wait = [&](bool stores, int later) {
    if (!stores && later == 1) {
      KF_WAIT_VMCNT(NL);
    } else {
      static_for<0, 6>([&](auto cc) {
        constexpr int c = decltype(cc)::value;
        constexpr int n = (c & 1 ? NS : 0) + (c >= 2 ? NL : 0) + (c >= 4 ? NQ : 0);
        if (c != 2 && 2 * later + stores == c) KF_WAIT_VMCNT(n < 63 ? n : 63);
      });
    }
  };
  bool ended = false;
  // Of two workers on a SIMD the older one goes first, ends first, and leaves the
  // other alone with half the loads in flight (291 MB, D=64: after 40 and 50 us).
  // The younger one goes first in three units of four: 60.2 -> 58.6 us; in every
  // other one 59.7, always 60.1.
  const bool late = worker >= (int)gridDim.x / 2;
  for (int j0 = -2; j0 < count; j0 += 2) {
    static_for<0, 2>([&](auto sc) {
      constexpr int slot = decltype(sc)::value;
      const int j = j0 + slot;
      if constexpr (KV8 && NW == 1 && workers_per_cu(DT, NW, true) > 4) {
        if (late && j % 4 != 0) __builtin_amdgcn_s_setprio(1);
        else __builtin_amdgcn_s_setprio(0);
      }
      if (j >= 0 && j < count) {
        const bool next = j + 1 < count;
        wait(ended, next ? held[1 - slot].begin ? 2 : 1 : 0);
        worker_barrier<NW>();  // the other waves' loads of the unit are done too
        const Unit w = held[slot];
        if (w.begin) begin_segment(w, sc);
        step(w, sc);
        ended = !next || w.rem <= STEP;
        if (ended) end_segment(w);
        __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the slot has been read,
        worker_barrier<NW>();                // by the other waves too
      }
      if (j + 2 < count) issue(j + 3 < count, sc);
    });
  }
}

// Packed rows per row group, and the waves that they take.
inline int paged_rows(int64_t R) { return (int)(R < 64 ? R : 64); }
inline int paged_waves(int64_t R) { return R <= 16 ? 1 : R <= 32 ? 2 : 4; }

// Head-dim tile: of 8-bit rows one that whole 1 KB loads make 16 rows of.
inline int paged_tile(int64_t D, bool kv8) { return kv8 ? (D <= 64 ? 64 : 128) : head_tile(D); }

// The workers' launch over 8-bit pools (paged_fp8.hip).
void launch_workers_fp8(const PagedParams& p, int dtype, hipStream_t stream);

}  // namespace kf
