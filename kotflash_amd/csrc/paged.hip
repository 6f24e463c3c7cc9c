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
// requests' keys are numbered in steps of 32: unit u = (request, KV head and
// row block, step). A fixed number of workers (one wave each, as many as LDS
// lets the GPU hold) take equal runs of consecutive units, wherever requests
// begin and end in them: every worker streams the same number of bytes however
// the lengths differ, which a grid of (request, head, split) does not give.
//  * A worker finds its run from the lengths: a sum over the batch, and the
//    request in which the run begins.
//  * Within a run the part in one (request, head) is a segment: the packed
//    query rows of the group against its steps, with a wave-private LDS ring
//    that direct-to-LDS loads fill two steps ahead (S^T = K Q^T, online
//    softmax, O^T += V^T P^T on 16x16x32 MFMAs, as in the contiguous decode).
//  * A segment that is a whole request writes O; others write an fp32 partial
//    (O, LSE) to slot worker + row group. Both numbers grow along the units
//    and one of them at every segment, so the slots are distinct, and those of
//    one row group are consecutive. The second launch merges them in order
//    (no atomics, same bits every time) and zeroes the rows that see nothing.
//  * One wave per worker: no barrier anywhere, and while one worker of a CU
//    starts or ends a segment the others stream.
//
// Pages: 16 rows of one page at a time have a buffer resource of their own,
// from a page number read by the scalar unit, with 64-bit bases (a pool may be
// larger than 4 GiB) and an extent that ends at the last visible row: rows
// behind it load as zeros, whatever the page holds there (NaN included), and a
// page number outside the pool reads nothing and its keys are masked.
#include "decode_merge.hpp"
#include "kf_common.hpp"
#include "kf_host.hpp"

namespace kf {

int check_attn_common(const char* what, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t Sk,
                      int64_t D, int dtype);
int check_tensor(const char* what, const char* name, const void* ptr, const int64_t* strides);

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
  int64_t k_sp, k_sh, k_ss;  // page, head, row
  int64_t v_sp, v_sh, v_ss;
  int64_t o_sb, o_sh, o_ss;
  int B, Hq, Hkv, Sq, D, G;
  int pages, gpp;  // pages of the pool; 16-row groups per page
  uint32_t gpp_inv;  // floor(2^32 / gpp)
  int cap;         // tokens that a table has columns for
  int rows, nrb;   // packed rows per row group, row groups per KV head
  int heads;       // Hkv * nrb
  int workers, least;
  int causal;
  float scale_log2;
};

// Direct-to-LDS load (kf_common.hpp) whose resource may have been written by
// the vector unit just before (a spilled scalar comes back by v_readlane): a
// vector-memory instruction may read such a register five wait states later.
// STREAM: marked as read once (nt).
template <bool STREAM>
__device__ inline void dma16_r(__amdgpu_buffer_rsrc_t r, uint32_t lds_m0, uint32_t voff) {
  if constexpr (STREAM) {
    asm volatile(
        "s_mov_b32 m0, %0\n\t"
        "s_nop 4\n\t"
        "buffer_load_dwordx4 %1, %2, 0 offen nt lds"
        :
        : "s"(__builtin_amdgcn_readfirstlane(lds_m0)), "v"(voff), "s"(r)
        : "memory", "m0");
  } else {
    asm volatile(
        "s_mov_b32 m0, %0\n\t"
        "s_nop 4\n\t"
        "buffer_load_dwordx4 %1, %2, 0 offen lds"
        :
        : "s"(__builtin_amdgcn_readfirstlane(lds_m0)), "v"(voff), "s"(r)
        : "memory", "m0");
  }
}

constexpr int kStep = 32;     // keys per unit
constexpr int kPagedRing = 2; // steps of a worker in flight

// K/V bytes of a call from which its loads are marked as read once. Such loads
// do not go through the 256 MB memory-side cache, which costs the others a
// tenth of their rate (measured, three sets of inputs in turn: 1158 MB 209 us
// plain and 188 marked, 537 MB 103 and 93, 300 MB 64 and 57, 294 MB 62 and
// 54); but a call of which the cache still holds a part from the last time is
// faster plain (59 MB 21 and 23).
constexpr int64_t kStreamBytes = 128 << 20;

__device__ inline int wave_sum(int x) { return __builtin_amdgcn_readlane(wave_scan(x), 63); }

__device__ inline int visible(const PagedParams& p, int len) { return min(max(len, 0), p.cap); }
__device__ inline int steps_of(const PagedParams& p, int len) { return (visible(p, len) + kStep - 1) / kStep; }
__device__ inline int lane_steps(const PagedParams& p, int b) {
  return b < p.B ? steps_of(p, p.lengths[b]) : 0;
}
// Steps (of one head) of the requests from b0 on.
__device__ inline int steps_from(const PagedParams& p, int b0, int lane) {
  int n = 0;
  for (; b0 < p.B; b0 += 64) n += lane_steps(p, b0 + lane);
  return wave_sum(n);
}
// Units per worker.
__device__ inline int run_length(const PagedParams& p, int total) {
  return max(p.least, (total * p.heads + p.workers - 1) / p.workers);
}

template <typename T> struct PBias;  // P = 2^(s - m + bias), see paged_kernel
template <> struct PBias<_Float16> { static constexpr float v = 7.f; };
template <> struct PBias<__bf16> { static constexpr float v = 0.f; };

template <typename T, int DT, int QB>
__global__ __launch_bounds__(64) void paged_kernel(const PagedParams p) {
  constexpr int CPR = DT / 8;         // 16-byte chunks per row
  constexpr int NDC = DT / 32;        // 32-wide head-dim chunks (S contraction)
  constexpr int NDB = DT / 16;        // 16-wide head-dim blocks of O^T
  constexpr int VT = kStep * DT;      // elements of one K (or V) step tile
  constexpr int NGI = 16 * CPR / 64;  // 1 KB loads per 16-row group of K (or V)
  constexpr int NL = 4 * NGI;         // loads per step: two groups of K and of V
  using Tile = SwizzledTile<CPR>;
  __shared__ __attribute__((aligned(16))) uint16_t ring[kPagedRing * 2 * VT];

  const int lane = threadIdx.x;
  const int l16 = lane & 15, g16 = lane >> 4;
  const const_i32 lengths = (const_i32)(uintptr_t)p.lengths;

  // This worker's run of units, and where it begins: request b, whose first
  // unit is `start`. The first 64 requests' lengths are read once.
  const int worker = blockIdx.x;
  const int len0 = lane < p.B ? visible(p, p.lengths[lane]) : 0;
  const int mine0 = (len0 + kStep - 1) / kStep;
  const int sum0 = wave_scan(mine0);
  int total = __builtin_amdgcn_readlane(sum0, 63);
  if (p.B > 64) total += steps_from(p, 64, lane);
  const int run = run_length(p, total);
  const int u = worker * run;
  if (u >= total * p.heads) return;  // more workers than runs
  int b, start, len;
  uint64_t past = __builtin_amdgcn_ballot_w64(sum0 * p.heads > u);
  if (past) {
    b = __builtin_ctzll(past);
    len = __builtin_amdgcn_readlane(len0, b);
    start = (__builtin_amdgcn_readlane(sum0, b) - __builtin_amdgcn_readlane(mine0, b)) * p.heads;
  } else {
    start = __builtin_amdgcn_readlane(sum0, 63) * p.heads;
    for (b = 64;; b += 64) {
      const int mine = lane_steps(p, b + lane) * p.heads;
      const int sum = wave_scan(mine);
      past = __builtin_amdgcn_ballot_w64(start + sum > u);
      if (past) {
        const int at = __builtin_ctzll(past);
        start += __builtin_amdgcn_readlane(sum, at) - __builtin_amdgcn_readlane(mine, at);
        b += at;
        break;
      }
      start += __builtin_amdgcn_readlane(sum, 63);
    }
    len = visible(p, lengths[b]);
  }
  int n = (len + kStep - 1) / kStep;
  int hh = (u - start) / n;
  int s0 = (u - start) - hh * n;
  int left = run;

  // Per-lane plan of a group's loads: this lane's 16-byte chunk within the 16
  // rows (kOOB for head-dim padding). The swizzle key has a period of 16 rows,
  // so both groups of a step share it.
  uint32_t koff[NGI], voff[NGI];
#pragma unroll
  for (int k = 0; k < NGI; ++k) {
    const int pc = k * 64 + lane;
    const int r = pc / CPR;
    const int c = (pc % CPR) ^ Tile::key(r);
    const bool ok = c * 8 < p.D;
    koff[k] = ok ? (uint32_t)(r * p.k_ss + c * 8) * 2u : kOOB;
    voff[k] = ok ? (uint32_t)(r * p.v_ss + c * 8) * 2u : kOOB;
  }
  const uint32_t ring0 = lds_addr(ring);
  const bool stream = (int64_t)total * p.heads * (kStep * 4 * p.D) > kStreamBytes;

  for (;;) {
    // One segment: steps [s0, s1) of row group hh of request b.
    const int s1 = min(n, s0 + left);
    const int kvh = hh / p.nrb, rb = hh % p.nrb;
    const int R = p.G * p.Sq;
    const uint16_t* kh = p.k + kvh * p.k_sh;
    const uint16_t* vh = p.v + kvh * p.v_sh;
    const const_i32 table = (const_i32)(uintptr_t)(p.tables + b * p.t_sb);

    // Q rows as MFMA B operands: lane l = packed row qb * 16 + l % 16, k slots
    // = head dims 32 dc + 8 (l / 16) .. + 7.
    u32x4 qf[QB][NDC];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      const int rho = rb * p.rows + qb * 16 + l16;
      const bool row = qb * 16 + l16 < p.rows && rho < R;
      const int g = row ? rho / p.Sq : 0, i = row ? rho % p.Sq : 0;
      const uint16_t* qrow = p.q + b * p.q_sb + (kvh * p.G + g) * p.q_sh + i * p.q_ss;
#pragma unroll
      for (int dc = 0; dc < NDC; ++dc) {
        const int d = 32 * dc + 8 * g16;
        qf[qb][dc] = row && d < p.D ? ldg16(qrow + d) : zero_u4();
      }
    }

    // The pages of a step's two 16-row groups (column and first row of each,
    // the last visible group's where the second lies behind it). Read one
    // step before they are needed, all of a ring's at the segment's start.
    struct StepPages {
      int page[2], row0[2];
    };
    auto look_up = [&](int s) {
      StepPages sp;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const uint32_t gi = min(2 * s + g, (len - 1) >> 4);
        uint32_t column = __umulhi(gi, p.gpp_inv);
        uint32_t rest = gi - column * p.gpp;
        const bool up = rest >= (uint32_t)p.gpp;  // the quotient may be one short
        column += up;
        rest -= up ? p.gpp : 0;
        sp.page[g] = table[column];
        sp.row0[g] = (int)rest * 16;
      }
      return sp;
    };
    // Loads of step s into its slot; visible rows per group, 0 where the page
    // is not in the pool.
    int vis[kPagedRing][2];
    auto issue = [&](int s, const StepPages& sp, auto slot_c) {
      constexpr int slot = decltype(slot_c)::value;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const uint32_t m0 = ring0 + slot * 2 * VT * 2 + g * 16 * DT * 2;
        const int page = __builtin_amdgcn_readfirstlane(sp.page[g]);
        int seen = min(max(len - 32 * s - 16 * g, 0), 16);
        if (page < 0 || page >= p.pages) seen = 0;
        const int64_t at = seen > 0 ? page : 0;
        const auto kr = make_rsrc(kh + at * p.k_sp + sp.row0[g] * p.k_ss, rows_extent(seen, p.k_ss, p.D));
        const auto vr = make_rsrc(vh + at * p.v_sp + sp.row0[g] * p.v_ss, rows_extent(seen, p.v_ss, p.D));
        if (stream) {
#pragma unroll
          for (int k = 0; k < NGI; ++k) {
            dma16_r<true>(kr, m0 + k * 1024u, koff[k]);
            dma16_r<true>(vr, m0 + VT * 2 + k * 1024u, voff[k]);
          }
        } else {
#pragma unroll
          for (int k = 0; k < NGI; ++k) {
            dma16_r<false>(kr, m0 + k * 1024u, koff[k]);
            dma16_r<false>(vr, m0 + VT * 2 + k * 1024u, voff[k]);
          }
        }
        vis[slot][g] = seen;
      }
    };
    StepPages first[kPagedRing];
    static_for<0, kPagedRing>([&](auto sc) { first[decltype(sc)::value] = look_up(s0 + decltype(sc)::value); });
    StepPages next = look_up(s0 + kPagedRing);
    static_for<0, kPagedRing>([&](auto sc) {
      if (s0 + decltype(sc)::value < s1) issue(s0 + decltype(sc)::value, first[decltype(sc)::value], sc);
    });

    f32x4 oacc[QB][NDB];  // O^T: lane l, register r = head dim 16 db + 4 (l / 16) + r of row l % 16
    float m_i[QB], l_i[QB];
    int lim[QB];  // keys before lim are visible to this lane's row
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      m_i[qb] = kNegInf;
      l_i[qb] = 0.f;
      lim[qb] = p.causal ? len - (p.Sq - 1 - (rb * p.rows + qb * 16 + l16) % p.Sq) : len;
#pragma unroll
      for (int db = 0; db < NDB; ++db) oacc[qb][db] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const int least_lim = p.causal ? len - (p.Sq - 1) : len;

    auto step = [&](int s, auto slot_c) {
      constexpr int slot = decltype(slot_c)::value;
      const uint16_t* Ks = ring + slot * 2 * VT;
      const uint16_t* Vs = Ks + VT;
      // K rows as MFMA A operands: lane = key kb * 16 + l % 16, slots = head dims.
      u32x4 ka[2][NDC];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int dc = 0; dc < NDC; ++dc) ka[kb][dc] = lds_read16(Ks + Tile::chunk(kb * 16 + l16, 4 * dc + g16) * 8);
      const bool masked = vis[slot][0] + vis[slot][1] < kStep || (s + 1) * kStep > least_lim;
      u32x4 pk[QB];
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        // S^T: lane l, register r = key kb * 16 + 4 (l / 16) + r of row l % 16.
        f32x4 sc[2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          sc[kb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int dc = 0; dc < NDC; ++dc) sc[kb] = Elem<T>::mfma16(ka[kb][dc], qf[qb][dc], sc[kb]);
          sc[kb] *= p.scale_log2;
        }
        // Masked after the scale, so that a scale of zero leaves -inf.
        if (masked) {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int c = 4 * g16 + r;
              const bool seen = c < vis[slot][kb] && s * kStep + 16 * kb + c < lim[qb];
              sc[kb][r] = seen ? sc[kb][r] : kNegInf;
            }
        }
        float mx = kNegInf;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int r = 0; r < 4; ++r) mx = fmaxf(mx, sc[kb][r]);
        mx = wave_group16_max(mx);
        if (m_i[qb] == kNegInf) {
          m_i[qb] = mx;
        } else {
          const bool grow = mx > m_i[qb] + kRescaleThreshold;
          if (wave_any(grow)) {
            const float alpha = grow ? fast_exp2(m_i[qb] - mx) : 1.f;
            l_i[qb] *= alpha;
#pragma unroll
            for (int db = 0; db < NDB; ++db) oacc[qb][db] *= alpha;
            m_i[qb] = grow ? mx : m_i[qb];
          }
        }
        // P in 16 bits for the second product. With m up to 8 below the
        // maximum and the bias, P stays below 2^8 in bf16 and 2^15 in fp16,
        // whose smallest value 2^-24 is then 2^-31 of the maximum: a long tail
        // of small P is not lost.
        const float msub = (m_i[qb] == kNegInf) ? 0.f : m_i[qb] - PBias<T>::v;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int r = 0; r < 4; ++r) sc[kb][r] = fast_exp2(sc[kb][r] - msub);
        // P^T as the B operand of O^T += V^T P^T: slot t of lane group g holds
        // key 4 g + t (t < 4) or 16 + 4 g + t - 4 (t >= 4).
        pk[qb][0] = pack2<T>(sc[0][0], sc[0][1]);
        pk[qb][1] = pack2<T>(sc[0][2], sc[0][3]);
        pk[qb][2] = pack2<T>(sc[1][0], sc[1][1]);
        pk[qb][3] = pack2<T>(sc[1][2], sc[1][3]);
        // The denominator sums the rounded P that the second product uses.
        l_i[qb] += sum2_acc<T>(pk[qb][0], sum2_acc<T>(pk[qb][1], 0.f)) +
                   sum2_acc<T>(pk[qb][2], sum2_acc<T>(pk[qb][3], 0.f));
      }
      // V^T A operands by transposed reads: lane (g, i) receives V[key][16 db + i]
      // for the keys of slot t above.
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
        const int col = 16 * db + 4 * (l16 & 3);
        const u32x2 lo = lds_read_tr16(Vs + Tile::elem(4 * g16 + (l16 >> 2), col));
        const u32x2 hi = lds_read_tr16(Vs + Tile::elem(16 + 4 * g16 + (l16 >> 2), col));
        const u32x4 a = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) oacc[qb][db] = Elem<T>::mfma16(a, pk[qb], oacc[qb][db]);
      }
    };

    for (int j0 = s0; j0 < s1; j0 += kPagedRing) {
      static_for<0, kPagedRing>([&](auto sc) {
        const int s = j0 + decltype(sc)::value;
        if (s < s1) {
          // This step's loads are done once only those of later ones are left.
          const int later = min(kPagedRing - 1, s1 - 1 - s);
          static_for<0, kPagedRing>([&](auto lc) {
            if (later == decltype(lc)::value) KF_WAIT_VMCNT(decltype(lc)::value * NL);
          });
          step(s, sc);
          if (s + kPagedRing < s1) {
            __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the slot has been read
            issue(s + kPagedRing, next, sc);
            next = look_up(s + kPagedRing + 1);
          }
        }
      });
    }
    static_assert((kPagedRing - 1) * NL < 64, "the counter of outstanding loads has six bits");

    // O and LSE, or the partial of this worker.
    const bool whole = s0 == 0 && s1 == n;
    const int64_t slot = (int64_t)(worker + b * p.heads + hh) * p.rows;
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      const int r = qb * 16 + l16;
      const int rho = rb * p.rows + r;
      const float lt = wave_group16_sum(l_i[qb]);
      if (r >= p.rows || rho >= R) continue;
      const float inv = lt > 0.f ? 1.f / lt : 0.f;
      const float lse = lt > 0.f ? (m_i[qb] - PBias<T>::v + fast_log2(lt)) * kLn2 : kNegInf;
      const int h = kvh * p.G + rho / p.Sq, i = rho % p.Sq;
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
        const int d = 16 * db + 4 * g16;
        if (d >= p.D) continue;
        const f32x4 ov = oacc[qb][db] * inv;
        if (whole) {
          u32x2 w;
          w[0] = pack2<T>(ov[0], ov[1]);
          w[1] = pack2<T>(ov[2], ov[3]);
          *reinterpret_cast<u32x2*>(p.o + b * p.o_sb + h * p.o_sh + i * p.o_ss + d) = w;
        } else {
          *reinterpret_cast<f32x4*>(p.part_o + (slot + r) * p.D + d) = ov;
        }
      }
      if (g16 == 0) {
        if (!whole) p.part_lse[slot + r] = lse;
        else if (p.lse) p.lse[((int64_t)b * p.Hq + h) * p.Sq + i] = lse;
      }
    }

    // The row group's first worker says how many there are: the steps behind
    // its own fill whole runs.
    if (s0 == 0 && lane == 0) {
      p.parts[2 * (b * p.heads + hh)] = worker;
      p.parts[2 * (b * p.heads + hh) + 1] = 1 + (n - s1 + run - 1) / run;
    }

    left -= s1 - s0;
    if (left <= 0) break;
    // The next segment: next row group, or the next request that holds keys.
    s0 = 0;
    if (++hh == p.heads) {
      hh = 0;
      do {
        if (++b == p.B) return;
        len = visible(p, lengths[b]);
      } while (len == 0);
      n = steps_of(p, len);
    }
  }
}

// One workgroup of W waves per output row: merges the row's partials, writes
// zeros where the request holds nothing, and leaves rows that one worker wrote
// whole. Bound by its chain of loads: which partials, then all of them. The
// first wave alone takes what one round trip brings; more partials the waves
// share, and combine through LDS in their order.
template <typename T, int QL, int W>
__global__ __launch_bounds__(64 * W) void paged_merge_kernel(const PagedParams p) {
  const int lane = threadIdx.x & 63, wave = wave_index();
  const int r = blockIdx.x % p.rows;
  const int bh = blockIdx.x / p.rows;
  const int hh = bh % p.heads, b = bh / p.heads;
  const int kvh = hh / p.nrb, rho = (hh % p.nrb) * p.rows + r;
  // What the workers wrote is not there for a request without keys.
  const int len = ((const_i32)(uintptr_t)p.lengths)[b];
  const int w0 = ((const_i32)(uintptr_t)p.parts)[2 * bh], parts = ((const_i32)(uintptr_t)p.parts)[2 * bh + 1];
  if (rho >= p.G * p.Sq) return;
  const bool alone = W == 1 || len <= 0 || parts <= kMergeU * (64 / QL);
  if (alone && wave > 0) return;
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
    merge_row<T, QL>(orr, lrr, ostride, lstride, parts, p.D, out, lse);
    return;
  }
  if constexpr (W > 1) {
    __shared__ float sums[W][QL][6];
    const int share = (parts + W - 1) / W;
    const MergeState mine = merge_splits<QL>(orr, lrr, ostride, lstride, min(wave * share, parts),
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

// Packed rows per worker: 16-row MFMA blocks, up to four of them.
static int paged_row_blocks(int64_t R) { return R <= 16 ? 1 : R <= 32 ? 2 : 4; }
static int paged_rows(int64_t R) { return (int)(R < 64 ? R : 64); }

// Workers: what the LDS of 256 CUs holds of their rings, 4 KB short of 160.
static int paged_workers(int64_t D) {
  const int ring = kPagedRing * 2 * kStep * head_tile(D) * 2;
  const int per_cu = 156 * 1024 / ring;
  return 256 * (per_cu < 8 ? per_cu : 8);
}

static int64_t paged_slots(int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t D) {
  const int64_t R = Hq / Hkv * Sq;
  return paged_workers(D) + B * Hkv * ((R + paged_rows(R) - 1) / paged_rows(R));
}

// Waves per row of the merge, from the most partials a row group can have: a
// head's share of the workers (all of them on one request), cut at both ends.
// More waves cost launch time, a few tenths of a us where they are not needed
// (1158 MB over 64 requests: 4.6 us with one wave, 5.0 with four, 7.2 with
// eight), and save round trips where one row has many partials (131072 keys of
// one request, 128 partials: 5.9 us with one wave, 4.6 with four).
template <typename T, int QL>
static void launch_merge(const PagedParams& p, hipStream_t stream) {
  constexpr int kTrip = kMergeU * (64 / QL);  // partials that a wave takes at once
  const int64_t rows = (int64_t)p.B * p.heads * p.rows;
  const int share = p.workers / p.heads + 2, steps = p.cap / kStep + 1;
  const int most = share < steps ? share : steps;
  const dim3 grid((unsigned)rows);
  if (most > 16 * kTrip && rows <= 256)
    hipLaunchKernelGGL((paged_merge_kernel<T, QL, 16>), grid, dim3(1024), 0, stream, p);
  else if (most > kTrip && (rows <= 256 || most > 8 * kTrip))
    hipLaunchKernelGGL((paged_merge_kernel<T, QL, 4>), grid, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((paged_merge_kernel<T, QL, 1>), grid, dim3(64), 0, stream, p);
}

template <typename T, int DT>
static int launch_paged(const PagedParams& p, hipStream_t stream) {
  const dim3 grid((unsigned)p.workers);
  switch (paged_row_blocks(p.rows)) {
    case 1: hipLaunchKernelGGL((paged_kernel<T, DT, 1>), grid, dim3(64), 0, stream, p); break;
    case 2: hipLaunchKernelGGL((paged_kernel<T, DT, 2>), grid, dim3(64), 0, stream, p); break;
    default: hipLaunchKernelGGL((paged_kernel<T, DT, 4>), grid, dim3(64), 0, stream, p); break;
  }
  const int rc = check_launch("kf_paged_decode(workers)");
  if (rc) return rc;
  if (p.D <= 64) launch_merge<T, 16>(p, stream);
  else launch_merge<T, 32>(p, stream);
  return check_launch("kf_paged_decode(merge)");
}

template <typename T>
static int dispatch_paged(const PagedParams& p, hipStream_t stream) {
  switch (head_tile(p.D)) {
    case 32: return launch_paged<T, 32>(p, stream);
    case 64: return launch_paged<T, 64>(p, stream);
    case 96: return launch_paged<T, 96>(p, stream);
    default: return launch_paged<T, 128>(p, stream);
  }
}

}  // namespace kf

using namespace kf;

extern "C" size_t kf_paged_decode_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t D) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Sq <= 0 || D <= 0 || D > 128 || Hq % Hkv) return 0;
  const int64_t R = Hq / Hkv * Sq;
  const size_t rows = (size_t)paged_slots(B, Hq, Hkv, Sq, D) * paged_rows(R);
  const size_t groups = (size_t)(B * Hkv * ((R + paged_rows(R) - 1) / paged_rows(R)));
  return (rows * (size_t)D * sizeof(float) + 255) / 256 * 256 + (rows * sizeof(float) + 255) / 256 * 256 +
         groups * 2 * sizeof(int32_t);
}

extern "C" int kf_paged_decode(const void* q, const void* k_pages, const void* v_pages, void* o, float* lse,
                               const int32_t* tables, const int32_t* lengths, int64_t B, int64_t Hq, int64_t Hkv,
                               int64_t Sq, int64_t D, int64_t num_pages, int64_t page_size, int64_t columns,
                               int64_t table_stride, const int64_t* q_strides, const int64_t* k_strides,
                               const int64_t* v_strides, const int64_t* o_strides, float scale, int causal,
                               int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "kf_paged_decode";
  int rc = check_attn_common(what, B, Hq, Hkv, Sq, 1, D, dtype);
  if (rc) return rc;
  if ((rc = check_tensor(what, "q", q, q_strides)) || (rc = check_tensor(what, "k_pages", k_pages, k_strides)) ||
      (rc = check_tensor(what, "v_pages", v_pages, v_strides)) || (rc = check_tensor(what, "o", o, o_strides)))
    return rc;
  if (tables == nullptr || lengths == nullptr)
    return set_error(KF_EINVAL, "%s: tables and lengths must be non-null", what);
  if (!(scale == scale) || scale - scale != 0.f) return set_error(KF_EINVAL, "%s: scale must be finite", what);
  if (num_pages <= 0 || columns <= 0 || num_pages > 0x7fffffff)
    return set_error(KF_EINVAL, "%s: num_pages and table columns must be positive", what);
  if (page_size <= 0 || page_size % 16 != 0)
    return set_error(KF_EUNSUPPORTED, "%s: page_size must be a multiple of 16, got %lld", what, (long long)page_size);
  if (columns > 1 && table_stride < 0) return set_error(KF_EINVAL, "%s: negative table stride", what);
  if (page_size > 0x3fffffff / columns)
    return set_error(KF_EUNSUPPORTED, "%s: a table of %lld pages of %lld tokens is beyond 32-bit positions", what,
                     (long long)columns, (long long)page_size);
  const int64_t R = Hq / Hkv * Sq;
  if (R > 0x3fffffff) return set_error(KF_EUNSUPPORTED, "%s: too many query rows", what);
  const int rows = paged_rows(R);
  const int64_t nrb = (R + rows - 1) / rows, heads = Hkv * nrb;
  const int64_t cap = columns * page_size;
  if (heads * ((cap + kStep - 1) / kStep) > 0x7fffffff / B)
    return set_error(KF_EUNSUPPORTED, "%s: %lld tables of %lld tokens are beyond 32-bit step numbers", what,
                     (long long)B, (long long)cap);
  if (B * heads * rows > 0x7fffffff) return set_error(KF_EUNSUPPORTED, "%s: grid too large", what);
  if ((15 * k_strides[2] + D) * 2 > 0x7fffffffLL || (15 * v_strides[2] + D) * 2 > 0x7fffffffLL)
    return set_error(KF_EUNSUPPORTED, "%s: 16 rows of a page span more than 2 GiB", what);
  const size_t need = kf_paged_decode_workspace_bytes(B, Hq, Hkv, Sq, D);
  if (workspace == nullptr || workspace_bytes < need)
    return set_error(KF_EINVAL, "%s: workspace of %zu bytes required, got %zu", what, need,
                     workspace == nullptr ? (size_t)0 : workspace_bytes);
  if (!aligned16(workspace)) return set_error(KF_EINVAL, "%s: workspace must be 16-byte aligned", what);
  PagedParams p{};
  p.q = (const uint16_t*)q; p.k = (const uint16_t*)k_pages; p.v = (const uint16_t*)v_pages;
  p.o = (uint16_t*)o; p.lse = lse; p.tables = tables; p.lengths = lengths;
  const size_t slot_rows = (size_t)paged_slots(B, Hq, Hkv, Sq, D) * rows;
  p.part_o = (float*)workspace;
  p.part_lse = (float*)((char*)workspace + (slot_rows * (size_t)D * sizeof(float) + 255) / 256 * 256);
  p.parts = (int32_t*)((char*)p.part_lse + (slot_rows * sizeof(float) + 255) / 256 * 256);
  p.t_sb = table_stride;
  p.q_sb = q_strides[0]; p.q_sh = q_strides[1]; p.q_ss = q_strides[2];
  p.k_sp = k_strides[0]; p.k_sh = k_strides[1]; p.k_ss = k_strides[2];
  p.v_sp = v_strides[0]; p.v_sh = v_strides[1]; p.v_ss = v_strides[2];
  p.o_sb = o_strides[0]; p.o_sh = o_strides[1]; p.o_ss = o_strides[2];
  p.B = (int)B; p.Hq = (int)Hq; p.Hkv = (int)Hkv; p.Sq = (int)Sq; p.D = (int)D; p.G = (int)(Hq / Hkv);
  p.pages = (int)num_pages; p.gpp = (int)(page_size / 16);
  p.gpp_inv = (uint32_t)((1ull << 32) / p.gpp > 0xffffffffull ? 0xffffffffull : (1ull << 32) / p.gpp);
  p.cap = (int)cap;
  p.rows = rows; p.nrb = (int)nrb; p.heads = (int)heads;
  p.workers = paged_workers(D); p.least = 1;
  p.causal = causal != 0;
  p.scale_log2 = scale * kLog2e;
  hipStream_t s = (hipStream_t)stream;
  return dtype == KF_F16 ? dispatch_paged<_Float16>(p, s) : dispatch_paged<__bf16>(p, s);
}
