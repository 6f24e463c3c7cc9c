// The workers of attention over 8-bit pools (paged_attn.hpp).
#include "paged_attn.hpp"

namespace kf {

template <typename T, int DT, PoolKind POOL>
static void launch_pool(const PagedParams& p, hipStream_t stream) {
  const dim3 grid((unsigned)p.workers);
  switch (paged_waves(p.rows)) {
    case 1: hipLaunchKernelGGL((paged_kernel<T, DT, 1, false, POOL>), grid, dim3(64), 0, stream, p); break;
    case 2: hipLaunchKernelGGL((paged_kernel<T, DT, 2, false, POOL>), grid, dim3(128), 0, stream, p); break;
    default: hipLaunchKernelGGL((paged_kernel<T, DT, 4, false, POOL>), grid, dim3(256), 0, stream, p); break;
  }
}

// Rows with padding are kernels of their own: silencing it costs the others
// scalars that no longer fit the registers (48 requests up to 6000 tokens, one
// KV head of 96 dims: 18.6 us against 17.3).
template <typename T, int DT>
static void launch_tile(const PagedParams& p, hipStream_t stream) {
  if (p.D % 16) launch_pool<T, DT, kPool8Padded>(p, stream);
  else launch_pool<T, DT, kPool8>(p, stream);
}

void launch_workers_fp8(const PagedParams& p, int dtype, hipStream_t stream) {
  const bool small = paged_tile(p.D, true) == 64;
  if (dtype == KF_F16) small ? launch_tile<_Float16, 64>(p, stream) : launch_tile<_Float16, 128>(p, stream);
  else small ? launch_tile<__bf16, 64>(p, stream) : launch_tile<__bf16, 128>(p, stream);
}

}  // namespace kf
