// The workers of attention over 8-bit pools (paged_attn.hpp).
#include "paged_attn.hpp"

namespace kf {

template <typename T, int DT>
static void launch_tile(const PagedParams& p, hipStream_t stream) {
  const dim3 grid((unsigned)p.workers);
  switch (paged_waves(p.rows)) {
    case 1: hipLaunchKernelGGL((paged_kernel<T, DT, 1, false, true>), grid, dim3(64), 0, stream, p); break;
    case 2: hipLaunchKernelGGL((paged_kernel<T, DT, 2, false, true>), grid, dim3(128), 0, stream, p); break;
    default: hipLaunchKernelGGL((paged_kernel<T, DT, 4, false, true>), grid, dim3(256), 0, stream, p); break;
  }
}

void launch_workers_fp8(const PagedParams& p, int dtype, hipStream_t stream) {
  const bool small = paged_tile(p.D, true) == 64;
  if (dtype == KF_F16) small ? launch_tile<_Float16, 64>(p, stream) : launch_tile<_Float16, 128>(p, stream);
  else small ? launch_tile<__bf16, 64>(p, stream) : launch_tile<__bf16, 128>(p, stream);
}

}  // namespace kf
