// e4m3 caches of the windowed decode attention (paged_window_kernel.h)
#include "paged_window_kernel.h"

namespace pe {
int launch_window_fp8(const WinArgs& a, int head_size, int block_size, int waves, int dtype, dim3 grid, hipStream_t st) {
  PE_DISPATCH_16(dtype, T, return (dispatch_window<T, Fp8>(a, head_size, block_size, waves, grid, st)));
  return PE_OK;
}
int window_fp8_diag_fetch(unsigned int* out, int reset) { return window_diag_fetch_tu(out, reset); }
}  // namespace pe
