// int8 caches of the decode step that appends its row itself (paged_window_kernel.h, STEP)
#include "paged_window_kernel.h"

namespace pe {
int launch_step_int8(const WinArgs& a, int head_size, int block_size, int waves, int dtype, dim3 grid, hipStream_t st) {
  PE_DISPATCH_16(dtype, T, return (dispatch_window<T, Int8, true>(a, head_size, block_size, waves, grid, st)));
  return PE_OK;
}
int step_int8_diag_fetch(unsigned int* out, int reset) { return window_diag_fetch_tu(out, reset); }
}  // namespace pe
