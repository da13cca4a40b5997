// Varlen prefill attention with a sliding window and sink tokens (pe_prefill_window): dispatch of the
// windowed form of the matrix-core kernel in prefill_kernel.h.
#include "prefill_kernel.h"

extern "C" int pe_prefill_window(void* out, const void* q, const void* k, const void* v,
                                 const int32_t* cu_q, const int32_t* cu_kv, int num_seqs,
                                 int max_q_len, int num_heads, int num_kv_heads, int head_size,
                                 int64_t q_stride, int64_t k_stride, int64_t v_stride,
                                 int64_t out_stride, float scale, int sliding_window, int num_sinks,
                                 int dtype, void* stream) {
  using namespace pe;
  PE_REQUIRE(num_seqs >= 0 && max_q_len >= 0, PE_ERR_INVALID_ARG, "prefill_window: negative size");
  PE_REQUIRE(sliding_window >= 0 && num_sinks >= 0, PE_ERR_INVALID_ARG,
             "prefill_window: sliding_window %d and num_sinks %d must not be negative", sliding_window, num_sinks);
  if (num_seqs == 0 || max_q_len == 0) return PE_OK;
  PE_REQUIRE(out && q && k && v && cu_q && cu_kv, PE_ERR_INVALID_ARG, "prefill_window: null pointer");
  PE_REQUIRE(num_heads > 0 && num_kv_heads > 0 && num_heads % num_kv_heads == 0, PE_ERR_INVALID_ARG,
             "prefill_window: num_heads %d must be a positive multiple of num_kv_heads %d", num_heads, num_kv_heads);
  PE_REQUIRE(head_size == 32 || head_size == 64 || head_size == 80 || head_size == 96 || head_size == 112 ||
                 head_size == 120 || head_size == 128 || head_size == 192 || head_size == 256,
             PE_ERR_UNSUPPORTED, "prefill_window: head size %d is not built", head_size);
  PE_REQUIRE(dtype == PE_BF16 || dtype == PE_F16, PE_ERR_UNSUPPORTED, "prefill_window: dtype %d (bf16 or f16)", dtype);
  // the maxima are kept in scaled units
  PE_REQUIRE(scale > 0.f && scale < INFINITY, PE_ERR_UNSUPPORTED, "prefill_window: scale must be positive and finite");
  PE_REQUIRE(max_q_len <= (1 << 22) && num_seqs <= 65535 && num_heads <= 65535, PE_ERR_UNSUPPORTED,
             "prefill_window: grid too large");
  PE_REQUIRE(q_stride % 8 == 0 && k_stride % 8 == 0 && v_stride % 8 == 0 && out_stride % 8 == 0 && k_stride > 0 &&
                 v_stride > 0 && k_stride < (1 << 24) && v_stride < (1 << 24) &&
                 ((uintptr_t)out | (uintptr_t)q | (uintptr_t)k | (uintptr_t)v) % 16 == 0,
             PE_ERR_INVALID_ARG, "prefill_window: rows must be 16-byte aligned and k/v strides below 2^24 elements");
  if (sliding_window > (1 << 30)) sliding_window = 0;  // longer than any prompt: no window
  if (num_sinks > (1 << 30)) num_sinks = 1 << 30;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const float sl2 = scale * 1.4426950408889634f;
#define PE_LAUNCH_PW(T, HS, NR, WAVES, WPE)                                                             \
  do {                                                                                                  \
    const int bm = 16 * NR * WAVES;                                                                     \
    dim3 grid((unsigned)num_heads, (unsigned)num_seqs, (unsigned)((max_q_len + bm - 1) / bm));          \
    const size_t lds = 4 * (size_t)PF_BN * HS * 2;                                                      \
    if (lds > 64 * 1024)                                                                                \
      (void)hipFuncSetAttribute(                                                                        \
          reinterpret_cast<const void*>(&prefill_mfma_kernel<T, HS, NR, WAVES, WPE, true>),             \
          hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);                                        \
    hipLaunchKernelGGL((prefill_mfma_kernel<T, HS, NR, WAVES, WPE, true>), grid, dim3(WAVES * 64), lds, \
                       st, (T*)out, (const T*)q, (const T*)k, (const T*)v, cu_q, cu_kv, num_heads,      \
                       num_kv_heads, head_size, q_stride, k_stride, v_stride, out_stride, sl2,          \
                       sliding_window, num_sinks);                                                      \
  } while (0)
  PE_DISPATCH_16(dtype, T, {
    if (head_size <= 64) PE_LAUNCH_PW(T, 64, 2, 4, 2);
    else if (head_size <= 128) PE_LAUNCH_PW(T, 128, 2, 4, 2);
    else PE_LAUNCH_PW(T, 256, 1, 8, 2);
  });
#undef PE_LAUNCH_PW
  return check_launch("prefill_window");
}
