// Varlen prefill attention with a sliding window and sink tokens (pe_prefill_window): dispatch of the
// windowed form of the matrix-core kernel in prefill_kernel.h.
#include "prefill_kernel.h"

extern "C" int pe_prefill_window(void* out, const void* q, const void* k, const void* v,
                                 const int32_t* cu_q, const int32_t* cu_kv, int num_seqs,
                                 int max_q_len, int64_t num_q_rows, int64_t num_kv_rows,
                                 int num_heads, int num_kv_heads, int head_size,
                                 int64_t q_stride, int64_t k_stride, int64_t v_stride,
                                 int64_t out_stride, float scale, int sliding_window, int num_sinks,
                                 int dtype, void* stream) {
  using namespace pe;
  PE_REQUIRE(num_seqs >= 0 && max_q_len >= 0 && num_q_rows >= 0 && num_kv_rows >= 0, PE_ERR_INVALID_ARG,
             "prefill_window: negative size");
  PE_REQUIRE(sliding_window >= 0 && num_sinks >= 0, PE_ERR_INVALID_ARG,
             "prefill_window: sliding_window %d and num_sinks %d must not be negative", sliding_window, num_sinks);
  if (num_seqs == 0 || max_q_len == 0 || num_q_rows == 0) return PE_OK;
  // (without kv rows k and v are not read, and an empty tensor has no address)
  PE_REQUIRE(out && q && (num_kv_rows == 0 || (k && v)) && cu_q && cu_kv, PE_ERR_INVALID_ARG,
             "prefill_window: null pointer");
  PE_REQUIRE(num_heads > 0 && num_kv_heads > 0 && num_heads % num_kv_heads == 0, PE_ERR_INVALID_ARG,
             "prefill_window: num_heads %d must be a positive multiple of num_kv_heads %d", num_heads, num_kv_heads);
  PE_REQUIRE(head_size == 32 || head_size == 64 || head_size == 80 || head_size == 96 || head_size == 112 ||
                 head_size == 120 || head_size == 128 || head_size == 192 || head_size == 256,
             PE_ERR_UNSUPPORTED, "prefill_window: head size %d is not built", head_size);
  PE_REQUIRE(dtype == PE_BF16 || dtype == PE_F16, PE_ERR_UNSUPPORTED, "prefill_window: dtype %d (bf16 or f16)", dtype);
  // the maxima are kept in scaled units
  PE_REQUIRE(scale > 0.f && scale < INFINITY, PE_ERR_UNSUPPORTED, "prefill_window: scale must be positive and finite");
  // (the prefix sums are int32: rows past 2^31 - 1 belong to no request)
  if (num_q_rows > INT32_MAX) num_q_rows = INT32_MAX;
  if (num_kv_rows > INT32_MAX) num_kv_rows = INT32_MAX;
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
  // Tile shape: 16 x NR query rows per wave, 4 waves (8 at the 256 pitch), BN keys per tile; the waves
  // take the query heads of a KV head side by side (hpw of them; fewer where the blocks of 16 * NR * waves / hpw
  // rows would be more than the 65535 of a grid dimension).  Measured on MI355X (us per pass, passes over
  // three sets of inputs replayed from a graph; NR x BN = 2 x 64 / 1 x 64 / 1 x 32; 32 query and 8 KV heads x 128
  // unless given, 4 sinks; none = no window):
  //   8 x 1024 tokens, window 64: 58 / 67 / 46, 128: 63 / 74 / 54, 256: 73 / 86 / 68, 384: 79 / 96 / 79,
  //   none: 91 / 112 / 100; 4 x 4096, window 64: 114 / 138 / 92, 256: 154 / 189 / 147, 512: 204 / 254 / 225,
  //   none: 568 / 708 / 676; 1 x 512, window 64: 12.1 / 8.4 / 8.3, 256: 16.7 / 11.6 / 12.8, none: 18.1 / 13.0 / 16.4;
  //   12 heads x 64, 8 x 1024, window 64: 25 / 17 / 18, 256: 30 / 21 / 24, none: 31 / 26 / 31; 1 x 8192, window 256:
  //   34 / 26 / 29, 1024: 61 / 51 / 62; 32 / 8 heads x 64, 4 x 8192, window 256: 215 / 187 / 197, 1024: 433 / 405 / 467,
  //   none: 1377 / 1364 / 1641.
  // So: head sizes up to 64, and launches that leave CUs idle, take the 1 x 64 shape (more and smaller
  // workgroups; at 64 elements a key costs half the LDS reads); rows that see few keys the 1 x 32 shape, whose
  // tiles waste less at the window's two ends; everything else 2 x 64, which reads each K/V fragment from
  // LDS once for 32 rows.
  const int gqa = num_heads / num_kv_heads;
  const int64_t span = sliding_window > 0 ? (int64_t)sliding_window + num_sinks : max_q_len;
  const int64_t wgs = (int64_t)num_seqs * num_heads * ((max_q_len + 127) / 128);  // of 2 x 64
#define PE_LAUNCH_PW(T, HS, NR, WAVES, WPE, BN)                                                         \
  do {                                                                                                  \
    int hpw = WAVES;                                                                                    \
    auto row_blocks = [&] { return (max_q_len + 16 * NR * WAVES / hpw - 1) / (16 * NR * WAVES / hpw); }; \
    while (gqa % hpw || (hpw > 1 && row_blocks() > 65535)) hpw /= 2;                                    \
    PE_REQUIRE(row_blocks() <= 65535, PE_ERR_UNSUPPORTED, "prefill_window: grid too large");             \
    dim3 grid((unsigned)(num_heads / hpw), (unsigned)num_seqs, (unsigned)row_blocks());                 \
    const size_t lds = 4 * (size_t)BN * HS * 2;                                                         \
    if (lds > 64 * 1024)                                                                                \
      (void)hipFuncSetAttribute(                                                                        \
          reinterpret_cast<const void*>(&prefill_mfma_kernel<T, HS, NR, WAVES, WPE, true, BN>),         \
          hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);                                        \
    hipLaunchKernelGGL((prefill_mfma_kernel<T, HS, NR, WAVES, WPE, true, BN>), grid, dim3(WAVES * 64),  \
                       lds, st, (T*)out, (const T*)q, (const T*)k, (const T*)v, cu_q, cu_kv, num_heads, \
                       num_kv_heads, head_size, q_stride, k_stride, v_stride, out_stride, sl2,          \
                       sliding_window, num_sinks, hpw, (int)num_q_rows, (int)num_kv_rows);              \
  } while (0)
  PE_DISPATCH_16(dtype, T, {
    if (head_size <= 64) PE_LAUNCH_PW(T, 64, 1, 4, 2, 64);
    else if (head_size > 128) PE_LAUNCH_PW(T, 256, 1, 8, 2, 64);
    else if (wgs <= 256) PE_LAUNCH_PW(T, 128, 1, 4, 2, 64);
    else if (span <= 288) PE_LAUNCH_PW(T, 128, 1, 4, 4, 32);
    else PE_LAUNCH_PW(T, 128, 2, 4, 2, 64);
  });
#undef PE_LAUNCH_PW
  return check_launch("prefill_window");
}
