// Varlen causal prefill attention on gfx950: dispatch of the matrix-core kernel (prefill_kernel.h, with
// the description of the algorithm) and the general kernel.
#include "prefill_kernel.h"

namespace pe {

// Generic path: one wave per (query row, head); logits of the row in LDS.
template <typename T>
__global__ __launch_bounds__(64) void prefill_generic_kernel(
    T* __restrict__ out, const T* __restrict__ q, const T* __restrict__ k,
    const T* __restrict__ v, const int32_t* __restrict__ cu_q, const int32_t* __restrict__ cu_kv,
    int num_heads, int num_kv_heads, int head_size, int64_t q_stride, int64_t k_stride,
    int64_t v_stride, int64_t out_stride, float scale) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  float* qs = reinterpret_cast<float*>(smem);
  float* logits = qs + ((head_size + 3) & ~3);
  const int seq = blockIdx.z, head = blockIdx.y, i = blockIdx.x;
  const int kvh = head / (num_heads / num_kv_heads);
  const int q0 = cu_q[seq], lq = cu_q[seq + 1] - q0;
  const int kv0 = cu_kv[seq], lkv = cu_kv[seq + 1] - kv0;
  if (i >= lq) return;
  const int lane = threadIdx.x;
  const int n = min(i + 1, lkv);
  const T* qp = q + (int64_t)(q0 + i) * q_stride + (int64_t)head * head_size;
  for (int d = lane; d < head_size; d += 64) qs[d] = to_f32(qp[d]);
  __syncthreads();
  float mx = PF_NEG;
  for (int t = lane; t < n; t += 64) {
    const T* kp = k + (int64_t)(kv0 + t) * k_stride + (int64_t)kvh * head_size;
    float dot = 0.f;
    for (int d = 0; d < head_size; ++d) dot += qs[d] * to_f32(kp[d]);
    dot *= scale;
    logits[t] = dot;
    mx = fmaxf(mx, dot);
  }
  mx = wave_max(mx);
  float sum = 0.f;
  for (int t = lane; t < n; t += 64) {
    const float e = __expf(logits[t] - mx);
    logits[t] = e;
    sum += e;
  }
  sum = wave_sum(sum);
  __syncthreads();
  const float inv = sum > 0.f ? 1.f / sum : 0.f;
  T* op = out + (int64_t)(q0 + i) * out_stride + (int64_t)head * head_size;
  for (int d = lane; d < head_size; d += 64) {
    float a = 0.f;
    for (int t = 0; t < n; ++t)
      a += logits[t] * to_f32(v[(int64_t)(kv0 + t) * v_stride + (int64_t)kvh * head_size + d]);
    op[d] = from_f32<T>(a * inv);
  }
}

}  // namespace pe

extern "C" int pe_prefill_causal(void* out, const void* q, const void* k, const void* v,
                                 const int32_t* cu_q, const int32_t* cu_kv, int num_seqs,
                                 int max_q_len, int num_heads, int num_kv_heads, int head_size,
                                 int64_t q_stride, int64_t k_stride, int64_t v_stride,
                                 int64_t out_stride, float scale, int dtype, void* stream) {
  using namespace pe;
  PE_REQUIRE(num_seqs >= 0 && max_q_len >= 0, PE_ERR_INVALID_ARG, "prefill: negative size");
  if (num_seqs == 0 || max_q_len == 0) return PE_OK;
  PE_REQUIRE(out && q && k && v && cu_q && cu_kv, PE_ERR_INVALID_ARG, "prefill: null pointer");
  PE_REQUIRE(num_heads > 0 && num_kv_heads > 0 && num_heads % num_kv_heads == 0 && head_size > 0,
             PE_ERR_INVALID_ARG, "prefill: bad head layout");
  PE_REQUIRE(num_seqs <= 65535 && num_heads <= 65535, PE_ERR_UNSUPPORTED, "prefill: grid too large");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool hs_ok = head_size == 32 || head_size == 64 || head_size == 80 || head_size == 96 ||
                     head_size == 112 || head_size == 120 || head_size == 128 || head_size == 192 ||
                     head_size == 256;
  static EnvInt force_generic("PE_PREFILL_FORCE_GENERIC", 0);
  const bool mfma = (dtype == PE_BF16 || dtype == PE_F16) && hs_ok && !force_generic.get() &&
                    scale > 0.f && max_q_len / 64 < 65535 &&
                    k_stride > 0 && v_stride > 0 && k_stride < (1 << 24) && v_stride < (1 << 24) &&
                    q_stride % 8 == 0 && k_stride % 8 == 0 && v_stride % 8 == 0 &&
                    out_stride % 8 == 0 &&
                    (((uintptr_t)out | (uintptr_t)q | (uintptr_t)k | (uintptr_t)v) % 16 == 0);
  if (mfma) {
    // Tile shape <NR><WAVES> = rows per wave / waves per workgroup: 24 = 32 rows x 4 waves (128-row
    // workgroups, two per CU), 18 = 16 x 8 (128 rows, four waves per SIMD), 28 = 32 x 8 (256 rows,
    // one workgroup per CU), 14 = 16 x 4.  All give the same bits.  Measured on MI355X (32 query /
    // 8 KV heads x 128 unless noted, us per launch, 24 / 18 / 28): 32 x 256 tokens 53.8 / 49.4 / 69.3;
    // 16 x 512 70.4 / 68.0 / 83.8 (12 heads x 64: 20.9 / 19.5 / 21.4); 8 x 1024 100 / 104 / 117;
    // 8 x 1536 200 / 212 / 220; 8 x 2048 381 / - / 378; 8 x 4096 1243 / - / 1221; 8 x 8192 4238 / - / 4073;
    // 1 x 32768 7572 / - / 7292; 8 x 4096 with 8 query heads on 1 KV head 320 / 351 / 326; one
    // prompt alone, 24 / 14 / 28: 1 x 1024 26.3 / 25.0 / 33.9 (12 heads x 64: 19.7 / 12.6 / 24.9,
    // 8 heads on 1 KV head: 24.2 / 21.2 / 31.7), 2 x 1024 32.2 / 36.6 / 37.2, 1 x 4096
    // 177 / 224 / 167, 1 x 8192 581 / 780 / 568; 18 / 14: 1 x 512 15.6 / 13.2, 2 x 512 16.8 / 15.5.
    // So: a launch with no more 128-row tiles than the chip has CUs takes 64-row workgroups (twice
    // as many of them); other short prompts take the four-waves-per-SIMD shape (their workgroups
    // are mostly start-up and diagonal tiles, which more resident waves hide better); long prompts take the
    // 256-row shape (half the K/V tile traffic per flop) from 4096 tokens on with up to 4 query
    // heads per KV head, or from 2048 with enough tiles to fill the chip several times over;
    // everything else the 128-row default.  PE_PREFILL_SHAPE overrides (tuning runs).
    static EnvInt shape_env("PE_PREFILL_SHAPE", 0);
    int shape = shape_env.get();
    if (shape == 0) {
      const int64_t tiles256 = (int64_t)num_seqs * num_heads * ((max_q_len + 255) / 256);
      const int64_t tiles128 = (int64_t)num_seqs * num_heads * ((max_q_len + 127) / 128);
      if (tiles128 <= 256) shape = 14;
      else if (max_q_len <= 512) shape = 18;
      else if ((max_q_len >= 4096 && num_heads / num_kv_heads <= 4) ||
               (max_q_len >= 2048 && tiles256 >= 2048)) shape = 28;
      else shape = PF_DEFAULT_SHAPE;
    }
    const float sl2 = scale * 1.4426950408889634f;
#define PE_LAUNCH_PF(T, HS, NR, WAVES, WPE)                                                        \
  do {                                                                                             \
    const int bm = 16 * NR * WAVES;                                                                \
    dim3 grid((unsigned)num_heads, (unsigned)num_seqs, (unsigned)((max_q_len + bm - 1) / bm));     \
    const size_t lds = 4 * (size_t)PF_BN * HS * 2;                                                 \
    if (lds > 64 * 1024)                                                                           \
      (void)hipFuncSetAttribute(                                                                   \
          reinterpret_cast<const void*>(&prefill_mfma_kernel<T, HS, NR, WAVES, WPE>),              \
          hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);                                   \
    hipLaunchKernelGGL((prefill_mfma_kernel<T, HS, NR, WAVES, WPE>), grid, dim3(WAVES * 64), lds,  \
                       st, (T*)out, (const T*)q, (const T*)k, (const T*)v, cu_q, cu_kv, num_heads, \
                       num_kv_heads, head_size, q_stride, k_stride, v_stride, out_stride, sl2, 0, 0, 1, \
                       0, 0);                                                                      \
  } while (0)
#define PE_LAUNCH_PF_SHAPE(T, HS)                                                                  \
  do {                                                                                             \
    switch (shape) {                                                                               \
      case 18: PE_LAUNCH_PF(T, HS, 1, 8, 4); break;                                                \
      case 28: PE_LAUNCH_PF(T, HS, 2, 8, 2); break;                                                \
      case 14: PE_LAUNCH_PF(T, HS, 1, 4, 4); break;                                                \
      default: PE_LAUNCH_PF(T, HS, 2, 4, 2); break;                                                \
    }                                                                                              \
  } while (0)
    // row pitch 256 (head sizes 192, 256): four 64-row tiles of K and V take 128 KiB of LDS, so
    // one workgroup per CU - 8 waves x 16 rows, whose staging writes 16 tile rows per step
    PE_DISPATCH_16(dtype, T, {
      if (head_size <= 64) PE_LAUNCH_PF_SHAPE(T, 64);
      else if (head_size <= 128) PE_LAUNCH_PF_SHAPE(T, 128);
      else PE_LAUNCH_PF(T, 256, 1, 8, 2);
    });
#undef PE_LAUNCH_PF_SHAPE
#undef PE_LAUNCH_PF
    return check_launch("prefill_causal");
  }
  const size_t lds = (size_t)(((head_size + 3) & ~3) + max_q_len) * 4;
  PE_REQUIRE(lds <= 160 * 1024, PE_ERR_UNSUPPORTED,
             "generic prefill path keeps a row of logits in LDS: max_q_len %d too long", max_q_len);
  dim3 grid((unsigned)max_q_len, (unsigned)num_heads, (unsigned)num_seqs);
#define PE_LAUNCH_PFG(T)                                                                          \
  do {                                                                                            \
    if (lds > 64 * 1024)                                                                          \
      (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&prefill_generic_kernel<T>),        \
                                hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);            \
    hipLaunchKernelGGL(prefill_generic_kernel<T>, grid, dim3(64), lds, st, (T*)out, (const T*)q,   \
                       (const T*)k, (const T*)v, cu_q, cu_kv, num_heads, num_kv_heads, head_size,  \
                       q_stride, k_stride, v_stride, out_stride, scale);                          \
  } while (0)
  PE_DISPATCH_ALL(dtype, T, PE_LAUNCH_PFG(T));
#undef PE_LAUNCH_PFG
  return check_launch("prefill_generic");
}
