// KV write into the 8-bit paged cache (pe_reshape_and_cache_8bit).
//
//   value = code * s,  s = f32 per (block, KV head) of K and of V, a power of two:
//   need = 2^ceil(log2(max |x| / FMAX)) over the block's new (finite) elements,
//   s    = max(s_old, need),  s_old = 0 when the call writes the block's offset 0,
//   code = rn(x / s);  older codes of a block whose s grew:  code <- rn(code * s_old / s).
// With powers of two x / s is exact and a code is rounded once; re-expressing e4m3 codes only
// rounds those that become subnormal.
//
// One workgroup owns one (sequence, block, KV head): the maximum over the block's new rows, the
// re-expression of its older codes and the scale are decided in one place, without atomics.
// Bound: HBM (2 bytes read, 1 written per element); a decode step (one row per sequence) by the
// chain of dependent loads lengths -> table -> scale / rows.
#include "kv8.h"

namespace pe {

constexpr int W8_THREADS = 256;

static __device__ unsigned int cache8_diag_word;

// I: 16-byte chunks of a block's new K (or V) rows per thread = block_size * head_size / 8 / 256
template <typename T, typename F, int I>
__global__ __launch_bounds__(W8_THREADS) void cache8_write_kernel(
    const T* __restrict__ key, const T* __restrict__ value, uint8_t* __restrict__ key_cache,
    uint8_t* __restrict__ value_cache, float* __restrict__ kv_scales,
    const int32_t* __restrict__ block_tables, const int32_t* __restrict__ seq_lens,
    const int32_t* __restrict__ cu_q, int64_t num_tokens, int64_t key_stride, int64_t value_stride,
    int num_kv_heads, int head_size, int block_size, int64_t num_blocks, int table_width,
    int64_t kv_block_stride, int64_t kv_head_stride) {
  extern __shared__ __attribute__((aligned(16))) uint8_t w8_smem[];  // K image, V image of the block
  __shared__ uint32_t red[2][W8_THREADS / 64];
  const int seq = blockIdx.z, h = blockIdx.y, tid = threadIdx.x;
  const int64_t row0 = cu_q ? cu_q[seq] : seq;
  const int64_t row1 = cu_q ? cu_q[seq + 1] : seq + 1;
  const int64_t len = seq_lens[seq];
  if (len <= 0 || row1 <= row0) return;
  // lengths that do not fit together (more new rows than the sequence's length, rows past the
  // tensors, a length past the table row): nothing of the sequence is written
  if (row0 < 0 || row1 > num_tokens || row1 - row0 > len || len > (int64_t)table_width * block_size) {
    if (tid == 0) atomicOr(&cache8_diag_word, (unsigned)PE_DIAG_APPEND_MISMATCH);
    return;
  }
  const int64_t ctx = len - (row1 - row0);
  const int CH = head_size >> 3;  // 16-byte chunks of a row
  uint8_t* const k_img = w8_smem;
  uint8_t* const v_img = w8_smem + block_size * head_size;

  for (int64_t j = ctx / block_size + blockIdx.x; j * block_size < len; j += gridDim.x) {
    const int64_t p0 = j * block_size > ctx ? j * block_size : ctx;
    const int64_t p1 = (j + 1) * block_size < len ? (j + 1) * block_size : len;
    const int o0 = (int)(p0 - j * block_size), m = (int)(p1 - p0);  // first offset, new rows
    const int64_t blk = block_tables[(int64_t)seq * table_width + j];
    if (blk < 0 || blk >= num_blocks) {  // workgroup-uniform
      if (tid == 0) atomicOr(&cache8_diag_word, (unsigned)PE_DIAG_BLOCK_ID);
      continue;
    }
    float* sc = kv_scales + (blk * num_kv_heads + h) * 2;
    const float ks_old = o0 ? sc[0] : 0.f, vs_old = o0 ? sc[1] : 0.f;

    // ---- the new rows, kept in registers; the largest finite magnitudes ----------------------
    u32x4 kr[I], vr[I];
    uint32_t ka = 0, va = 0;
    const int64_t r0 = row0 + (p0 - ctx);
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const int it = tid + i * W8_THREADS;
      kr[i] = vr[i] = u32x4{0u, 0u, 0u, 0u};
      if (it < m * CH) {
        const int64_t row = r0 + it / CH;
        const int c = it % CH;
        kr[i] = *reinterpret_cast<const u32x4*>(key + row * key_stride + (int64_t)h * head_size + c * 8);
        vr[i] = *reinterpret_cast<const u32x4*>(value + row * value_stride + (int64_t)h * head_size + c * 8);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        ka = max(ka, max(finite_bits<T>(kr[i][e] & 0xffffu), finite_bits<T>(kr[i][e] >> 16)));
        va = max(va, max(finite_bits<T>(vr[i][e] & 0xffffu), finite_bits<T>(vr[i][e] >> 16)));
      }
    }
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) {
      ka = max(ka, (uint32_t)__shfl_xor((int)ka, x));
      va = max(va, (uint32_t)__shfl_xor((int)va, x));
    }
    if ((tid & 63) == 0) {
      red[0][tid >> 6] = ka;
      red[1][tid >> 6] = va;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W8_THREADS / 64; ++w) {
      ka = max(ka, red[0][w]);
      va = max(va, red[1][w]);
    }
    const float ks = fmaxf(ks_old, pow2_scale<F>(bits_value<T>(ka)));
    const float vs = fmaxf(vs_old, pow2_scale<F>(bits_value<T>(va)));
    // exact for powers of two (a scale of 0 has no finite element but zeros to divide)
    const float ki = ks > 0.f ? 1.f / ks : 1.f, vi = vs > 0.f ? 1.f / vs : 1.f;

    uint8_t* kb = key_cache + blk * kv_block_stride + (int64_t)h * kv_head_stride;
    uint8_t* vb = value_cache + blk * kv_block_stride + (int64_t)h * kv_head_stride;
    // ---- older codes at the grown scale (rare: a row larger than everything before it) --------
    if (ks_old > 0.f && ks > ks_old) {
      const float f = ks_old * ki;
      for (int it = tid; it < (head_size >> 4) * o0 * 4; it += W8_THREADS) {
        const int c = it / (o0 * 4), w = it % (o0 * 4);
        reencode_word<F>(reinterpret_cast<uint32_t*>(kb + c * block_size * 16) + w, f);
      }
    }
    if (vs_old > 0.f && vs > vs_old) {
      const float f = vs_old * vi;
      for (int it = tid; it < head_size * o0; it += W8_THREADS)
        reencode_byte<F>(vb + (it / o0) * block_size + it % o0, f);
    }
    if (tid == 0) {
      sc[0] = ks;
      sc[1] = vs;
    }
    // ---- the new codes ------------------------------------------------------------------------
    const bool whole = m == block_size;
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const int it = tid + i * W8_THREADS;
      if (it >= m * CH) continue;
      const int off = o0 + it / CH, c = it % CH;
      auto enc = [&](const u32x4& r, float inv) {
        float f[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f[2 * e] = bits_value<T>(r[e] & 0xffffu) * inv;
          f[2 * e + 1] = bits_value<T>(r[e] >> 16) * inv;
        }
        return u32x2{encode4<F>(f[0], f[1], f[2], f[3]), encode4<F>(f[4], f[5], f[6], f[7])};
      };
      const u32x2 kc = enc(kr[i], ki), vc = enc(vr[i], vi);
      const int k_at = ((c >> 1) * block_size + off) * 16 + (c & 1) * 8;
      if (whole) {
        *reinterpret_cast<u32x2*>(k_img + k_at) = kc;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          v_img[(c * 8 + e) * block_size + off] = (uint8_t)(vc[e >> 2] >> (8 * (e & 3)));
      } else {
        *reinterpret_cast<u32x2*>(kb + k_at) = kc;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          vb[(c * 8 + e) * block_size + off] = (uint8_t)(vc[e >> 2] >> (8 * (e & 3)));
      }
    }
    __syncthreads();  // images complete; the next block's maxima may overwrite `red`
    if (whole) {
      for (int it = tid; it < block_size * head_size / 16; it += W8_THREADS) {
        reinterpret_cast<u32x4*>(kb)[it] = reinterpret_cast<const u32x4*>(k_img)[it];
        reinterpret_cast<u32x4*>(vb)[it] = reinterpret_cast<const u32x4*>(v_img)[it];
      }
      __syncthreads();
    }
  }
}

int cache8_diag_fetch(unsigned int* out, int reset) {
  void* p = nullptr;
  hipError_t e = hipGetSymbolAddress(&p, HIP_SYMBOL(cache8_diag_word));
  if (e == hipSuccess) e = hipMemcpy(out, p, sizeof(unsigned int), hipMemcpyDeviceToHost);
  if (e == hipSuccess && reset && *out != 0) e = hipMemset(p, 0, sizeof(unsigned int));
  if (e != hipSuccess) return fail(PE_ERR_LAUNCH, "8-bit cache diagnostics: %s", hipGetErrorString(e));
  return PE_OK;
}

}  // namespace pe

extern "C" int pe_reshape_and_cache_8bit(
    const void* key, const void* value, void* key_cache, void* value_cache, float* kv_scales,
    const int32_t* block_tables, const int32_t* seq_lens, const int32_t* cu_q, int num_seqs,
    int64_t num_tokens, int max_q_len, int64_t key_stride, int64_t value_stride, int num_kv_heads,
    int head_size, int block_size, int64_t num_blocks, int max_num_blocks_per_seq,
    int64_t kv_block_stride, int64_t kv_head_stride, int dtype, int kv_format, void* stream) {
  using namespace pe;
  PE_REQUIRE(num_seqs >= 0 && num_tokens >= 0 && max_q_len >= 0, PE_ERR_INVALID_ARG,
             "reshape_and_cache_8bit: negative size");
  if (num_seqs == 0 || num_tokens == 0 || max_q_len == 0) return PE_OK;
  PE_REQUIRE(key && value && key_cache && value_cache && kv_scales && block_tables && seq_lens,
             PE_ERR_INVALID_ARG, "reshape_and_cache_8bit: null pointer");
  if (int rc = check_cache8("reshape_and_cache_8bit", key_cache, value_cache, kv_scales, num_kv_heads,
                            head_size, block_size, num_blocks, max_num_blocks_per_seq, kv_block_stride,
                            kv_head_stride, dtype, kv_format))
    return rc;
  PE_REQUIRE(cu_q || num_tokens >= num_seqs, PE_ERR_INVALID_ARG,
             "reshape_and_cache_8bit: without cu_q there is one row per sequence (%lld rows, %d sequences)",
             (long long)num_tokens, num_seqs);
  PE_REQUIRE(key_stride % 8 == 0 && value_stride % 8 == 0 && ((uintptr_t)key | (uintptr_t)value) % 16 == 0,
             PE_ERR_INVALID_ARG, "reshape_and_cache_8bit: key/value rows must be 16-byte aligned");
  PE_REQUIRE(num_seqs <= 65535 && num_kv_heads <= 65535, PE_ERR_UNSUPPORTED, "reshape_and_cache_8bit: grid too large");
  const int most = max_q_len == 1 ? 1 : (max_q_len + block_size - 2) / block_size + 1;  // blocks a sequence touches
  dim3 grid((unsigned)most, (unsigned)num_kv_heads, (unsigned)num_seqs);
  const size_t lds = 2 * (size_t)block_size * head_size;
  hipStream_t st = static_cast<hipStream_t>(stream);
#define PE_W8(T, F, I)                                                                               \
  hipLaunchKernelGGL((cache8_write_kernel<T, F, I>), grid, dim3(W8_THREADS), lds, st, (const T*)key, \
                     (const T*)value, (uint8_t*)key_cache, (uint8_t*)value_cache, kv_scales,         \
                     block_tables, seq_lens, cu_q, num_tokens, key_stride, value_stride,             \
                     num_kv_heads, head_size, block_size, num_blocks, max_num_blocks_per_seq,        \
                     kv_block_stride, kv_head_stride)
#define PE_W8_I(T, F)                                                     \
  do {                                                                    \
    const int chunks = block_size * head_size / 8;                        \
    if (chunks <= W8_THREADS) PE_W8(T, F, 1);                             \
    else if (chunks <= 2 * W8_THREADS) PE_W8(T, F, 2);                    \
    else PE_W8(T, F, 4);                                                  \
  } while (0)
  PE_DISPATCH_16(dtype, T, {
    if (kv_format == PE_KV_FP8_E4M3) PE_W8_I(T, Fp8);
    else PE_W8_I(T, Int8);
  });
#undef PE_W8_I
#undef PE_W8
  return check_launch("reshape_and_cache_8bit");
}
