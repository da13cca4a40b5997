// KV write into the 8-bit paged cache (pe_reshape_and_cache_8bit).
//
//   value = code * s,  s = f32 per (block, KV head) of K and of V, a power of two:
//   need = 2^ceil(log2(max |x| / FMAX)) over the block's new (finite) elements,
//   s    = max(s_old, need),  s_old = 0 when the call writes the block's offset 0,
//   code = rn(x / s);  older codes of a block whose s grew:  code <- rn(code * s_old / s).
// With powers of two x / s is exact and a code is rounded once (under a caller's scale, which may be any
// number, x / s is rounded to f32 first); re-expressing e4m3 codes only rounds those that become subnormal.
//
// One workgroup owns one (sequence, block, KV head): the maximum over the block's new rows, the
// re-expression of its older codes and the scale are decided in one place, without atomics.  A wave
// takes four tokens x 16 chunks of 16 bytes (lane group g: token 4k + g), so rows come in 256-byte runs
// and the codes of a value row's four tokens meet in one dword by two row swaps and four byte permutes;
// the block goes through LDS in the cache's layout and is stored 16 bytes per lane.  The KV heads of a
// block are dispatched side by side: their pieces of a token's row lie side by side.
// Bound: HBM (2 bytes read, 1 written per element): 4 x 8192 rows of 8 x 128, int8, 39 us a pass (4.7 TB/s, a
// copy's rate; passes follow each other and share their start and end, a launch alone takes 43); a decode step
// (one row per sequence) by the chain of dependent loads lengths -> rows / table -> scale: 64 x 8 x 128, 4.9 us.
#include <type_traits>

#include "kv8.h"

namespace pe {

constexpr int w8_groups(int head_size) { return (head_size / 8 + 15) / 16; }            // chunk groups of a row
constexpr int w8_items(int head_size, int block_size) { return block_size / 4 * w8_groups(head_size); }
constexpr int w8_waves(int head_size, int block_size) {
  return w8_items(head_size, block_size) < 4 ? w8_items(head_size, block_size) : 4;
}

static __device__ unsigned int cache8_diag_word;

template <typename T, typename F, int D, int BLK>
__global__ __launch_bounds__(64 * w8_waves(D, BLK)) void cache8_write_kernel(
    const T* __restrict__ key, const T* __restrict__ value, uint8_t* __restrict__ key_cache,
    uint8_t* __restrict__ value_cache, float* __restrict__ kv_scales,
    const int32_t* __restrict__ block_tables, const int32_t* __restrict__ seq_lens,
    const int32_t* __restrict__ cu_q, int64_t num_tokens, int64_t key_stride, int64_t value_stride,
    int num_kv_heads, int64_t num_blocks, int table_width, int64_t kv_block_stride, int64_t kv_head_stride) {
  constexpr int CH = D / 8;                  // 16-byte chunks of a row
  constexpr int WAVES = w8_waves(D, BLK), THREADS = 64 * WAVES;
  constexpr int CG = w8_groups(D);
  constexpr int I = w8_items(D, BLK) / WAVES;  // (token quad, chunk group) pairs per wave
  // value image: rows of BLK bytes, 16 more after every 8 rows (spreads the dword writes over the banks)
  constexpr int V_IMG = D * BLK + D / 8 * 16;
  __shared__ __attribute__((aligned(16))) uint8_t k_img[D * BLK];
  __shared__ __attribute__((aligned(16))) uint8_t v_img[V_IMG];
  __shared__ uint32_t red[2][WAVES];
  const int h = blockIdx.x, seq = blockIdx.z, tid = threadIdx.x;
  const int lane = tid & 63, wave = tid >> 6, g = lane >> 4, c16 = lane & 15;
  const int64_t row0 = cu_q ? cu_q[seq] : seq;
  const int64_t row1 = cu_q ? cu_q[seq + 1] : seq + 1;
  const int64_t len = seq_lens[seq];
  if (len <= 0 || row1 <= row0) return;
  // lengths that do not fit together (more new rows than the sequence's length, rows past the
  // tensors, a length past the table row): nothing of the sequence is written
  if (row0 < 0 || row1 > num_tokens || row1 - row0 > len || len > (int64_t)table_width * BLK) {
    if (tid == 0) atomicOr(&cache8_diag_word, (unsigned)PE_DIAG_APPEND_MISMATCH);
    return;
  }
  const int64_t ctx = len - (row1 - row0);

  for (int64_t j = ctx / BLK + blockIdx.y; j * BLK < len; j += gridDim.y) {
    const int o0 = (int)(j * BLK > ctx ? 0 : ctx - j * BLK);                  // first new slot
    const int o1 = (int)((j + 1) * BLK < len ? (int64_t)BLK : len - j * BLK);  // behind the last one
    const int blk = block_tables[(int64_t)seq * table_width + j];

    // ---- the new rows, kept in registers; the largest finite magnitudes ----------------------
    u32x4 kr[I], vr[I];
    uint32_t ka = 0, va = 0;
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const int item = wave * I + i, slot = item / CG * 4 + g, c = item % CG * 16 + c16;
      kr[i] = vr[i] = u32x4{0u, 0u, 0u, 0u};
      if (slot >= o0 && slot < o1 && c < CH) {
        const int64_t row = row0 + (j * BLK + slot - ctx);
        kr[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(key + row * key_stride + (int64_t)h * D + c * 8));
        vr[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(value + row * value_stride + (int64_t)h * D + c * 8));
      }
    }
    if (blk < 0 || blk >= num_blocks) {  // workgroup-uniform
      if (tid == 0) atomicOr(&cache8_diag_word, (unsigned)PE_DIAG_BLOCK_ID);
      continue;
    }
    float* sc = kv_scales + ((int64_t)blk * num_kv_heads + h) * 2;
    const float ks_old = o0 ? sc[0] : 0.f, vs_old = o0 ? sc[1] : 0.f;  // (requested before the maxima)
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        ka = max(ka, max(finite_bits<T>(kr[i][e] & 0xffffu), finite_bits<T>(kr[i][e] >> 16)));
        va = max(va, max(finite_bits<T>(vr[i][e] & 0xffffu), finite_bits<T>(vr[i][e] >> 16)));
      }
    // (both are 16-bit magnitudes: one word carries the two maxima through the wave)
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) {
      const uint32_t other = (uint32_t)__shfl_xor((int)(ka | va << 16), x);
      ka = max(ka, other & 0xffffu);
      va = max(va, other >> 16);
    }
    if (lane == 0) {
      red[0][wave] = ka;
      red[1][wave] = va;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      ka = max(ka, red[0][w]);
      va = max(va, red[1][w]);
    }
    const Joined kj = join_scale<F>(o0 > 0, ks_old, bits_value<T>(ka));
    const Joined vj = join_scale<F>(o0 > 0, vs_old, bits_value<T>(va));

    uint8_t* kb = key_cache + blk * kv_block_stride + (int64_t)h * kv_head_stride;
    uint8_t* vb = value_cache + blk * kv_block_stride + (int64_t)h * kv_head_stride;
    // ---- older codes at the grown scale (rare: a row larger than everything before it) --------
    if (kj.grew) {
      for (int it = tid; it < D / 16 * o0 * 4; it += THREADS)
        reencode_word<F>(reinterpret_cast<uint32_t*>(kb + it / (o0 * 4) * (BLK * 16)) + it % (o0 * 4), kj.factor());
    }
    if (vj.grew) {
      for (int it = tid; it < D * o0; it += THREADS) reencode_byte<F>(vb + it / o0 * BLK + it % o0, vj.factor());
    }
    if (tid == 0) {
      sc[0] = kj.scale;
      sc[1] = vj.scale;
    }
    // ---- the new codes ------------------------------------------------------------------------
    const bool whole = o0 == 0 && o1 == BLK;
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const int item = wave * I + i, slot = item / CG * 4 + g, c = item % CG * 16 + c16;
      auto enc = [&](const u32x4& r, const Joined& j, auto exact) {
        constexpr bool EXACT = decltype(exact)::value;
        float f[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f[2 * e] = j.divide<EXACT>(bits_value<T>(r[e] & 0xffffu));
          f[2 * e + 1] = j.divide<EXACT>(bits_value<T>(r[e] >> 16));
        }
        return u32x2{encode4<F>(f[0], f[1], f[2], f[3]), encode4<F>(f[4], f[5], f[6], f[7])};
      };
      u32x2 kc = enc(kr[i], kj, std::true_type{}), vc = enc(vr[i], vj, std::true_type{});
      const int k_at = ((c >> 1) * BLK + slot) * 16 + (c & 1) * 8;
      if (whole) {
        // 8 elements x 4 tokens of a chunk, spread over the four lane groups -> two dwords per lane:
        // elements 2g and 2g + 1, four tokens each
        const auto x = __builtin_amdgcn_permlane32_swap(vc[0], vc[1], false, false);
        // groups 0, 1: elements 0-3 of tokens g, g + 2; groups 2, 3: elements 4-7 of tokens g - 2, g
        const uint32_t p = __builtin_amdgcn_perm(x[1], x[0], 0x05010400u), q = __builtin_amdgcn_perm(x[1], x[0], 0x07030602u);
        const auto y = __builtin_amdgcn_permlane16_swap(p, q, false, false);
        const uint32_t d0 = __builtin_amdgcn_perm(y[1], y[0], 0x05010400u), d1 = __builtin_amdgcn_perm(y[1], y[0], 0x07030602u);
        if (c < CH) {
          *reinterpret_cast<u32x2*>(k_img + k_at) = kc;
          uint32_t* v = reinterpret_cast<uint32_t*>(v_img + (c * 8 + 2 * g) * BLK + c * 16 + item / CG * 4);
          v[0] = d0;
          v[BLK / 4] = d1;
        }
      } else if (slot >= o0 && slot < o1 && c < CH) {
        // (only a block with older rows has a scale from elsewhere)
        if (!kj.exact) kc = enc(kr[i], kj, std::false_type{});
        if (!vj.exact) vc = enc(vr[i], vj, std::false_type{});
        *reinterpret_cast<u32x2*>(kb + k_at) = kc;
#pragma unroll
        for (int e = 0; e < 8; ++e) vb[(c * 8 + e) * BLK + slot] = (uint8_t)(vc[e >> 2] >> (8 * (e & 3)));
      }
    }
    __syncthreads();  // images complete; the next block's maxima may overwrite `red`
    if (whole) {
      for (int it = tid; it < D * BLK / 16; it += THREADS) {
        // (8 value rows are BLK / 2 pieces of 16 bytes.  Rows in and codes out pass the caches once: with the
        //  non-temporal hint 39.1 us, without 41.9)
        __builtin_nontemporal_store(reinterpret_cast<const u32x4*>(k_img)[it], reinterpret_cast<u32x4*>(kb) + it);
        __builtin_nontemporal_store(reinterpret_cast<const u32x4*>(v_img)[it + it / (BLK / 2)],
                                    reinterpret_cast<u32x4*>(vb) + it);
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
  // blocks a sequence touches (the kernel goes on in strides of the grid where there are more)
  const int64_t most = max_q_len == 1 ? 1 : ((int64_t)max_q_len + block_size - 2) / block_size + 1;
  dim3 grid((unsigned)num_kv_heads, (unsigned)(most < 65535 ? most : 65535), (unsigned)num_seqs);
  hipStream_t st = static_cast<hipStream_t>(stream);
#define PE_W8(T, F, D, BLK)                                                                               \
  hipLaunchKernelGGL((cache8_write_kernel<T, F, D, BLK>), grid, dim3(64 * w8_waves(D, BLK)), 0, st,       \
                     (const T*)key, (const T*)value, (uint8_t*)key_cache, (uint8_t*)value_cache,          \
                     kv_scales, block_tables, seq_lens, cu_q, num_tokens, key_stride, value_stride,       \
                     num_kv_heads, num_blocks, max_num_blocks_per_seq, kv_block_stride, kv_head_stride)
#define PE_W8_BLK(T, F, D)                  \
  case D:                                   \
    if (block_size == 8) PE_W8(T, F, D, 8); \
    else if (block_size == 16) PE_W8(T, F, D, 16); \
    else PE_W8(T, F, D, 32);                \
    break
#define PE_W8_D(T, F)                                                                                     \
  switch (head_size) {                                                                                    \
    PE_W8_BLK(T, F, 32); PE_W8_BLK(T, F, 64); PE_W8_BLK(T, F, 80); PE_W8_BLK(T, F, 96);                   \
    PE_W8_BLK(T, F, 112); PE_W8_BLK(T, F, 128); PE_W8_BLK(T, F, 192); PE_W8_BLK(T, F, 256);               \
  }
  PE_DISPATCH_16(dtype, T, {
    if (kv_format == PE_KV_FP8_E4M3) PE_W8_D(T, Fp8)
    else PE_W8_D(T, Int8)
  });
#undef PE_W8_D
#undef PE_W8_BLK
#undef PE_W8
  return check_launch("reshape_and_cache_8bit");
}
