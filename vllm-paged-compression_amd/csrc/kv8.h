// Element formats of the 8-bit paged cache (value = code * scale, one f32 scale per block, KV head
// and tensor) and their conversions.  e4m3 (largest value 448) and int8 (codes -127 .. 127): every
// code is exact in bf16 and in f16, so the matrix instructions of the 16-bit types multiply the
// codes themselves and the scales are applied to f32 results.
#pragma once
#include "pe_common.h"

namespace pe {

// diagnostic words behind pe_device_diagnostics (defined in paged_window.hip / cache_8bit.hip)
int window_diag_fetch(unsigned int* out, int reset);
int cache8_diag_fetch(unsigned int* out, int reset);

struct Fp8 {  // e4m3: 1 sign, 4 exponent, 3 mantissa bits; 0x7f / 0xff are NaN, no infinities
  static constexpr float MAX = 448.f;
  // 448 = 1.75 * 2^8: a scale 2^k holds amax = m * 2^e (1 <= m < 2) when k >= e - 8 + (m > 1.75)
  static constexpr int MAX_EXP = 8;
  static constexpr uint32_t MAX_MANT = 0x600000u;  // mantissa bits of 1.75f
};
struct Int8 {
  static constexpr float MAX = 127.f;
  static constexpr int MAX_EXP = 6;                // 127 = 1.984375 * 2^6
  static constexpr uint32_t MAX_MANT = 0x7e0000u;  // mantissa bits of 1.984375f
};

typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;

// two codes (the low or the high half of a dword) -> two values of T, exactly
template <typename T, typename F, bool HI>
__device__ __forceinline__ uint32_t codes_pair(uint32_t w) {
  if constexpr (__is_same(F, Fp8)) {
    if constexpr (__is_same(T, __bf16))
      return __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
    else
      return __builtin_bit_cast(uint32_t, (f16x2)__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
  } else {
    const int lo = (int)(int8_t)(w >> (HI ? 16 : 0)), hi = (int)(int8_t)(w >> (HI ? 24 : 8));
    if constexpr (__is_same(T, __bf16))
      return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)(float)lo, (__bf16)(float)hi});
    else
      return __builtin_bit_cast(uint32_t, f16x2{(_Float16)(float)lo, (_Float16)(float)hi});
  }
}
// eight codes -> a matrix operand of T
template <typename T, typename F>
__device__ __forceinline__ typename Traits<T>::vec8 codes8(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(typename Traits<T>::vec8,
                            u32x4{codes_pair<T, F, false>(a), codes_pair<T, F, true>(a),
                                  codes_pair<T, F, false>(b), codes_pair<T, F, true>(b)});
}

template <typename F>
__device__ __forceinline__ float code_value(uint32_t byte) {
  if constexpr (__is_same(F, Fp8)) return __builtin_amdgcn_cvt_f32_fp8((int)byte, 0);
  else return (float)(int)(int8_t)byte;
}

// f32 values, already divided by the scale -> codes: one rounding to nearest even (half a step:
// 2^-4 of the value in e4m3, half a unit in int8), infinities to the largest code; a NaN stays a
// NaN in e4m3 and becomes 0 in int8, which has none
template <typename F>
__device__ __forceinline__ float clamp_code(float x) {
  const float c = __builtin_amdgcn_fmed3f(x, -F::MAX, F::MAX);
  if constexpr (__is_same(F, Fp8)) return x != x ? x : c;
  else return x != x ? 0.f : c;
}
template <typename F>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  a = clamp_code<F>(a);
  b = clamp_code<F>(b);
  c = clamp_code<F>(c);
  d = clamp_code<F>(d);
  if constexpr (__is_same(F, Fp8)) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  } else {
    const uint32_t i0 = (uint32_t)(int)__builtin_rintf(a) & 255u, i1 = (uint32_t)(int)__builtin_rintf(b) & 255u;
    const uint32_t i2 = (uint32_t)(int)__builtin_rintf(c) & 255u, i3 = (uint32_t)(int)__builtin_rintf(d) & 255u;
    return i0 | (i1 << 8) | (i2 << 16) | (i3 << 24);
  }
}

// older codes of a block whose scale grew, f = old scale / new scale
template <typename F>
__device__ __forceinline__ void reencode_word(uint32_t* p, float f) {
  const uint32_t q = *p;
  *p = encode4<F>(code_value<F>(q & 255u) * f, code_value<F>((q >> 8) & 255u) * f,
                  code_value<F>((q >> 16) & 255u) * f, code_value<F>(q >> 24) * f);
}
template <typename F>
__device__ __forceinline__ void reencode_byte(uint8_t* p, float f) {
  *p = (uint8_t)encode4<F>(code_value<F>(*p) * f, 0.f, 0.f, 0.f);
}

// smallest power of two s with amax / s <= F::MAX, at least 2^-100 (its reciprocal and the
// quotients stay far from f32's ends); 0 for amax = 0.  amax is finite and not negative.
template <typename F>
__device__ __forceinline__ float pow2_scale(float amax) {
  if (amax == 0.f) return 0.f;
  const uint32_t u = __float_as_uint(amax);
  // a subnormal amax has a biased exponent of 0 and ends at the floor like its neighbours
  int k = (int)(u >> 23) - 127 - F::MAX_EXP + ((u & 0x7fffffu) > F::MAX_MANT ? 1 : 0);
  if (k < -100) k = -100;
  return __uint_as_float((uint32_t)(k + 127) << 23);
}

// The scale of a block that new rows join, 1 / scale, and what its older codes are multiplied by where the
// scale grew.  `older`: the block has rows in front of the new ones; without them it begins anew, and what
// memory holds as its scale does not count.  A scale of 0 stands for elements that all read as 0 (rows of
// zeros and infinities leave non-zero codes under it): once it grows, the older codes become 0.
// All arguments are the same in every lane of the wave.
struct Joined {
  float old, scale, inv;
  bool grew, exact;
  __device__ __forceinline__ float factor() const { return old * inv; }
  // x / scale, rounded once to f32.  Scales that a write chose are powers of two (and a scale of 0 has no finite
  // element but zeros to divide): x times 1 / scale is the quotient itself.  A cache made elsewhere may hold any
  // scale, also one whose 1 / scale is rounded or past f32's largest number.
  // (EXACT: the caller has looked)
  template <bool EXACT>
  __device__ __forceinline__ float divide(float x) const {
    return EXACT || exact ? x * inv : x / scale;
  }
};
template <typename F>
__device__ __forceinline__ Joined join_scale(bool older, float stored, float amax) {
  Joined j;
  j.old = older ? stored : 0.f;
  j.scale = fmaxf(j.old, pow2_scale<F>(amax));
  j.inv = j.scale > 0.f ? 1.f / j.scale : 1.f;
  j.exact = __builtin_amdgcn_readfirstlane((int)(__float_as_uint(j.scale) & 0x7fffffu)) == 0;  // 0, or 2^k >= 2^-126
  j.grew = older && j.scale > j.old;
  return j;
}

// magnitude bits of the finite elements of a packed pair of 16-bit values (0 for infinities and
// NaN): they order like the magnitudes
template <typename T>
__device__ __forceinline__ uint32_t finite_bits(uint32_t half) {
  constexpr uint32_t INF = __is_same(T, __bf16) ? 0x7f80u : 0x7c00u;
  const uint32_t m = half & 0x7fffu;
  return m < INF ? m : 0u;
}
template <typename T>
__device__ __forceinline__ float bits_value(uint32_t m) {
  return (float)__builtin_bit_cast(T, (uint16_t)m);
}

// host checks shared by the entry points that take an 8-bit cache
inline int check_cache8(const char* who, const void* key_cache, const void* value_cache,
                        const float* kv_scales, int num_kv_heads, int head_size, int block_size,
                        int64_t num_blocks, int table_width, int64_t kv_block_stride,
                        int64_t kv_head_stride, int dtype, int kv_format) {
  PE_REQUIRE(kv_format == PE_KV_FP8_E4M3 || kv_format == PE_KV_INT8, PE_ERR_UNSUPPORTED,
             "%s: kv_format %d is not an 8-bit format", who, kv_format);
  PE_REQUIRE(dtype == PE_BF16 || dtype == PE_F16, PE_ERR_UNSUPPORTED,
             "%s: dtype %d (bf16 or f16 rows)", who, dtype);
  PE_REQUIRE(num_kv_heads > 0 && num_blocks > 0 && table_width > 0, PE_ERR_INVALID_ARG, "%s: bad sizes", who);
  PE_REQUIRE(head_size == 32 || head_size == 64 || head_size == 80 || head_size == 96 || head_size == 112 ||
                 head_size == 128 || head_size == 192 || head_size == 256,
             PE_ERR_UNSUPPORTED, "%s: head size %d (32, 64, 80, 96, 112, 128, 192 or 256: whole 16-byte "
             "pieces of 8-bit elements)", who, head_size);
  PE_REQUIRE(block_size == 8 || block_size == 16 || block_size == 32, PE_ERR_UNSUPPORTED,
             "%s: block size %d (8, 16 or 32)", who, block_size);
  PE_REQUIRE((int64_t)table_width * block_size <= (1 << 30), PE_ERR_UNSUPPORTED,
             "%s: block tables of %d blocks address more than 2^30 tokens", who, table_width);
  PE_REQUIRE(kv_block_stride % 16 == 0 && kv_head_stride % 16 == 0 &&
                 ((uintptr_t)key_cache | (uintptr_t)value_cache) % 16 == 0 && (uintptr_t)kv_scales % 8 == 0,
             PE_ERR_INVALID_ARG, "%s: caches must be 16-byte aligned", who);
  return PE_OK;
}

}  // namespace pe
