// Entry points of the windowed and the 8-bit decode attention (kernel: paged_window_kernel.h)
//   pe_paged_decode_window   16-bit cache, sliding window + sink tokens
//   pe_paged_decode_8bit     8-bit cache, with or without a window
//   pe_decode_step_8bit      KV write of the step's token + the attention, in one launch for head sizes up to
//                            128 with up to 16 query heads per KV head
#include <initializer_list>

#include "paged_window_kernel.h"

namespace pe {

int launch_window_16(const WinArgs& a, int head_size, int block_size, int waves, int dtype, dim3 grid, hipStream_t st);
int launch_window_fp8(const WinArgs& a, int head_size, int block_size, int waves, int dtype, dim3 grid, hipStream_t st);
int launch_window_int8(const WinArgs& a, int head_size, int block_size, int waves, int dtype, dim3 grid, hipStream_t st);
int launch_step_fp8(const WinArgs& a, int head_size, int block_size, int waves, int dtype, dim3 grid, hipStream_t st);
int launch_step_int8(const WinArgs& a, int head_size, int block_size, int waves, int dtype, dim3 grid, hipStream_t st);
int window_16_diag_fetch(unsigned int* out, int reset);
int window_fp8_diag_fetch(unsigned int* out, int reset);
int window_int8_diag_fetch(unsigned int* out, int reset);
int step_fp8_diag_fetch(unsigned int* out, int reset);
int step_int8_diag_fetch(unsigned int* out, int reset);

int window_diag_fetch(unsigned int* out, int reset) {
  *out = 0;
  for (auto fetch : {window_16_diag_fetch, window_fp8_diag_fetch, window_int8_diag_fetch, step_fp8_diag_fetch,
                     step_int8_diag_fetch}) {
    unsigned int one = 0;
    if (int rc = fetch(&one, reset)) return rc;
    *out |= one;
  }
  return PE_OK;
}

// Workgroup width (waves) and number of splits over the keys of a launch.  A split costs a merge launch
// (about 2.5 us of GPU time, 2 us of host time where launches are not replayed from a graph); a wave
// takes its tiles (16 KiB at head size 128) one memory round trip after the other, so a launch that
// cannot fill the chip wants them on many waves.  Long launches end with their fullest CU (of 256): the
// splits are those that spread the workgroups evenly.  Measured on MI355X (us graph-replayed, | issued one
// by one; waves/splits; workgroups without splits x tiles of a sequence; head size 128, w: the wide form):
//   512 x 112 (64 x 8192 tokens, 8 bit): 4/1 154, 4/2 156, 8/1 172; 512 x 32: 42 / 45 / 49; 512 x 13: 19 / 24 / 22
//   512 x 33 (16 bit): 4/1 45, 4/2 49, 8/1 52; 512 x 64: 75 / 80 / 86; 2048 x 4: 22 / 41 / 43
//   320 x 128 (16 bit): 4/1 113, 4/2 101; 320 x 64: 62 / 56; 320 x 32: 33 / 31; 320 x 13: 16 / 18; 400 x 64: 61 / 65
//   256 x 13: 4/1 12.5, 8/1 13.1, 4/2 15.0; 224 x 65: 4/1 37, 4/2 40, w/1 41; 192 x 65: 34 / 37 / 37
//   240 x 79 (head 64): 4/1 35, 4/2 29, w/1 31; 204 x 79 (head 64): 35 / 26 / 27; (head 32): 33 / 24 / 19
//   136 x 65: 4/1 32, 4/2 33, 4/3 28, w/1 31; 136 x 129 (16 bit): 50 / 57 / 46 / 55
//   192 x 33: w/1 18, 4/1 20; 160 x 33: w/1 16, 4/1 19, 4/3 19; 136 x 33: 15 / 19 / 18; 136 x 41 (16 bit): 16 / 19 / 19
//    96 x 42 (16 bit): w/1 12.8, 4/2 14.6; 96 x 65 (16 bit): 23 / 19; 136 x 54 (16 bit, head 96): 17, 4/3 18
//   128 x 128: 4/1 58, 4/2 43, 4/4 43, 8/1 55; 96 x 129 (16 bit): 4/2 33, 4/3 43, 4/5 33; 32 x 512: 4/4 60, 4/8 43, 8/8 50
//    64 x 65: 4/4 16.7, 4/8 15.7, 8/1 22; 64 x 49: 4/4 14.5, 4/8 15.9, 8/1 19; 40 x 257 (16 bit): 4/6 28, 4/7 35
//    64 x 13: 12/1 8.4 | 7.8, 4/4 8.7 | 8.5, 4/1 10; 32 x 13: 12/1 7.5 | 7.3, 4/4 8.4 | 8.4
//    12 x 13 (head 64): 16/1 7.4 | 7.1, 4/4 6.7 | 8.4, 4/1 8.5; 8 x 7: 12/1 6.5 | 6.2, 4/2 7.5 | 8.4
//     8 x 32: 12/3 8.6 | 8.5, 4/8 8.5 | 8.5, 12/1 11; 8 x 65: 8/9 8.2, 4/8 11; 6 x 24 (head 64): 16/1 7.7 | 7.4
struct WinShape {
  int waves, splits;
};
static WinShape window_shape(int num_seqs, int num_heads, int num_kv_heads, int head_size, int max_seq_len,
                             int window, int sinks, int kv_format, bool step) {
  const int gqa = num_heads / num_kv_heads;
  const int64_t wgs = (int64_t)num_seqs * num_kv_heads * ((gqa + 15) / 16);
  const int tok = kv_format == PE_KV_SAME ? 32 : 64;
  const int64_t seen = window > 0 && (int64_t)window + sinks < max_seq_len ? (int64_t)window + sinks : max_seq_len;
  // (a window and its sinks may each begin and end inside a tile)
  const int64_t tiles = (seen + tok - 1) / tok + (window > 0 && seen < max_seq_len ? 1 + (sinks > 0) : 0);
  const int wide = win_wide(head_size, step);
  WinShape s{4, 1};
  if (tiles <= 4) return s;  // nothing to share out
  if (wgs >= 256) {          // the chip is full; one and a half rounds instead of two
    if (wgs > 256 && wgs <= 352 && tiles >= 32) s.splits = 2;
  } else if (wgs * tiles <= 4352 && tiles <= 2 * wide) {  // one launch, at most two tiles per wave
    s.waves = wide;
  } else if (wgs * tiles <= 1024) {  // one tile per wave
    if (tiles > 32) s.waves = wide;
    s.splits = (int)((tiles + s.waves - 1) / s.waves);
  } else if (wgs > 64 && tiles * head_size <= 56 * 128 && wgs * tiles * head_size <= 6000 * 128) {
    s.waves = wide;  // splits would not fill the chip evenly, or cost more than they give
  } else if (wgs <= 128) {  // bound by bandwidth: a workgroup per CU (below 8 workgroups WIN_MAX_SPLITS leaves CUs idle)
    s.splits = (int)(256 / wgs);
  } else {  // three splits on every second CU; tiles of 8 KiB and less want the waves of two
    s.splits = wgs <= 170 ? 3 : head_size <= 64 ? 2 : 1;
  }
  if (s.splits > WIN_MAX_SPLITS) s.splits = WIN_MAX_SPLITS;
  return s;
}

static int check_window(const char* who, int window, int sinks) {
  PE_REQUIRE(window >= 0 && sinks >= 0, PE_ERR_INVALID_ARG,
             "%s: sliding_window %d and num_sinks %d must not be negative", who, window, sinks);
  return PE_OK;
}

static int window_decode(const char* who, void* out, const void* query, const void* key_cache,
                         const void* value_cache, const float* kv_scales, const int32_t* block_tables,
                         const int32_t* seq_lens, int num_seqs, int num_heads, int num_kv_heads,
                         int head_size, int block_size, int64_t num_blocks, int table_width,
                         int64_t q_stride, int64_t kv_block_stride, int64_t kv_head_stride, float scale,
                         int max_seq_len, int window, int sinks, int dtype, int kv_format,
                         void* workspace, int64_t workspace_bytes, void* stream,
                         const void* new_key = nullptr, const void* new_value = nullptr,
                         int64_t new_k_stride = 0, int64_t new_v_stride = 0) {
  PE_REQUIRE(out && query && key_cache && value_cache && block_tables && seq_lens, PE_ERR_INVALID_ARG,
             "%s: null pointer", who);
  PE_REQUIRE(num_heads > 0 && num_kv_heads > 0 && num_heads % num_kv_heads == 0, PE_ERR_INVALID_ARG,
             "%s: num_heads %d must be a positive multiple of num_kv_heads %d", who, num_heads, num_kv_heads);
  PE_REQUIRE(max_seq_len >= 0, PE_ERR_INVALID_ARG, "%s: negative max_seq_len", who);
  PE_REQUIRE(q_stride % 8 == 0 && (uintptr_t)query % 16 == 0, PE_ERR_INVALID_ARG,
             "%s: query rows must be 16-byte aligned", who);
  const int gqa = num_heads / num_kv_heads, groups = (gqa + 15) / 16;
  PE_REQUIRE(num_seqs <= 65535 && (int64_t)num_kv_heads * groups <= 65535, PE_ERR_UNSUPPORTED,
             "%s: grid too large", who);
  // The row is written by a launch of its own where several workgroups read the block that it joins (more
  // than 16 query heads on a KV head) and where the kernel has no registers left for it
  const bool step = new_key != nullptr && groups == 1 && head_size <= 128;
  const WinShape shape = window_shape(num_seqs, num_heads, num_kv_heads, head_size, max_seq_len, window, sinks, kv_format, step);
  const int splits = shape.splits, waves = shape.waves;
  if (splits > 1) {
    const int64_t need = (int64_t)splits * num_seqs * num_heads * win_ws_stride(head_size) * 4;
    PE_REQUIRE(workspace && workspace_bytes >= need, PE_ERR_WORKSPACE, "%s needs %lld workspace bytes, got %lld",
               who, (long long)need, (long long)workspace_bytes);
  }
  const WinArgs a{out, (float*)workspace, query, key_cache, value_cache, kv_scales, block_tables, seq_lens,
                  num_heads, num_kv_heads, table_width, window, sinks, splits, groups, num_blocks, q_stride,
                  kv_block_stride, kv_head_stride, scale * 1.4426950408889634f,
                  new_key, new_value, new_k_stride, new_v_stride};
  const dim3 grid((unsigned)splits, (unsigned)(num_kv_heads * groups), (unsigned)num_seqs);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (new_key != nullptr && !step) {
    if (int rc = pe_reshape_and_cache_8bit(new_key, new_value, const_cast<void*>(key_cache),
                                           const_cast<void*>(value_cache), const_cast<float*>(kv_scales), block_tables,
                                           seq_lens, nullptr, num_seqs, num_seqs, 1, new_k_stride, new_v_stride,
                                           num_kv_heads, head_size, block_size, num_blocks, table_width,
                                           kv_block_stride, kv_head_stride, dtype, kv_format, stream))
      return rc;
  }
  int rc;
  if (kv_format == PE_KV_FP8_E4M3)
    rc = (step ? launch_step_fp8 : launch_window_fp8)(a, head_size, block_size, waves, dtype, grid, st);
  else if (kv_format == PE_KV_INT8)
    rc = (step ? launch_step_int8 : launch_window_int8)(a, head_size, block_size, waves, dtype, grid, st);
  else
    rc = launch_window_16(a, head_size, block_size, waves, dtype, grid, st);
  if (rc) return rc;
  return check_launch(who);
}

}  // namespace pe

extern "C" {

int64_t pe_paged_window_workspace_bytes(int num_seqs, int num_heads, int num_kv_heads, int head_size,
                                        int max_seq_len, int sliding_window, int num_sinks, int kv_format) {
  using namespace pe;
  if (num_seqs <= 0 || num_heads <= 0 || num_kv_heads <= 0) return 0;
  int64_t splits = 1;  // of the attention alone and of the step
  for (bool step : {false, true}) {
    const WinShape w = window_shape(num_seqs, num_heads, num_kv_heads, head_size, max_seq_len, sliding_window,
                                    num_sinks, kv_format, step);
    splits = splits < w.splits ? w.splits : splits;
  }
  return splits <= 1 ? 0 : splits * num_seqs * num_heads * win_ws_stride(head_size) * 4;
}

int pe_paged_decode_window(void* out, const void* query, const void* key_cache, const void* value_cache,
                           const int32_t* block_tables, const int32_t* seq_lens, int num_seqs,
                           int num_heads, int num_kv_heads, int head_size, int block_size,
                           int64_t num_blocks, int max_num_blocks_per_seq, int64_t q_stride,
                           int64_t kv_block_stride, int64_t kv_head_stride, float scale,
                           int max_seq_len, int sliding_window, int num_sinks, int dtype,
                           void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace pe;
  const char* who = "paged_decode_window";
  PE_REQUIRE(num_seqs >= 0, PE_ERR_INVALID_ARG, "%s: negative num_seqs", who);
  if (num_seqs == 0) return PE_OK;
  if (int rc = check_window(who, sliding_window, num_sinks)) return rc;
  PE_REQUIRE(dtype == PE_BF16 || dtype == PE_F16, PE_ERR_UNSUPPORTED, "%s: dtype %d (bf16 or f16)", who, dtype);
  PE_REQUIRE(num_blocks > 0 && max_num_blocks_per_seq > 0, PE_ERR_INVALID_ARG, "%s: bad sizes", who);
  PE_REQUIRE((int64_t)max_num_blocks_per_seq * block_size <= (1 << 30), PE_ERR_UNSUPPORTED,
             "%s: block tables of %d blocks address more than 2^30 tokens", who, max_num_blocks_per_seq);
  PE_REQUIRE(kv_block_stride % 8 == 0 && kv_head_stride % 8 == 0 &&
                 ((uintptr_t)key_cache | (uintptr_t)value_cache) % 16 == 0,
             PE_ERR_INVALID_ARG, "%s: caches must be 16-byte aligned", who);
  return window_decode(who, out, query, key_cache, value_cache, nullptr, block_tables, seq_lens, num_seqs,
                       num_heads, num_kv_heads, head_size, block_size, num_blocks, max_num_blocks_per_seq,
                       q_stride, kv_block_stride, kv_head_stride, scale, max_seq_len, sliding_window,
                       num_sinks, dtype, PE_KV_SAME, workspace, workspace_bytes, stream);
}

int pe_paged_decode_8bit(void* out, const void* query, const void* key_cache, const void* value_cache,
                         const float* kv_scales, const int32_t* block_tables, const int32_t* seq_lens,
                         int num_seqs, int num_heads, int num_kv_heads, int head_size, int block_size,
                         int64_t num_blocks, int max_num_blocks_per_seq, int64_t q_stride,
                         int64_t kv_block_stride, int64_t kv_head_stride, float scale, int max_seq_len,
                         int sliding_window, int num_sinks, int dtype, int kv_format, void* workspace,
                         int64_t workspace_bytes, void* stream) {
  using namespace pe;
  const char* who = "paged_decode_8bit";
  PE_REQUIRE(num_seqs >= 0, PE_ERR_INVALID_ARG, "%s: negative num_seqs", who);
  if (num_seqs == 0) return PE_OK;
  PE_REQUIRE(kv_scales, PE_ERR_INVALID_ARG, "%s: null pointer", who);
  if (int rc = check_window(who, sliding_window, num_sinks)) return rc;
  if (int rc = check_cache8(who, key_cache, value_cache, kv_scales, num_kv_heads, head_size, block_size,
                            num_blocks, max_num_blocks_per_seq, kv_block_stride, kv_head_stride, dtype, kv_format))
    return rc;
  return window_decode(who, out, query, key_cache, value_cache, kv_scales, block_tables, seq_lens, num_seqs,
                       num_heads, num_kv_heads, head_size, block_size, num_blocks, max_num_blocks_per_seq,
                       q_stride, kv_block_stride, kv_head_stride, scale, max_seq_len, sliding_window,
                       num_sinks, dtype, kv_format, workspace, workspace_bytes, stream);
}

int pe_decode_step_8bit(void* out, const void* query, const void* new_key, const void* new_value,
                        void* key_cache, void* value_cache, float* kv_scales, const int32_t* block_tables,
                        const int32_t* seq_lens, int num_seqs, int num_heads, int num_kv_heads,
                        int head_size, int block_size, int64_t num_blocks, int max_num_blocks_per_seq,
                        int64_t q_stride, int64_t new_k_stride, int64_t new_v_stride,
                        int64_t kv_block_stride, int64_t kv_head_stride, float scale, int max_seq_len,
                        int sliding_window, int num_sinks, int dtype, int kv_format, void* workspace,
                        int64_t workspace_bytes, void* stream) {
  using namespace pe;
  const char* who = "decode_step_8bit";
  PE_REQUIRE(num_seqs >= 0, PE_ERR_INVALID_ARG, "%s: negative num_seqs", who);
  if (num_seqs == 0) return PE_OK;
  PE_REQUIRE(kv_scales && new_key && new_value, PE_ERR_INVALID_ARG, "%s: null pointer", who);
  if (int rc = check_window(who, sliding_window, num_sinks)) return rc;
  if (int rc = check_cache8(who, key_cache, value_cache, kv_scales, num_kv_heads, head_size, block_size,
                            num_blocks, max_num_blocks_per_seq, kv_block_stride, kv_head_stride, dtype, kv_format))
    return rc;
  PE_REQUIRE(new_k_stride % 8 == 0 && new_v_stride % 8 == 0 && ((uintptr_t)new_key | (uintptr_t)new_value) % 16 == 0,
             PE_ERR_INVALID_ARG, "%s: key/value rows must be 16-byte aligned", who);
  return window_decode(who, out, query, key_cache, value_cache, kv_scales, block_tables, seq_lens, num_seqs,
                       num_heads, num_kv_heads, head_size, block_size, num_blocks, max_num_blocks_per_seq,
                       q_stride, kv_block_stride, kv_head_stride, scale, max_seq_len, sliding_window,
                       num_sinks, dtype, kv_format, workspace, workspace_bytes, stream, new_key, new_value,
                       new_k_stride, new_v_stride);
}

}  // extern "C"
