// Paged decode attention over a 16-bit or an 8-bit cache, optionally through a sliding window with
// sink tokens (the kernel template; the translation units paged_window*.hip instantiate it per
// cache element type).
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q.k_j - max),  j in the visible set:
//   j < len and (window == 0 or j >= len - window or j < sinks);  nothing visible: o = 0.
//
// Layout.  A tile is four units of U = 16 / (element bytes) tokens (8 in 16 bits, 16 in 8 bits).
// The 16x16x32 matrix instruction computes S^T = K.Q^T with the tile's tokens as rows: row 4g + r
// of row block b is token 4b + r of unit g, so lane group g (16 lanes, one per query head) ends up
// with the scores of unit g's tokens, in order.  That is the order in which one 16-byte piece of a
// value row holds them, so P meets V in O^T += V^T.P^T without moving across lanes, every load is
// 16 bytes per lane, and with 8-bit elements a lane's tokens share one block's scales.
//   K: lane (g, c) loads chunk 4*kk + g of token 4b + (c & 3) of unit c >> 2 (64-byte runs)
//   V: lane (g, c) loads row 16*dt + c of unit g
// 8-bit codes are converted to the query's type exactly; K's scale multiplies the f32 scores, V's
// scale the probabilities.
#pragma once
#include "kv8.h"

namespace pe {

constexpr float WIN_NEG = -1.0e30f;

// Conditions a launch survives (this translation unit's copy; read through pe_device_diagnostics)
static __device__ unsigned int window_diag_word;

struct WinArgs {
  void* out;
  float* ws;
  const void *query, *key_cache, *value_cache;
  const float* kv_scales;  // [num_blocks, num_kv_heads, 2], 8-bit caches only
  const int32_t *block_tables, *seq_lens;
  int num_heads, num_kv_heads, table_width, window, sinks, num_splits, head_groups;
  int64_t num_blocks, q_stride, kv_block_stride, kv_head_stride;  // strides in elements
  float scale_log2;
};

__host__ __device__ inline int64_t win_ws_stride(int head_size) { return head_size + 2; }

// max over the four lanes l, l^16, l^32, l^48 by row swaps (no LDS round trip)
__device__ __forceinline__ float win_max_groups(float x) {
  unsigned u = __float_as_uint(x);
  auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  u = __float_as_uint(x);
  auto b = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// The tiles of a sequence that hold visible tokens: [0, sink_tiles) and [first, first + window
// tiles); tokens are visible when tok < len and (tok >= lo or tok < sink_end).
struct WinRange {
  int len, lo, sink_end, sink_tiles, first, tiles;
  __device__ __forceinline__ int tile(int i) const { return i < sink_tiles ? i : first + i - sink_tiles; }
};
template <int TOK>
__host__ __device__ inline WinRange win_range(int len, int window, int sinks) {
  WinRange r;
  r.len = len;
  r.lo = window > 0 && len > window ? len - window : 0;
  r.sink_end = sinks < r.lo ? sinks : r.lo;
  r.first = r.lo / TOK;
  r.sink_tiles = (r.sink_end + TOK - 1) / TOK;
  if (r.sink_tiles > r.first) r.sink_tiles = r.first;  // the last sink tile is the window's first
  r.tiles = len > 0 ? r.sink_tiles + (len + TOK - 1) / TOK - r.first : 0;
  return r;
}

// T: query / output type; C: cache element (T, Fp8 or Int8); D: head size; BLK: tokens per block
template <typename T, typename C, int D, int WAVES, int BLK>
__global__ __launch_bounds__(WAVES * 64, 2) void paged_window_kernel(const WinArgs a) {
  using TR = Traits<T>;
  using vec8 = typename TR::vec8;
  constexpr bool Q8 = !__is_same(C, T);
  constexpr int ES = Q8 ? 1 : 2;          // bytes per cache element
  constexpr int U = 16 / ES;              // tokens per unit
  constexpr int TOK = 4 * U;              // tokens per tile
  constexpr int NB = U / 4;               // row blocks of S^T
  constexpr int NP = U / 8;               // P.V k-steps
  constexpr int KC = (D * ES + 63) / 64;  // K chunks per lane and token
  constexpr int DT = (D + 15) / 16;
  constexpr int CHUNKS = D * ES / 16;     // chunks of a K row
  constexpr int PB = BLK < U ? 2 : 1;     // blocks per unit
  static_assert(D * ES % 16 == 0 && BLK * PB >= U, "head size / block size");

  const int split = blockIdx.x;
  const int kvh = blockIdx.y / a.head_groups, hgrp = blockIdx.y % a.head_groups;
  const int seq = blockIdx.z;
  const int gqa = a.num_heads / a.num_kv_heads;
  const int head0 = kvh * gqa + hgrp * 16;
  const int nh = min(16, gqa - hgrp * 16);  // query heads of this workgroup
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c = lane & 15;

  const int32_t* table = a.block_tables + (int64_t)seq * a.table_width;
  const int raw_len = a.seq_lens[seq];
  const int64_t most = (int64_t)a.table_width * BLK;
  const int len = raw_len > most ? (int)most : max(raw_len, 0);
  if (raw_len > most && threadIdx.x == 0 && split == 0 && blockIdx.y == 0)
    atomicOr(&window_diag_word, (unsigned)PE_DIAG_DECODE_LEN_CLAMPED);
  const WinRange R = win_range<TOK>(len, a.window, a.sinks);
  const int per_split = (R.tiles + a.num_splits - 1) / a.num_splits;
  const int i_begin = split * per_split, i_end = min(R.tiles, i_begin + per_split);

  // ---- Q: the lane's chunks of head c, matched to the K chunks -------------------------------
  vec8 qf[KC][ES == 1 ? 2 : 1];
  {
    const T* qp = (const T*)a.query + (int64_t)seq * a.q_stride + (int64_t)(head0 + c) * D;
#pragma unroll
    for (int kk = 0; kk < KC; ++kk)
#pragma unroll
      for (int e = 0; e < (Q8 ? 2 : 1); ++e) {
        u32x4 raw = {0u, 0u, 0u, 0u};
        if (c < nh && 4 * kk + g < CHUNKS)
          raw = *reinterpret_cast<const u32x4*>(qp + (4 * kk + g) * U + 8 * e);
        qf[kk][e] = __builtin_bit_cast(vec8, raw);
      }
  }

  struct Tile {
    u32x4 k[NB][KC];
    u32x4 v[DT];
    float ks[PB], vs[PB];  // scales of unit g
    uint32_t ok;           // unit g: bit h = its block h has a valid id
  };
  struct Ids {
    int k[PB], v[PB];
  };
  const char* kbase = (const char*)a.key_cache + (int64_t)kvh * a.kv_head_stride * ES;
  const char* vbase = (const char*)a.value_cache + (int64_t)kvh * a.kv_head_stride * ES;
  const int64_t blk_bytes = a.kv_block_stride * ES;

  // a unit without visible tokens is replaced by the last one of the sequence: its own blocks may
  // have been given away already
  auto unit_of = [&](int t, int u) {
    const int unit = t * 4 + u;
    const int tok = unit * U;
    const bool seen = tok < R.len && (tok + U > R.lo || tok < R.sink_end);
    return seen ? unit : (R.len - 1) / U;
  };
  auto load_ids = [&](Ids& id, int i) {
    const int t = R.tile(i);
    const int uk = unit_of(t, c >> 2), uv = unit_of(t, g);
#pragma unroll
    for (int h = 0; h < PB; ++h) {
      // the second half of the last unit may lie past the sequence's blocks: the last block again
      id.k[h] = table[min(uk * U + h * BLK, R.len - 1) / BLK];
      id.v[h] = table[min(uv * U + h * BLK, R.len - 1) / BLK];
    }
  };
  auto issue = [&](Tile& t, const Ids& id, int i) {
    const int tile = R.tile(i);
    const int uk = unit_of(tile, c >> 2), uv = unit_of(tile, g);
    t.ok = 0;
    const char *kp[PB], *vp[PB];
#pragma unroll
    for (int h = 0; h < PB; ++h) {
      const bool k_ok = (unsigned)id.k[h] < (uint64_t)a.num_blocks, v_ok = (unsigned)id.v[h] < (uint64_t)a.num_blocks;
      t.ok |= v_ok ? 1u << h : 0u;
      const int64_t kb = k_ok ? id.k[h] : 0, vb = v_ok ? id.v[h] : 0;
      // K: [chunk][BLK tokens][16 bytes]; V: [d][BLK tokens]
      kp[h] = kbase + kb * blk_bytes + (PB == 1 ? uk * U % BLK : 0) * 16 + (c & 3) * 16 + g * (BLK * 16);
      vp[h] = vbase + vb * blk_bytes + (PB == 1 ? uv * U % BLK : 0) * ES + c * (BLK * ES);
      if constexpr (Q8) {
        const float* sc = a.kv_scales + (vb * a.num_kv_heads + kvh) * 2;
        t.ks[h] = sc[0];
        t.vs[h] = sc[1];
      }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const char* p = PB == 1 ? kp[0] + b * 64 : kp[b / (NB / PB)] + (b % (NB / PB)) * 64;
#pragma unroll
      for (int kk = 0; kk < KC; ++kk) {
        t.k[b][kk] = u32x4{0u, 0u, 0u, 0u};
        if (4 * kk + 3 < CHUNKS || 4 * kk + g < CHUNKS)
          t.k[b][kk] = *reinterpret_cast<const u32x4*>(p + kk * (4 * BLK * 16));
      }
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      t.v[dt] = u32x4{0u, 0u, 0u, 0u};
      if (16 * dt + 15 < D || 16 * dt + c < D) {
        if constexpr (PB == 1) {
          t.v[dt] = *reinterpret_cast<const u32x4*>(vp[0] + dt * (16 * BLK * ES));
        } else {
          const u32x2 lo = *reinterpret_cast<const u32x2*>(vp[0] + dt * (16 * BLK * ES));
          const u32x2 hi = *reinterpret_cast<const u32x2*>(vp[1] + dt * (16 * BLK * ES));
          t.v[dt] = u32x4{lo[0], lo[1], hi[0], hi[1]};
        }
      }
    }
  };

  float m_run = WIN_NEG, l_run = 0.f;  // log2 units; l_run: this lane's tokens only
  float w_run = WIN_NEG;               // f16 with 8-bit values: reference point of p * scale
  // f16 products p * scale of V may leave f16's normal range; they are kept relative to their own
  // running maximum.  bf16 has the range.
  constexpr bool WREF = Q8 && __is_same(T, _Float16);
  f32x4 acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x4{0.f, 0.f, 0.f, 0.f};

  auto compute = [&](Tile& t, int i) {
    const int tile = R.tile(i);
    const int t0 = tile * TOK;
    f32x4 s[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      s[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < KC; ++kk) {
        const u32x4 w = t.k[b][kk];
        if constexpr (Q8) {
          s[b] = TR::mfma16(codes8<T, C>(w[0], w[1]), qf[kk][0], s[b]);
          s[b] = TR::mfma16(codes8<T, C>(w[2], w[3]), qf[kk][1], s[b]);
        } else {
          s[b] = TR::mfma16(__builtin_bit_cast(vec8, w), qf[kk][0], s[b]);
        }
      }
    }
    const bool inside = t0 + TOK <= R.len && (t0 >= R.lo || t0 + TOK <= R.sink_end);
    const bool good = __builtin_amdgcn_ballot_w64(t.ok != (1u << PB) - 1u) == 0;
    const bool masked = !(inside && good);  // wave-uniform
    const int tok0 = t0 + g * U;
    auto hidden = [&](int e) {  // token e of the lane's unit
      const int tok = tok0 + e;
      const bool block_ok = (t.ok >> (PB == 1 ? 0 : e / (U / PB))) & 1u;
      return !(tok < R.len && (tok >= R.lo || tok < R.sink_end) && block_ok);
    };
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const float f = Q8 ? a.scale_log2 * t.ks[b / (NB / PB)] : a.scale_log2;
      s[b] *= f;
    }
    if (masked) {
      if (!good && lane % 16 == 0 && t.ok != (1u << PB) - 1u) {
        // report an id outside the cache only where one of its tokens would have been visible
        for (int e = 0; e < U; ++e) {
          const int tok = tok0 + e;
          if (tok < R.len && (tok >= R.lo || tok < R.sink_end) && hidden(e))
            atomicOr(&window_diag_word, (unsigned)PE_DIAG_BLOCK_ID);
        }
      }
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[b][r] = hidden(4 * b + r) ? -INFINITY : s[b][r];
    }
    float mx[PB], lv[PB];
#pragma unroll
    for (int h = 0; h < PB; ++h) {
      mx[h] = -INFINITY;
#pragma unroll
      for (int b = h * (NB / PB); b < (h + 1) * (NB / PB); ++b)
        mx[h] = fmaxf(mx[h], fmaxf(fmaxf(s[b][0], s[b][1]), fmaxf(s[b][2], s[b][3])));
    }
    const float m_new = fmaxf(m_run, win_max_groups(PB == 1 ? mx[0] : fmaxf(mx[0], mx[PB - 1])));
    float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
    l_run *= alpha;
    float wf[PB];  // factor of the lane's probabilities in front of V
    if constexpr (WREF) {
      float y = -INFINITY;
#pragma unroll
      for (int h = 0; h < PB; ++h) {
        lv[h] = __builtin_amdgcn_logf(t.vs[h]);  // log2; -inf for a block of zeros
        y = fmaxf(y, mx[h] + lv[h]);
      }
      const float w_new = fmaxf(w_run, win_max_groups(y));
      alpha = __builtin_amdgcn_exp2f(w_run - w_new);
#pragma unroll
      for (int h = 0; h < PB; ++h) wf[h] = __builtin_amdgcn_exp2f(lv[h] + (m_new - w_new));
      w_run = w_new;
    } else {
#pragma unroll
      for (int h = 0; h < PB; ++h) wf[h] = Q8 ? t.vs[h] : 1.f;
    }
    m_run = m_new;
    vec8 pf[NP];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float p = __builtin_amdgcn_exp2f(s[b][r] - m_new);
        l_run += p;
        float w = Q8 ? p * wf[b / (NB / PB)] : p;
        if (Q8 && masked) w = hidden(4 * b + r) ? 0.f : w;  // the scale may be anything there
        pf[b >> 1][(b & 1) * 4 + r] = (T)w;
      }
    // hidden slots may hold anything (NaN included): their values become zero
    if (masked) {
      u32x4 keep;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t mk = 0;
#pragma unroll
        for (int e = 0; e < 4 / ES; ++e)
          mk |= hidden(w * (4 / ES) + e) ? 0u : (ES == 1 ? 0xffu : 0xffffu) << (8 * ES * e);
        keep[w] = mk;
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) t.v[dt] &= keep;
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      acc[dt] *= alpha;
      const u32x4 w = t.v[dt];
      if constexpr (Q8) {
        acc[dt] = TR::mfma16(codes8<T, C>(w[0], w[1]), pf[0], acc[dt]);
        acc[dt] = TR::mfma16(codes8<T, C>(w[2], w[3]), pf[NP - 1], acc[dt]);
      } else {
        acc[dt] = TR::mfma16(__builtin_bit_cast(vec8, w), pf[0], acc[dt]);
      }
    }
  };

  {
    Tile t0;
    Ids id;
    for (int i = i_begin + wave; i < i_end; i += WAVES) {
      load_ids(id, i);
      issue(t0, id, i);
      compute(t0, i);
    }
  }

  // ---- join the lane groups' sums, then the waves through LDS ---------------------------------
  l_run += __shfl_xor(l_run, 16);
  l_run += __shfl_xor(l_run, 32);
  if constexpr (WREF) {  // numerators relative to the same point as the sum
    const float f = __builtin_amdgcn_exp2f(w_run - m_run);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt] *= f;
  }
  // dynamic LDS: o[WAVES][nh][16 * DT + 4], m[WAVES][16], l[WAVES][16] (f32)
  extern __shared__ __attribute__((aligned(16))) float win_smem[];
  constexpr int OROW = 16 * DT + 4;
  const int heads = min(16, gqa);
  float* sm_o = win_smem;
  float* sm_m = win_smem + WAVES * heads * OROW;
  float* sm_l = sm_m + WAVES * 16;
  if (c < nh) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      *reinterpret_cast<f32x4*>(&sm_o[(wave * heads + c) * OROW + 16 * dt + 4 * g]) = acc[dt];
    if (g == 0) {
      sm_m[wave * 16 + c] = m_run;
      sm_l[wave * 16 + c] = l_run;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nh * D; i += WAVES * 64) {
    const int h = i / D, d = i % D;
    float m_tot = sm_m[h];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) m_tot = fmaxf(m_tot, sm_m[w * 16 + h]);
    float o = 0.f, l = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float f = __builtin_amdgcn_exp2f(sm_m[w * 16 + h] - m_tot);
      o += f * sm_o[(w * heads + h) * OROW + d];
      l += f * sm_l[w * 16 + h];
    }
    const int head = head0 + h;
    if (a.num_splits == 1) {
      ((T*)a.out)[((int64_t)seq * a.num_heads + head) * D + d] = (T)(l == 0.f ? 0.f : o / l);
    } else {
      float* w = a.ws + (((int64_t)split * gridDim.z + seq) * a.num_heads + head) * win_ws_stride(D);
      if (d == 0) {
        w[0] = m_tot;
        w[1] = l;
      }
      w[2 + d] = o;
    }
  }
}

template <typename T, typename C, int D, int WAVES, int BLK>
inline void launch_window(const WinArgs& a, dim3 grid, hipStream_t st) {
  constexpr int DT = (D + 15) / 16;
  const int gqa = a.num_heads / a.num_kv_heads, heads = gqa < 16 ? gqa : 16;
  const size_t lds = ((size_t)WAVES * heads * (16 * DT + 4) + 2 * WAVES * 16) * 4;
  if (lds > 64 * 1024)
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&paged_window_kernel<T, C, D, WAVES, BLK>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  hipLaunchKernelGGL((paged_window_kernel<T, C, D, WAVES, BLK>), grid, dim3(WAVES * 64), lds, st, a);
}

template <typename T, typename C, int D>
inline int dispatch_window_block(const WinArgs& a, int block_size, dim3 grid, hipStream_t st) {
  switch (block_size) {
    case 8: launch_window<T, C, D, 4, 8>(a, grid, st); return PE_OK;
    case 16: launch_window<T, C, D, 4, 16>(a, grid, st); return PE_OK;
    case 32: launch_window<T, C, D, 4, 32>(a, grid, st); return PE_OK;
  }
  return fail(PE_ERR_UNSUPPORTED, "paged_decode_window: block size %d (8, 16 or 32)", block_size);
}

// head sizes of one translation unit; the 16-bit cache also has 120
template <typename T, typename C>
inline int dispatch_window(const WinArgs& a, int head_size, int block_size, dim3 grid, hipStream_t st) {
  switch (head_size) {
    case 32: return dispatch_window_block<T, C, 32>(a, block_size, grid, st);
    case 64: return dispatch_window_block<T, C, 64>(a, block_size, grid, st);
    case 80: return dispatch_window_block<T, C, 80>(a, block_size, grid, st);
    case 96: return dispatch_window_block<T, C, 96>(a, block_size, grid, st);
    case 112: return dispatch_window_block<T, C, 112>(a, block_size, grid, st);
    case 128: return dispatch_window_block<T, C, 128>(a, block_size, grid, st);
    case 192: return dispatch_window_block<T, C, 192>(a, block_size, grid, st);
    case 256: return dispatch_window_block<T, C, 256>(a, block_size, grid, st);
    case 120:
      if constexpr (__is_same(T, C)) return dispatch_window_block<T, C, 120>(a, block_size, grid, st);
  }
  return fail(PE_ERR_UNSUPPORTED, "paged_decode_window: head size %d is not built", head_size);
}

static int window_diag_fetch_tu(unsigned int* out, int reset) {
  void* p = nullptr;
  hipError_t e = hipGetSymbolAddress(&p, HIP_SYMBOL(window_diag_word));
  if (e == hipSuccess) e = hipMemcpy(out, p, sizeof(unsigned int), hipMemcpyDeviceToHost);
  if (e == hipSuccess && reset && *out != 0) e = hipMemset(p, 0, sizeof(unsigned int));
  if (e != hipSuccess) return fail(PE_ERR_LAUNCH, "window attention diagnostics: %s", hipGetErrorString(e));
  return PE_OK;
}

}  // namespace pe
