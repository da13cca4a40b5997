// Paged decode attention over a 16-bit or an 8-bit cache, optionally through a sliding window with
// sink tokens (the kernel template; the translation units paged_window*.hip instantiate it per
// cache element type).
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q.k_j - max),  j in the visible set:
//   j < len and (window == 0 or j >= len - window or j < sinks);  nothing visible: o = 0.
//
// Layout.  A tile is NG groups of 16 tokens.  The 16x16x32 matrix instruction computes S^T = K.Q^T
// with a group's tokens as rows: lane (g, c) (c = query head) ends up with the scores of tokens
// 4g .. 4g+3 of every group.  A group lies in one block (in two with 8-token blocks), so block ids and
// 8-bit scales are wave-uniform.
//   K: lane (g, c) loads the 16-byte chunk 4*kk + g of token c: 1 KiB in one piece with 16-token blocks
//   V, 16 bits: lane (g, c) loads tokens 4g .. 4g+3 (8 bytes) of row 16*dt + c of a group.  Two groups
//     make one k-step of O^T += V^T.P^T whose slots are ordered so that P is used where it lies.
//   V, 8 bits: lane (g, c) loads all 16 tokens (16 bytes) of row 16*dt + c of group g, and P goes to
//     the lane group of its tokens by a 4x4 transpose of row swaps (8 per tile of 64 tokens).  With P
//     left where it lies the loads are 4 bytes: 260 instead of 168 us on 945 MB (replayed from a graph).
// 8-bit codes are converted to the query's type exactly; K's scale multiplies the f32 scores, V's
// scale the probabilities.
//
// Bound: HBM.  64 sequences x 7168 tokens on average, 8 KV heads x 128, int8: 945 MB in 154 us, 6.1 TB/s; the
// same loads without conversion and second matrix product 150.  64 x 1028 of 8192 tokens in 16 bits: 270 MB in
// 45 us, 6.0 TB/s.  64 x 776 in e4m3: 90 MB in 18.5 us (4.3 us of start and merge, the rest at 6.3 TB/s).
#pragma once
#include <type_traits>

#include "kv8.h"

namespace pe {

// below every finite score: the reference point of the weights before a visible key (f32's lowest number, not
// -infinity, so that differences of two such points are 0)
constexpr float WIN_NEG = -3.402823466e38f;
constexpr int WIN_MAX_SPLITS = 32;

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
  // pe_decode_step_8bit only
  const void *new_key, *new_value;
  int64_t new_k_stride, new_v_stride;
};

// waves of the wide workgroup: as many as the registers of a head size allow
constexpr int win_wide(int head_size, bool step) {
  return step ? (head_size <= 64 ? 12 : 8) : head_size <= 64 ? 16 : head_size <= 128 ? 12 : 8;
}

__host__ __device__ inline int64_t win_ws_stride(int head_size) { return head_size + 2; }

template <bool NT, typename V>
__device__ __forceinline__ V win_load(const V* p) {
  if constexpr (NT) return __builtin_nontemporal_load(p);
  else return *p;
}

// max over the four lanes l, l^16, l^32, l^48 by row swaps (no LDS round trip)
__device__ __forceinline__ float win_max_groups(float x) {
  unsigned u = __float_as_uint(x);
  auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  u = __float_as_uint(x);
  auto b = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

typedef __attribute__((ext_vector_type(2))) float f32x2;

// max over the wave, in every lane: rotations inside the rows of 16 lanes, then row swaps
__device__ __forceinline__ uint32_t win_max_wave(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, 0x128, 0xf, 0xf, true));  // row_ror:8
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, 0x124, 0xf, 0xf, true));  // row_ror:4
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, 0x122, 0xf, 0xf, true));  // row_ror:2
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, 0x121, 0xf, 0xf, true));  // row_ror:1
  auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  x = max((uint32_t)a[0], (uint32_t)a[1]);
  auto b = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  return (uint32_t)__builtin_amdgcn_readfirstlane((int)max((uint32_t)b[0], (uint32_t)b[1]));
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

// T: query / output type; C: cache element (T, Fp8 or Int8); D: head size; BLK: tokens per block.
// STEP (pe_decode_step_8bit): the sequence's last token is appended first, as pe_reshape_and_cache_8bit
// does it.  Its block lies in the last tile, which one wave owns: that wave encodes the row, puts it
// (and, where the block's scale grows, the re-expressed older codes) into the tile's registers and into
// the cache, and goes on with the attention.  No other wave of the launch touches the block.
// 64 x 776 tokens in e4m3: 20.6 us with the row, 18.6 without (the write in a launch of its own: 4.9);
// 64 x 200: 11.3 and 8.6.  (Every lane encoding the chunks it holds: 21.8 and 13.6.)
template <typename T, typename C, int D, int WAVES, int BLK, bool STEP>
__global__ __launch_bounds__(WAVES * 64, WAVES > 8 ? WAVES / 4 : 2) void paged_window_kernel(const WinArgs a) {
  using TR = Traits<T>;
  using vec8 = typename TR::vec8;
  constexpr bool Q8 = !__is_same(C, T);
  constexpr int ES = Q8 ? 1 : 2;              // bytes per cache element
  constexpr int NG = Q8 ? 4 : 2;              // 16-token groups per tile
  constexpr int TOK = 16 * NG;                // tokens per tile
  constexpr int EPC = 16 / ES;                // elements per 16-byte chunk
  constexpr int CHUNKS = D / EPC;             // chunks of a K row
  constexpr int KC = (CHUNKS + 3) / 4;        // chunks per lane and token
  constexpr int DT = (D + 15) / 16;
  constexpr int PB = BLK == 8 ? 2 : 1;        // blocks per group
  // K/V loads of the throughput shape carry the non-temporal hint (945 MB, replayed from a graph: 168 against 187 us); the
  // latency shape serves launches of a few megabytes, which run faster with plain loads
  constexpr bool STREAM = WAVES < 8;
  static_assert(D % EPC == 0 && (BLK == 8 || BLK == 16 || BLK == 32), "head size / block size");
  constexpr int NV = Q8 ? 1 : NG;             // pieces of a value row per lane and tile
  using VP = typename std::conditional<Q8, u32x4, u32x2>::type;

  const int split = blockIdx.x;
  const int kvh = blockIdx.y / a.head_groups, hgrp = blockIdx.y % a.head_groups;
  const int seq = blockIdx.z, num_seqs = gridDim.z;
  const int gqa = a.num_heads / a.num_kv_heads;
  const int head0 = kvh * gqa + hgrp * 16;
  const int nh = min(16, gqa - hgrp * 16);  // query heads of this workgroup
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c = lane & 15;

  // Ids of the blocks of a tile's groups, requested a tile ahead through the scalar cache: they are
  // wave-uniform, and a vector load would queue behind (and so wait for) the tiles in flight.  The
  // first ones do not wait for the sequence's length unless there is a window.
  typedef const __attribute__((address_space(4))) int32_t* ConstInt;
  const ConstInt table = (ConstInt)(a.block_tables + (int64_t)seq * a.table_width);
  struct Ids {
    int e[NG * PB];
  };
  auto load_ids = [&](int tile) {
    Ids id;
#pragma unroll
    for (int e = 0; e < NG * PB; ++e)
      id.e[e] = table[min((tile * NG * PB + e) * (16 / PB) / BLK, a.table_width - 1)];
    return id;
  };
  // the waves of all splits take the tiles in turn
  const int i0 = split * WAVES + wave, step = WAVES * a.num_splits;
  Ids ids = load_ids(a.window == 0 ? i0 : 0);
  // STEP: the lane's two elements of the new row's key and of its value, requested in front of the tiles
  uint32_t k_new = 0, v_new = 0;
  if constexpr (STEP) {
    const int e = min(lane, D / 2 - 1);
    k_new = reinterpret_cast<const uint32_t*>((const T*)a.new_key + (int64_t)seq * a.new_k_stride + (int64_t)kvh * D)[e];
    v_new = reinterpret_cast<const uint32_t*>((const T*)a.new_value + (int64_t)seq * a.new_v_stride + (int64_t)kvh * D)[e];
  }
  const int raw_len = ((ConstInt)a.seq_lens)[seq];
  const int64_t most = (int64_t)a.table_width * BLK;
  const int len = raw_len > most ? (int)most : max(raw_len, 0);
  uint32_t diag = raw_len > most ? PE_DIAG_DECODE_LEN_CLAMPED : 0;
  const WinRange R = win_range<TOK>(len, a.window, a.sinks);
  // STEP: the last tile, which takes the new row, is the first one of the last wave (the one with the
  // fewest tiles); it changes places with the tile that is there in order
  const int early = STEP ? min(step, R.tiles) - 1 : 0;
  auto at = [&](int i) { return R.tile(!STEP ? i : i == early ? R.tiles - 1 : i == R.tiles - 1 ? early : i); };
  if (i0 < R.tiles && (a.window != 0 || at(i0) != i0)) ids = load_ids(at(i0));
  auto visible = [&](int tok) { return (int)(tok < R.len) & ((int)(tok >= R.lo) | (int)(tok < R.sink_end)); };

  // ---- Q: the lane's chunks of head c, matched to the K chunks -------------------------------
  vec8 qf[KC][Q8 ? 2 : 1];
  {
    // (a lane without a head or a chunk reads a valid one and drops it)
    const T* qp = (const T*)a.query + (int64_t)seq * a.q_stride + (int64_t)(head0 + min(c, nh - 1)) * D;
#pragma unroll
    for (int kk = 0; kk < KC; ++kk)
#pragma unroll
      for (int e = 0; e < (Q8 ? 2 : 1); ++e) {
        const bool in = c < nh && 4 * kk + g < CHUNKS;
        const u32x4 raw = *reinterpret_cast<const u32x4*>(qp + min(4 * kk + g, CHUNKS - 1) * EPC + 8 * e);
        qf[kk][e] = __builtin_bit_cast(vec8, in ? raw : u32x4{0u, 0u, 0u, 0u});
      }
  }

  struct Tile {
    u32x4 k[NG][KC];
    VP v[NV][DT];
    f32x2 sc;      // 8-bit: scales of K and V of entry (lane * entries / 64)
    uint32_t bad;  // bit e: the block of entry e is outside the cache (wave-uniform)
  };
  const char* kbase = (const char*)a.key_cache + (int64_t)kvh * a.kv_head_stride * ES;
  const char* vbase = (const char*)a.value_cache + (int64_t)kvh * a.kv_head_stride * ES;
  const int64_t blk_bytes = a.kv_block_stride * ES;
  const uint32_t k_lane = PB == 1 ? g * (BLK * 16) + c * 16 : g * (BLK * 16) + (c & 7) * 16;
  const uint32_t v_lane = c * (BLK * ES) + (Q8 ? 0 : (PB == 1 ? 4 * g : 4 * (g & 1)) * ES);

  auto issue = [&](Tile& t, int tile, const Ids& id) {
    // An entry (8 or 16 tokens) without visible tokens may name anything, its block can have been
    // given away: the entry before it is read instead, or the first visible one.
    constexpr int NE = NG * PB, ET = 16 / PB;
    int use[NE], at = 0, seen = 0;
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      const int tok = (tile * NE + e) * ET;
      int v = (int)(tok < R.len) & ((int)(tok + ET > R.lo) | (int)(tok < R.sink_end));
      // (the block that the step appends to is needed whole, also where a window hides its first half)
      if constexpr (STEP) v |= (int)(tok / BLK == (R.len - 1) / BLK);
      at = v ? id.e[e] : at;
      seen |= v << e;
      use[e] = at;
    }
#pragma unroll
    for (int e = NE - 1; e >= 0; --e) {
      at = (seen >> e & 1) ? id.e[e] : at;
      use[e] = (seen & ((2 << e) - 1)) ? use[e] : at;
    }
    t.bad = 0;
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      const bool out_of_cache = (uint32_t)use[e] >= (uint64_t)a.num_blocks;
      t.bad |= out_of_cache ? (uint32_t)(seen & (1 << e)) : 0u;
      use[e] = out_of_cache ? 0 : use[e];
    }
    diag |= t.bad ? PE_DIAG_BLOCK_ID : 0;
#pragma unroll
    for (int h = 0; h < NG; ++h) {
      const int sub = BLK == 32 ? (tile * NG + h) & 1 : 0;
      int64_t ko;  // bytes from kbase
      if constexpr (PB == 1) ko = use[h] * blk_bytes + sub * 256;
      else ko = (c < 8 ? use[2 * h] : use[2 * h + PB - 1]) * blk_bytes;
      const char* kl = kbase + ko + k_lane;
#pragma unroll
      for (int kk = 0; kk < KC; ++kk) {
        t.k[h][kk] = u32x4{0u, 0u, 0u, 0u};
        if (4 * kk + 3 < CHUNKS || 4 * kk + g < CHUNKS)
          t.k[h][kk] = win_load<STREAM>(reinterpret_cast<const u32x4*>(kl + kk * (4 * BLK * 16)));
      }
    }
    if constexpr (Q8) {
      // the lane's group: g.  Scales: a vector load in line with K and V (a scalar one would be waited
      // for together with the next tile's ids), each lane the entry that lane * entries / 64 names.
      const char* vl[PB];
      int mine[PB];
#pragma unroll
      for (int p = 0; p < PB; ++p) {
        const int lo = g == 0 ? use[p] : use[PB + p], hi = g == 2 ? use[(NG - 2) * PB + p] : use[(NG - 1) * PB + p];
        mine[p] = g < 2 ? lo : hi;
        vl[p] = vbase + mine[p] * blk_bytes + (BLK == 32 ? (g & 1) * 16 : 0) + v_lane;
      }
      const int scaled = PB == 1 || c < 8 ? mine[0] : mine[PB - 1];
      t.sc = *reinterpret_cast<const f32x2*>(a.kv_scales + ((int64_t)scaled * a.num_kv_heads + kvh) * 2);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        if constexpr (PB == 1) {
          t.v[0][dt] = win_load<STREAM>(reinterpret_cast<const u32x4*>(vl[0] + dt * (16 * BLK)));
        } else {
          const u32x2 lo = win_load<STREAM>(reinterpret_cast<const u32x2*>(vl[0] + dt * (16 * BLK)));
          const u32x2 hi = win_load<STREAM>(reinterpret_cast<const u32x2*>(vl[PB - 1] + dt * (16 * BLK)));
          t.v[0][dt] = u32x4{lo[0], lo[1], hi[0], hi[1]};
        }
      }
    } else {
#pragma unroll
      for (int h = 0; h < NG; ++h) {
        int64_t vo;
        if constexpr (PB == 1) vo = use[h] * blk_bytes + (BLK == 32 ? ((tile * NG + h) & 1) * 32 : 0);
        else vo = (g < 2 ? use[2 * h] : use[2 * h + PB - 1]) * blk_bytes;
        const char* vl = vbase + vo + v_lane;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          t.v[h][dt] = VP{};
          if (16 * dt + 15 < D || 16 * dt + c < D)
            t.v[h][dt] = win_load<STREAM>(reinterpret_cast<const VP*>(vl + dt * (16 * BLK * ES)));
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);  // the requests stay in front of the arithmetic that follows
  };

  float m_run = WIN_NEG, l_run = 0.f;  // log2 units; l_run: this lane's tokens only
  // f16 products p * scale of V may leave f16's normal range; they are kept relative to their own
  // running maximum 2^c_run (p being relative to 2^m_run).  bf16 has the range.  c_run follows differences
  // of scores, which stay small where they matter however large the scores are.
  float c_run = WIN_NEG;
  constexpr bool WREF = Q8 && __is_same(T, _Float16);
  f32x4 acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x4{0.f, 0.f, 0.f, 0.f};

  auto compute = [&](Tile& t, int tile) {
    // A score is rounded once, before its maximum is taken and before that is subtracted: contracted into one
    // multiply-add the subtraction would leave the rounding of the maximum, which is 2^8 for scores of 2^32.
#pragma clang fp contract(off)
    const int t0 = tile * TOK;
    f32x4 s[NG];
#pragma unroll
    for (int h = 0; h < NG; ++h) {
      s[h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < KC; ++kk) {
        const u32x4 k = t.k[h][kk];
        if constexpr (Q8) {
          s[h] = TR::mfma16(codes8<T, C>(k[0], k[1]), qf[kk][0], s[h]);
          s[h] = TR::mfma16(codes8<T, C>(k[2], k[3]), qf[kk][1], s[h]);
        } else {
          s[h] = TR::mfma16(__builtin_bit_cast(vec8, k), qf[kk][0], s[h]);
        }
      }
    }
    // the lane's tokens lie in block 0 or 1 of a group: 8-token blocks switch at g = 2
    const int mine = PB == 1 ? 0 : g >> 1;
    const bool inside = t0 + TOK <= R.len && (t0 >= R.lo || t0 + TOK <= R.sink_end);
    const bool masked = !inside || t.bad != 0;  // wave-uniform
    // token 4g + r of group h
    auto shown = [&](int h, int r) {
      return visible(t0 + 16 * h + 4 * g + r) & (int)(~t.bad >> (h * PB + mine) & 1u);
    };
    float ks[NG], vs[NG];
#pragma unroll
    for (int h = 0; h < NG; ++h) {
      ks[h] = a.scale_log2;
      vs[h] = 1.f;
      if constexpr (Q8) {
        // entry e lies in lanes e * 64 / entries ...
        auto scale_of = [&](int e, int i) {
          return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(t.sc[i]), e * (16 / PB)));
        };
        ks[h] *= mine == 0 ? scale_of(h * PB, 0) : scale_of(h * PB + PB - 1, 0);
        vs[h] = mine == 0 ? scale_of(h * PB, 1) : scale_of(h * PB + PB - 1, 1);
      }
      s[h] *= ks[h];
    }
    if (masked) {
#pragma unroll
      for (int h = 0; h < NG; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[h][r] = shown(h, r) ? s[h][r] : -INFINITY;
    }
    float mx[NG];
#pragma unroll
    for (int h = 0; h < NG; ++h) mx[h] = fmaxf(fmaxf(s[h][0], s[h][1]), fmaxf(s[h][2], s[h][3]));
    float top = mx[0];
#pragma unroll
    for (int h = 1; h < NG; ++h) top = fmaxf(top, mx[h]);
    const float m_new = fmaxf(m_run, win_max_groups(top));
    float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
    l_run *= alpha;
    if constexpr (WREF) {
      float y = -INFINITY, lv[NG];
#pragma unroll
      for (int h = 0; h < NG; ++h) {
        // log2; -inf for a block of zeros and where nothing is visible (the scale may be anything)
        lv[h] = mx[h] > -INFINITY ? __builtin_amdgcn_logf(vs[h]) : -INFINITY;
        // A block of zeros moves the scores' maximum and not c: a group may lie any distance below the one and
        // at the top of the other.  Counted as no lower than 2^-126 (where p becomes 0 anyway) it keeps its factor
        // 2^(lv - c) within 2^126, so that 0 times the factor is 0.
        y = fmaxf(y, fmaxf(mx[h] - m_new, -126.f) + lv[h]);
      }
      const float c_old = c_run + (m_run - m_new);
      c_run = fmaxf(fmaxf(c_old, win_max_groups(y)), WIN_NEG);
      alpha = __builtin_amdgcn_exp2f(c_old - c_run);
#pragma unroll
      for (int h = 0; h < NG; ++h) vs[h] = __builtin_amdgcn_exp2f(lv[h] - c_run);
    }
    m_run = m_new;
    float w[NG][4];
#pragma unroll
    for (int h = 0; h < NG; ++h)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float p = __builtin_amdgcn_exp2f(s[h][r] - m_new);
        l_run += p;
        w[h][r] = Q8 ? p * vs[h] : p;
      }
    if (Q8 && masked) {  // a hidden token's scale may be anything
#pragma unroll
      for (int h = 0; h < NG; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r) w[h][r] = shown(h, r) ? w[h][r] : 0.f;
    }
    // The second matrix product takes its weights in the row type: one rounding of each, by at most 2^-8
    // (bf16) or 2^-11 (f16) of it; their sum l_run is of the unrounded ones, in f32 like the statistics.
    vec8 pf[NG / 2];
#pragma unroll
    for (int h = 0; h < NG; ++h)
#pragma unroll
      for (int r = 0; r < 4; ++r) pf[h >> 1][(h & 1) * 4 + r] = (T)w[h][r];
    // hidden slots may hold anything (NaN included): their values become zero
    if constexpr (Q8) {
      if (masked) {
        u32x4 keep;
#pragma unroll
        for (int w4 = 0; w4 < 4; ++w4) {
          uint32_t mk = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int v = visible(t0 + 16 * g + 4 * w4 + e) & (int)(~t.bad >> (g * PB + (PB == 1 ? 0 : w4 >> 1)) & 1u);
            mk |= v ? 0xffu << (8 * e) : 0u;
          }
          keep[w4] = mk;
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) t.v[0][dt] &= keep;
      }
      // P to the lane group of its tokens: register j of lane group h <- register h of lane group j
      uint32_t pt[4][2];
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const u32x4 two = __builtin_bit_cast(u32x4, pf[h >> 1]);
        pt[h][0] = two[(h & 1) * 2];
        pt[h][1] = two[(h & 1) * 2 + 1];
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const auto x = __builtin_amdgcn_permlane32_swap(pt[h][e], pt[h + 2][e], false, false);
          pt[h][e] = x[0];
          pt[h + 2][e] = x[1];
        }
#pragma unroll
        for (int h = 0; h < 4; h += 2) {
          const auto x = __builtin_amdgcn_permlane16_swap(pt[h][e], pt[h + 1][e], false, false);
          pt[h][e] = x[0];
          pt[h + 1][e] = x[1];
        }
      }
      const vec8 p0 = __builtin_bit_cast(vec8, u32x4{pt[0][0], pt[0][1], pt[1][0], pt[1][1]});
      const vec8 p1 = __builtin_bit_cast(vec8, u32x4{pt[2][0], pt[2][1], pt[3][0], pt[3][1]});
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const u32x4 v = t.v[0][dt];
        acc[dt] *= alpha;
        acc[dt] = TR::mfma16(codes8<T, C>(v[0], v[1]), p0, acc[dt]);
        acc[dt] = TR::mfma16(codes8<T, C>(v[2], v[3]), p1, acc[dt]);
      }
    } else {
      if (masked) {
#pragma unroll
        for (int h = 0; h < NG; ++h) {
          const u32x2 keep = {(shown(h, 0) ? 0xffffu : 0u) | (shown(h, 1) ? 0xffff0000u : 0u),
                              (shown(h, 2) ? 0xffffu : 0u) | (shown(h, 3) ? 0xffff0000u : 0u)};
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) t.v[h][dt] &= keep;
        }
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const u32x2 lo = t.v[0][dt], hi = t.v[NV - 1][dt];
        acc[dt] *= alpha;
        acc[dt] = TR::mfma16(__builtin_bit_cast(vec8, u32x4{lo[0], lo[1], hi[0], hi[1]}), pf[0], acc[dt]);
      }
    }
  };

  // dynamic LDS: o[WAVES][nh][16 * DT + 4], m[WAVES][16], l[WAVES][16] (f32), STEP: codes of the new row
  extern __shared__ __attribute__((aligned(16))) float win_smem[];
  constexpr int OROW = 16 * DT + 4;
  const int heads = min(16, gqa);
  float* sm_o = win_smem;
  float* sm_m = win_smem + WAVES * heads * OROW;
  float* sm_l = sm_m + WAVES * 16;

  // ---- STEP: the new row into the cache and the last tile ---------------------------------------
  // Returns whether the tile has to be read again: a row larger than everything before it changes the
  // older codes of its block, in memory (rare).
  auto append = [&](Tile& t, int tile) -> bool {
    if constexpr (STEP) {
      constexpr int NE = NG * PB, ET = 16 / PB;
      const int pos = R.len - 1, o = pos % BLK;  // position, slot in its block
      const int hn = (pos >> 4) - tile * NG, en = pos / ET - tile * NE;
      if (t.bad >> en & 1) return false;  // its block is outside the cache
      const int64_t blk = table[pos / BLK];
      const uint32_t ka = win_max_wave(max(finite_bits<T>(k_new & 0xffffu), finite_bits<T>(k_new >> 16)));
      const uint32_t va = win_max_wave(max(finite_bits<T>(v_new & 0xffffu), finite_bits<T>(v_new >> 16)));
      auto old_scale = [&](int i) {
        return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(t.sc[i]), en * (64 / NE)));
      };
      const Joined kj = join_scale<C>(o > 0, old_scale(0), bits_value<T>(ka));
      const Joined vj = join_scale<C>(o > 0, old_scale(1), bits_value<T>(va));
      char* kw = const_cast<char*>(kbase) + blk * blk_bytes;
      char* vw = const_cast<char*>(vbase) + blk * blk_bytes;
      const bool grew = __builtin_amdgcn_ballot_w64(kj.grew || vj.grew) != 0;  // wave-uniform
      if (__builtin_expect(grew, 0)) {  // (17 x 1028 of 4104 tokens, 8-token blocks: 11.3 us, without the hint 11.6)
        if (kj.grew)
          for (int it = lane; it < CHUNKS * o * 4; it += 64)
            reencode_word<C>(reinterpret_cast<uint32_t*>(kw + it / (o * 4) * (BLK * 16)) + it % (o * 4), kj.factor());
        if (vj.grew)
          for (int it = lane; it < D * o; it += 64)
            reencode_byte<C>(reinterpret_cast<uint8_t*>(vw + it / o * BLK + it % o), vj.factor());
      }
      // The lane's four codes, to memory as they are (V) and through LDS to the lanes whose registers they
      // belong in: key codes in order, value codes (c, dt) at 8 c + dt.
      auto enc = [&](auto exact) {
        constexpr bool EXACT = decltype(exact)::value;
        return encode4<C>(kj.divide<EXACT>(bits_value<T>(k_new & 0xffffu)), kj.divide<EXACT>(bits_value<T>(k_new >> 16)),
                          vj.divide<EXACT>(bits_value<T>(v_new & 0xffffu)), vj.divide<EXACT>(bits_value<T>(v_new >> 16)));
      };
      const uint32_t codes = kj.exact && vj.exact ? enc(std::true_type{}) : enc(std::false_type{});
      uint8_t* row = reinterpret_cast<uint8_t*>(sm_l + WAVES * 16);
      if (lane < D / 2) {
        const int d = 2 * lane;
        reinterpret_cast<uint16_t*>(row)[lane] = (uint16_t)codes;
        row[128 + 8 * (d & 15) + (d >> 4)] = (uint8_t)(codes >> 16);
        row[128 + 8 * ((d + 1) & 15) + (d >> 4)] = (uint8_t)(codes >> 24);
        reinterpret_cast<uint8_t*>(vw)[d * BLK + o] = (uint8_t)(codes >> 16);
        reinterpret_cast<uint8_t*>(vw)[(d + 1) * BLK + o] = (uint8_t)(codes >> 24);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (one wave: its LDS accesses stay in order)
      __builtin_amdgcn_wave_barrier();
      // K: the row is token pos & 15 of group hn
      const bool here = c == (pos & 15);
#pragma unroll
      for (int kk = 0; kk < KC; ++kk) {
        const int ch = min(4 * kk + g, CHUNKS - 1);
        const u32x4 code = *reinterpret_cast<const u32x4*>(row + 16 * ch);
#pragma unroll
        for (int h = 0; h < NG; ++h)
          if (here && h == hn) t.k[h][kk] = code;
        if (here && 4 * kk + g < CHUNKS) *reinterpret_cast<u32x4*>(kw + (ch * BLK + o) * 16) = code;
      }
      // V: the lanes of group g hold its 16 tokens of row 16 dt + c; the row goes to byte pos & 15
      const bool mine = BLK == 32 ? (g >> 1) == (hn >> 1) : g == hn;
      const u32x2 vc = *reinterpret_cast<const u32x2*>(row + 128 + 8 * c);
      const uint32_t sh = 8 * (pos & 3);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t put = g == hn && ((pos & 15) >> 2) == w ? 0xffu << sh : 0u;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const uint32_t code = (vc[dt >> 2] >> (8 * (dt & 3)) & 0xffu) << sh;
          t.v[0][dt][w] = (t.v[0][dt][w] & ~put) | (code & put);
        }
      }
      const bool scaled = BLK == 8 ? lane * NE / 64 == en : mine;
      if (scaled) t.sc = f32x2{kj.scale, vj.scale};
      if (lane == 0) {
        float* sc = const_cast<float*>(a.kv_scales) + (blk * a.num_kv_heads + kvh) * 2;
        *reinterpret_cast<f32x2*>(sc) = f32x2{kj.scale, vj.scale};
      }
      if (grew) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "agent");  // the stores before the next loads
      return grew;
    }
    return false;
  };

  // ---- the wave's tiles ------------------------------------------------------------------------
  // (A second tile in flight gains nothing, replayed from a graph: 167.8 against 167.6 us on 945 MB, 21.5 against 20.3 on
  // 64 x 776 tokens; the waves of a CU hold 128 KiB in flight as it is.  A tile number past the end
  // only names table entries, which load_ids keeps inside the row.)
  for (int i = i0; i < R.tiles; i += step) {
    Tile t;
    bool owner = STEP && i == early;
    if (owner && raw_len > most) {
      diag |= PE_DIAG_APPEND_MISMATCH;
      owner = false;
    }
    while (true) {  // twice where the row grew its block's scale
      issue(t, at(i), ids);
      if (!owner || !append(t, at(i))) break;
      owner = false;
    }
    ids = load_ids(at(i + step));
    compute(t, at(i));
  }
  if (diag != 0 && lane == 0) atomicOr(&window_diag_word, diag);

  // ---- join the lane groups' sums, then the waves through LDS ---------------------------------
  l_run += __shfl_xor(l_run, 16);
  l_run += __shfl_xor(l_run, 32);
  if constexpr (WREF) {  // numerators relative to the same point as the sum
    const float f = __builtin_amdgcn_exp2f(c_run);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt] *= f;
  }
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
      float* w = a.ws + (((int64_t)split * num_seqs + seq) * a.num_heads + head) * win_ws_stride(D);
      if (d == 0) {
        w[0] = m_tot;
        w[1] = l;
      }
      w[2 + d] = o;
    }
  }
}

// Joins the splits of one (query head, sequence): all partials (at most MS) are read at once.
template <typename T, int MS>
__global__ __launch_bounds__(256) void paged_window_merge_kernel(T* __restrict__ out, const float* __restrict__ ws,
                                                                  int num_heads, int head_size, int num_splits) {
  const int head = blockIdx.x, seq = blockIdx.y, d = threadIdx.x;
  const int64_t split_stride = (int64_t)gridDim.y * num_heads * win_ws_stride(head_size);
  const float* w = ws + ((int64_t)seq * num_heads + head) * win_ws_stride(head_size);
  float m[MS], l[MS], o[MS];
#pragma unroll
  for (int s = 0; s < MS; ++s) {
    // (past the last split: the last one again, with a weight of 0)
    const float* p = w + min(s, num_splits - 1) * split_stride;
    m[s] = p[0];
    l[s] = s < num_splits ? p[1] : 0.f;
    o[s] = s < num_splits ? p[2 + min(d, head_size - 1)] : 0.f;
  }
  float m_tot = m[0], lt = 0.f, ot = 0.f;
#pragma unroll
  for (int s = 1; s < MS; ++s) m_tot = fmaxf(m_tot, m[s]);
#pragma unroll
  for (int s = 0; s < MS; ++s) {
    const float f = __builtin_amdgcn_exp2f(m[s] - m_tot);
    lt += f * l[s];
    ot += f * o[s];
  }
  if (d < head_size) out[((int64_t)seq * num_heads + head) * head_size + d] = (T)(lt == 0.f ? 0.f : ot / lt);
}

template <typename T, typename C, int D, int WAVES, int BLK, bool STEP>
inline void launch_window(const WinArgs& a, dim3 grid, hipStream_t st) {
  constexpr int DT = (D + 15) / 16;
  const int gqa = a.num_heads / a.num_kv_heads, heads = gqa < 16 ? gqa : 16;
  const size_t lds = ((size_t)WAVES * heads * (16 * DT + 4) + 2 * WAVES * 16) * 4 + (STEP ? 256 : 0);
  if (lds > 64 * 1024)
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&paged_window_kernel<T, C, D, WAVES, BLK, STEP>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  hipLaunchKernelGGL((paged_window_kernel<T, C, D, WAVES, BLK, STEP>), grid, dim3(WAVES * 64), lds, st, a);
  if (a.num_splits == 1) return;
  const dim3 mg((unsigned)a.num_heads, grid.z), mb(D <= 64 ? 64 : D <= 128 ? 128 : 256);
#define PE_WIN_MERGE(MS) \
  hipLaunchKernelGGL((paged_window_merge_kernel<T, MS>), mg, mb, 0, st, (T*)a.out, a.ws, a.num_heads, D, a.num_splits)
  if (a.num_splits <= 4) PE_WIN_MERGE(4);
  else if (a.num_splits <= 8) PE_WIN_MERGE(8);
  else if (a.num_splits <= 16) PE_WIN_MERGE(16);
  else PE_WIN_MERGE(32);
#undef PE_WIN_MERGE
}

template <typename T, typename C, int D, bool STEP>
inline int dispatch_window_block(const WinArgs& a, int block_size, int waves, dim3 grid, hipStream_t st) {
  constexpr int WIDE = win_wide(D, STEP);
  if (waves == WIDE) switch (block_size) {
    case 8: launch_window<T, C, D, WIDE, 8, STEP>(a, grid, st); return PE_OK;
    case 16: launch_window<T, C, D, WIDE, 16, STEP>(a, grid, st); return PE_OK;
    case 32: launch_window<T, C, D, WIDE, 32, STEP>(a, grid, st); return PE_OK;
  }
  switch (block_size) {
    case 8: launch_window<T, C, D, 4, 8, STEP>(a, grid, st); return PE_OK;
    case 16: launch_window<T, C, D, 4, 16, STEP>(a, grid, st); return PE_OK;
    case 32: launch_window<T, C, D, 4, 32, STEP>(a, grid, st); return PE_OK;
  }
  return fail(PE_ERR_UNSUPPORTED, "paged_decode_window: block size %d (8, 16 or 32)", block_size);
}

// head sizes of one translation unit; the 16-bit cache also has 120
template <typename T, typename C, bool STEP = false>
inline int dispatch_window(const WinArgs& a, int head_size, int block_size, int waves, dim3 grid, hipStream_t st) {
  switch (head_size) {
    case 32: return dispatch_window_block<T, C, 32, STEP>(a, block_size, waves, grid, st);
    case 64: return dispatch_window_block<T, C, 64, STEP>(a, block_size, waves, grid, st);
    case 128: return dispatch_window_block<T, C, 128, STEP>(a, block_size, waves, grid, st);
    case 80: return dispatch_window_block<T, C, 80, STEP>(a, block_size, waves, grid, st);
    case 96: return dispatch_window_block<T, C, 96, STEP>(a, block_size, waves, grid, st);
    case 112: return dispatch_window_block<T, C, 112, STEP>(a, block_size, waves, grid, st);
    // (larger heads have no registers left for the append: pe_decode_step_8bit writes their row first)
    case 192:
      if constexpr (!STEP) return dispatch_window_block<T, C, 192, STEP>(a, block_size, waves, grid, st);
      break;
    case 256:
      if constexpr (!STEP) return dispatch_window_block<T, C, 256, STEP>(a, block_size, waves, grid, st);
      break;
    case 120:
      if constexpr (__is_same(T, C)) return dispatch_window_block<T, C, 120, STEP>(a, block_size, waves, grid, st);
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
