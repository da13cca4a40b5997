// Varlen causal prefill attention on gfx950 (flash-style, no L_q x L_kv matrix in memory).
//
// Mask: query row i of a request attends kv rows 0..min(i, L_kv-1) — the top-left aligned
// lower triangle that scaled_dot_product_attention(is_causal=True) applies, which is what
// the reference runs when the prompt was pruned before attention (L_kv < L_q).
// Grouped KV heads are addressed directly (no repeat_interleave copy).
//
// MFMA path (16-bit types; head sizes 64 and 128 as they are, 256 with 8-wave workgroups, and the
// other sizes of the reference's list - 32, 80, 96, 112, 120, 192, vllm/attention/ops/paged_attn.py:37 -
// in the next larger of those row pitches with the chunks past the head never used):
// a workgroup of 4 waves owns 128 query rows of
// one (request, head); K/V tiles of 64 tokens stream global -> LDS directly (LDS-DMA loads,
// double-buffered: tile j+1 is in flight during the math of tile j).
//   S^T = K.Q^T   v_mfma_f32_16x16x32: A = K rows from LDS (ds_read_b128, XOR-swizzled
//                 chunks), B = Q fragments held in registers; a lane ends up with 4 tokens
//                 x 1 query row, so the row max/sum is a register reduction + 2 shuffles.
//   O^T += V^T.P^T  A = V^T read with ds_read_b64_tr_b16 from the row-major V tile, B = P
//                 taken straight from the S^T accumulators (k-slot order chosen to match).
// The finished O tile goes through LDS so that global stores are whole 16-byte row chunks.
//
// This file holds the kernel template; prefill.hip instantiates the causal form (and has the general
// kernel), prefill_window.hip the windowed one (WIN): query row i attends kv rows j <= min(i, L_kv-1)
// with j > i - window (window 0: all of them) or j < sinks.  A workgroup then visits the tiles that
// hold sinks and the tiles from its first row's window on, and a wave computes a tile only if one of
// its rows sees it, without mask code if all of them see all of it.  The waves of a workgroup take the same
// rows of several query heads of a KV head, so that they see the same keys.  Bound: matrix and vector
// instructions of a wave one after the other, as in the causal form, and at short windows the two partly
// visible ends: 4 x 8192 tokens, 32 / 8 heads x 128, window 1024, 16 sinks: 617 us a pass, 766 TFLOP/s (visible
// pairs only); 8 x 1024, window 256: 70 us, 392 TFLOP/s, with the inputs read at 2.2 TB/s beside it (passes over
// three sets of inputs, one after the other; a launch alone under the profiler takes 5 to 15 % longer).
#pragma once
#include "pe_common.h"

#include <cstdlib>
#include <type_traits>

namespace pe {

constexpr int PF_BN = 64;   // kv rows per tile
constexpr int PF_DEFAULT_SHAPE = 24;
constexpr float PF_NEG = -1.0e30f;
constexpr float PF_LAZY_LOG2 = 6.0f;  // weights may reach 2^6 before the reference point moves

typedef __attribute__((ext_vector_type(4))) short s16x4;

template <int D>
__device__ __forceinline__ int swz_off(int row, int chunk) {
  // byte offset of 16-byte chunk `chunk` of row `row` in the [rows][D] 16-bit K tile: the 16 rows
  // a ds_read_b128 lane group touches land on 16 different 16-byte slots of the 256-byte bank row
  constexpr int CPR = D / 8;
  const int x = (CPR >= 16) ? (row & 15) : ((row >> 1) & 7);
  return row * (D * 2) + ((chunk ^ x) << 4);
}

template <int D>
__device__ __forceinline__ int swz_off_v(int row, int chunk) {
  // V tile: a 32-lane half of ds_read_b64_tr_b16 takes 8 consecutive rows x 32 bytes (one chunk
  // pair per row); XOR-ing the pair index with the row puts the 8 rows on 8 different 32-byte
  // spans of the bank row
  constexpr int CPR = D / 8;
  const int x = (CPR >= 16) ? ((row & 7) << 1) : (((row >> 1) & 3) << 1);
  return row * (D * 2) + ((chunk ^ x) << 4);
}

// D: row pitch of the K/V tiles in LDS and width of the fragment loops (64, 128 or 256 elements);
// the head itself has head_size <= D elements (a multiple of 8).  NR: 16-row query tiles per wave;
// WAVES: waves per workgroup (query rows per workgroup = 16 * NR * WAVES); WPE: waves per SIMD the
// register budget is cut for.
// max over the four lanes l, l^16, l^32, l^48 with the row-swap permutes (VALU, no LDS round
// trip as a ds_bpermute shuffle would take): v_permlane32_swap exchanges the upper half of its
// first operand with the lower half of its second, v_permlane16_swap the odd 16-lane rows of the
// first with the even rows of the second; with both operands equal the two results hold, in
// every lane, the lane's own value and its partner's.
__device__ __forceinline__ float max_xor_16_32(float x) {
  unsigned u = __float_as_uint(x);
  auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  u = __float_as_uint(x);
  auto b = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

template <typename T, int D, int NR, int WAVES, int WPE, bool WIN = false, int BN = PF_BN>
__global__ __launch_bounds__(WAVES * 64, WPE) void prefill_mfma_kernel(
    T* __restrict__ out, const T* __restrict__ q, const T* __restrict__ k,
    const T* __restrict__ v, const int32_t* __restrict__ cu_q, const int32_t* __restrict__ cu_kv,
    int num_heads, int num_kv_heads, int head_size, int64_t q_stride, int64_t k_stride,
    int64_t v_stride, int64_t out_stride, float scale_log2e, int window, int sinks,
    int heads_per_wg, int num_q_rows, int num_kv_rows) {
  // window and what follows: WIN only
  using TR = Traits<T>;
  using vec8 = typename TR::vec8;
  constexpr int KS = D / 32;
  constexpr int DT = D / 16;
  constexpr int NS = BN / 16;                       // 16-key groups of a tile
  constexpr int CPR = D / 8;                        // 16-byte chunks per row
  constexpr int TILE_BYTES = BN * D * 2;         // one K or V tile
  constexpr int WROWS = 16 * NR;                    // query rows per wave
  constexpr int BM = WROWS * WAVES;                 // query rows per workgroup
  static_assert(BM % BN == 0 && BM * D * 2 <= 4 * TILE_BYTES, "tile shape");

  extern __shared__ __attribute__((aligned(16))) char smem[];
  // [buf][K|V][tile]
  auto k_tile = [&](int buf) { return smem + buf * 2 * TILE_BYTES; };
  auto v_tile = [&](int buf) { return smem + buf * 2 * TILE_BYTES + TILE_BYTES; };

  // grid (head, request, query tile): workgroups are dispatched x-fastest, so every request's
  // heaviest (last) query tiles start first and the short ones fill the tail.  Consecutive
  // workgroup ids go to consecutive XCDs; the (head, request) plane is re-enumerated so that all
  // query heads of one (request, KV head) - which read the same K/V - get ids that are equal
  // modulo 8 and share one XCD's L2 (needs num_kv_heads * num_requests to be a multiple of 8).
  // WIN: the waves of a workgroup take the same query rows of heads_per_wg query heads of one KV head
  // (and, where there are more waves, further rows), so that they see nearly the same keys: a
  // workgroup streams window + rows / heads_per_wg keys instead of window + rows.
  const int hpw = WIN ? heads_per_wg : 1;
  const int gqa = num_heads / num_kv_heads / hpw;  // workgroups side by side on a KV head
  const int lid = (int)blockIdx.x + (int)gridDim.x * (int)blockIdx.y;
  const int n_groups = num_kv_heads * (int)gridDim.y;
  int grp, hg;
  if (n_groups % 8 == 0) {
    grp = (lid / (8 * gqa)) * 8 + lid % 8;
    hg = (lid / 8) % gqa;
  } else {
    grp = lid / gqa;
    hg = lid % gqa;
  }
  const int seq = grp / num_kv_heads;
  const int kvh = grp % num_kv_heads;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int head = WIN ? (kvh * gqa + hg) * hpw + wave % hpw : kvh * gqa + hg;
  const int bm = WIN ? BM / hpw : BM;  // query rows per workgroup and head
  const int q0 = cu_q[seq], lq = (WIN ? min(cu_q[seq + 1], num_q_rows) : cu_q[seq + 1]) - q0;
  const int kv0 = cu_kv[seq], lkv = (WIN ? min(cu_kv[seq + 1], num_kv_rows) : cu_kv[seq + 1]) - kv0;
  if (WIN && ((q0 | kv0) < 0 || cu_q[seq + 1] < q0 || cu_kv[seq + 1] < kv0)) return;  // no prefix sums
  const int qt = (int)gridDim.z - 1 - (int)blockIdx.z;
  const int m0 = qt * bm;
  if (m0 >= lq) return;

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int g = lane >> 4, c = lane & 15;
  const int wrow0 = m0 + (WIN ? wave / hpw : wave) * WROWS;  // first query row of this wave
  const int hchunks = head_size >> 3;   // 16-byte chunks of a head row that exist (<= CPR)

  // ---- Q fragments (B operand): lane holds Q[row][32ks + 8g .. +8) for its row tiles ----
  vec8 qf[NR][KS];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const int row = min(wrow0 + n * 16 + c, lq - 1);
    const T* qp = q + (int64_t)(q0 + row) * q_stride + (int64_t)head * head_size + 8 * g;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      // a chunk past the head is zero in Q, so whatever its K slot holds contributes nothing
      u32x4 raw = {0u, 0u, 0u, 0u};
      if (4 * ks + g < hchunks) raw = *reinterpret_cast<const u32x4*>(qp + 32 * ks);
      qf[n][ks] = __builtin_bit_cast(vec8, raw);
    }
  }

  // The row sums ride on the matrix pipe: one more MFMA per P fragment with an all-ones A operand
  // adds the (storage-type rounded) probabilities of a query row over the fragment's 32 keys, in
  // every lane of the row's column - no vector adds per element, no cross-lane sum at the end,
  // and numerator and denominator use the same rounded weights.
  // WIN: a row starts below every finite score (f32's lowest number)
  constexpr float NEG = WIN ? -3.402823466e38f : PF_NEG;
  float m_run[NR];
  f32x4 acc_l[NR];
  f32x4 acc[DT][NR];
  vec8 ones;
#pragma unroll
  for (int j = 0; j < 8; ++j) ones[j] = (T)1.0f;
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    m_run[n] = NEG;
    acc_l[n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const int kv_end = min(lkv, m0 + bm);  // rows past the last query row are never attended
  const int n_tiles = (kv_end + BN - 1) / BN;
  // WIN: the tiles visited are [0, ns) (sinks) and [tw, n_tiles) (windows of the workgroup's rows)
  int ns = 0, tw = 0;
  if constexpr (WIN) {
    const int lo = window > 0 ? max(0, m0 - window + 1) : 0;
    tw = lo / BN;
    ns = min((min(sinks, kv_end) + BN - 1) / BN, tw);
  }

  // Staging: K/V tiles go global -> LDS directly (global_load_lds_dwordx4, no registers, no
  // ds_write).  One wave-instruction fills 1 KiB of LDS contiguously in lane order: RPI whole tile
  // rows, lane l -> row l / CPR, 16-byte slot l % CPR.  The XOR swizzle of the LDS image is applied
  // to the per-lane SOURCE chunk instead (slot s of a row holds chunk s ^ x(row)).  Wave w issues
  // instruction i for rows i * RSTEP + w * RPI ..., so x(row) does not depend on i (RSTEP is a
  // multiple of 16) and the per-lane source offset is one constant; tile and i go into the scalar
  // base.  Only the ragged last tile of a request clamps its rows per lane.  The loads are asm
  // statements the compiler does not count: stage_wait() + a barrier must separate them from the
  // reads of the tile.
  constexpr int RPI = 64 / CPR;            // tile rows per wave-instruction
  constexpr int RSTEP = WAVES * RPI;       // rows between a wave's consecutive instructions
  constexpr int NINST = BN / RSTEP;     // instructions per wave per operand tile
  static_assert(RSTEP % 16 == 0 && NINST >= 1 && NINST * RSTEP == BN, "staging shape");
  const int lrow = wave * RPI + lane / CPR;  // row within a RSTEP group
  const int lslot = lane % CPR;
  const char* k_seq = reinterpret_cast<const char*>(k + (int64_t)kv0 * k_stride + (int64_t)kvh * head_size);
  const char* v_seq = reinterpret_cast<const char*>(v + (int64_t)kv0 * v_stride + (int64_t)kvh * head_size);
  const uint32_t k_row_bytes = (uint32_t)k_stride * 2u, v_row_bytes = (uint32_t)v_stride * 2u;
  // source chunk for this lane's slot: the inverse of swz_off / swz_off_v (XOR is an involution)
  // (a slot whose chunk lies past the head is filled with the row's chunk 0 instead: finite data
  //  that meets the zero chunk of Q, or - in V - feeds output columns nobody stores)
  uint32_t k_chunk16 = (uint32_t)(swz_off<D>(lrow, lslot) - lrow * (D * 2));
  uint32_t v_chunk16 = (uint32_t)(swz_off_v<D>(lrow, lslot) - lrow * (D * 2));
  if ((int)(k_chunk16 >> 4) >= hchunks) k_chunk16 = 0;
  if ((int)(v_chunk16 >> 4) >= hchunks) v_chunk16 = 0;
  uint32_t k_lane_off = (uint32_t)lrow * k_row_bytes + k_chunk16;
  uint32_t v_lane_off = (uint32_t)lrow * v_row_bytes + v_chunk16;
  // (the multiply-add has a 64-bit result: opaque copies keep half of it alive through the tiles, not all)
  if constexpr (WIN) asm volatile("" : "+v"(k_lane_off), "+v"(v_lane_off), "+v"(k_chunk16), "+v"(v_chunk16));
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem +
                        (uint32_t)wave * 1024u;
  // M0 carries the LDS destination of an LDS-DMA load and nothing else in this kernel (the
  // compiler keeps no value in it: every access to M0 in the generated code is one of the moves
  // below).  A load may not read an SGPR that a vector
  // instruction wrote fewer than 5 issue slots earlier: the first load of a tile waits that out;
  // the operands of the following ones are scalar sums of values that existed before it.
  auto glds16 = [](const char* base, uint32_t lane_off, uint32_t lds_dst, auto first_tag) {
    if constexpr (decltype(first_tag)::value) {
      asm volatile(
          "s_nop 4\n\t"
          "s_mov_b32 m0, %2\n\t"
          "s_nop 0\n\t"
          "global_load_lds_dwordx4 %0, %1"
          :
          : "v"(lane_off), "s"(base), "s"(lds_dst)
          : "memory");
    } else {
      asm volatile(
          "s_mov_b32 m0, %2\n\t"
          "s_nop 0\n\t"
          "global_load_lds_dwordx4 %0, %1"
          :
          : "v"(lane_off), "s"(base), "s"(lds_dst)
          : "memory");
    }
  };
  auto stage = [&](int tile, int buf) {
    const int t0 = tile * BN;
    const char* kb = k_seq + (int64_t)t0 * k_row_bytes;
    const char* vb = v_seq + (int64_t)t0 * v_row_bytes;
    const uint32_t kd = lds0 + (uint32_t)buf * (2u * TILE_BYTES);
    const uint32_t vd = kd + TILE_BYTES;
    if (t0 + BN <= lkv) {
      glds16(kb, k_lane_off, kd, std::true_type{});
      glds16(vb, v_lane_off, vd, std::false_type{});
#pragma unroll
      for (int i = 1; i < NINST; ++i) {
        glds16(kb + (int64_t)(i * RSTEP) * k_row_bytes, k_lane_off, kd + i * RSTEP * D * 2, std::false_type{});
        glds16(vb + (int64_t)(i * RSTEP) * v_row_bytes, v_lane_off, vd + i * RSTEP * D * 2, std::false_type{});
      }
    } else {
      const int last = lkv - 1 - t0;  // >= 0: a staged tile starts inside the request
#pragma unroll
      for (int i = 0; i < NINST; ++i) {
        const uint32_t row = (uint32_t)min(lrow + i * RSTEP, last);
        // (the row offsets are per-lane values, the scalar operands are the first load's)
        if (i == 0) {
          glds16(kb, row * k_row_bytes + k_chunk16, kd, std::true_type{});
        } else {
          glds16(kb, row * k_row_bytes + k_chunk16, kd + i * RSTEP * D * 2, std::false_type{});
        }
        glds16(vb, row * v_row_bytes + v_chunk16, vd + i * RSTEP * D * 2, std::false_type{});
      }
    }
  };
  auto stage_wait = [] { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); };

  // O^T += V^T.P^T over 32 keys of a tile, and the row sums
  // transposed read: lane i of each 16-lane group addresses row (4g + i/4), columns
  // 16dt + 4*(i%4) .. +4 and receives column 16dt+i of the group's 4 rows
  auto pv_step = [&](const char* vt, int k2, const vec8 (&pf)[NR][NS / 2]) {
    const int tq = c >> 2, tp = c & 3;
#pragma unroll
    for (int n = 0; n < NR; ++n) acc_l[n] = TR::mfma16(ones, pf[n][k2], acc_l[n]);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const int row_lo = (2 * k2) * 16 + 4 * g + tq;
      const int row_hi = row_lo + 16;
      const int ch = 2 * dt + (tp >> 1);
      const int sub8 = (tp & 1) * 8;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4*)(vt + swz_off_v<D>(row_lo, ch) + sub8));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4*)(vt + swz_off_v<D>(row_hi, ch) + sub8));
      typedef __attribute__((ext_vector_type(8))) short s16x8;
      const s16x8 both = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      const vec8 vf = __builtin_bit_cast(vec8, both);
#pragma unroll
      for (int n = 0; n < NR; ++n) acc[dt][n] = TR::mfma16(vf, pf[n][k2], acc[dt][n]);
    }
  };

  // The reference point of the exponentials only has to be NEAR the row's maximum: it moves
  // (and the accumulators are rescaled) when some row of the wave outgrew it by more than
  // 2^PF_LAZY_LOG2, so the weights stay below that factor and the rescale, frequent with a
  // strict running maximum, becomes rare.  The normalised output does not depend on it.
  //
  // WIN, far: a weight's multiply-add subtracts the rounded point from an exact product, so all weights of a row
  // carry 2^(the point's rounding): up to 2^1 at scores of 2^24, past the weights' range at 2^28 (f16) and 2^31
  // (bf16).  A wave that has met scores of 2^24 rounds its scores before it subtracts.  (Costs 0.5 to 2 %: 8 x
  // 1024, window 256: 67.6 -> 68.1 us, 4 x 8192, window 1024: 606 -> 616, both replayed from a graph.)
  bool far = false;
  auto move_reference = [&](int n, float m_tile) {
    if (__builtin_amdgcn_ballot_w64(m_tile > m_run[n] + PF_LAZY_LOG2) == 0) return;  // wave-uniform
    const float m_new = fmaxf(m_run[n], m_tile);
    const float alpha = __builtin_amdgcn_exp2f(m_run[n] - m_new);
    m_run[n] = m_new;
    acc_l[n] *= alpha;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt][n] *= alpha;
    if constexpr (WIN) far |= __builtin_amdgcn_ballot_w64(m_new > NEG && fabsf(m_new) > 16777216.f) != 0;
  };
  // the weights of row tile n are 2^(s * (what this returns) - m_ref)
  auto weight_factor = [&](f32x4 (&s)[NS][NR], int n, float& m_ref) -> float {
    m_ref = m_run[n];
    if (!WIN || !far) return scale_log2e;
#pragma unroll
    for (int sub = 0; sub < NS; ++sub)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
#pragma clang fp contract(off)
        s[sub][n][r] = s[sub][n][r] * scale_log2e - m_ref;
      }
    m_ref = 0.f;
    return 1.f;
  };

  auto compute = [&](int tile, int buf, auto masked_tag) {
    constexpr bool MASKED = decltype(masked_tag)::value;
    const int n0 = tile * BN;
    const char* kt = k_tile(buf);
    const char* vt = v_tile(buf);
    // ---- S^T = K.Q^T ---------------------------------------------------------------
    // The K fragments of row group sub+1 are requested before the MFMAs of group sub are issued
    // (the scheduling fences keep that order), so that an MFMA waits for reads issued a whole
    // group earlier instead of for the read right in front of it.
    f32x4 s[NS][NR];
    vec8 kf[2][KS];
    auto load_k = [&](int sub, vec8* dst) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        dst[ks] = __builtin_bit_cast(
            vec8, *reinterpret_cast<const u32x4*>(kt + swz_off<D>(sub * 16 + c, 4 * ks + g)));
    };
    load_k(0, kf[0]);
#pragma unroll
    for (int sub = 0; sub < NS; ++sub) {
      if (sub + 1 < NS) load_k(sub + 1, kf[(sub + 1) & 1]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < NR; ++n) s[sub][n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
        for (int n = 0; n < NR; ++n) s[sub][n] = TR::mfma16(kf[sub & 1][ks], qf[n][ks], s[sub][n]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    // ---- mask, online softmax (the scale rides in the exponent's fma; maxima are kept in
    //      scaled log2 units, which needs scale > 0 - the launcher guarantees it) ----------
    vec8 pf[NR][NS / 2];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      float mx = WIN ? -INFINITY : PF_NEG;
      if constexpr (MASKED) {
        const int qrow = wrow0 + n * 16 + c;
        const int limit = min(qrow, lkv - 1) - n0 - 4 * g;  // last attended (sub*16 + r)
#pragma unroll
        for (int sub = 0; sub < NS; ++sub)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            s[sub][n][r] = (sub * 16 + r <= limit) ? s[sub][n][r] : PF_NEG;
      }
#pragma unroll
      for (int sub = 0; sub < NS; ++sub)
#pragma unroll
        for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[sub][n][r]);
      mx = max_xor_16_32(mx);
      move_reference(n, mx * scale_log2e);
      float m_ref;
      const float factor = weight_factor(s, n, m_ref);
#pragma unroll
      for (int sub = 0; sub < NS; ++sub) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[sub][n][r], factor, -m_ref));
          pf[n][sub >> 1][(sub & 1) * 4 + r] = (T)p;
        }
      }
    }
#pragma unroll
    for (int k2 = 0; k2 < NS / 2; ++k2) pv_step(vt, k2, pf);
  };

  // WIN: a tile that some of the wave's rows see only in part.  Row groups of 16 keys that no row of
  // the wave sees are left out (a few sinks then cost a quarter of a tile).  Hidden scores become
  // -inf, which makes their weights 0 whatever the (finite) reference point is: a row's first tiles
  // may hide all their keys from it.
  auto compute_part = [&](int tile, int buf) {
    const int n0 = tile * BN;
    const char* kt = k_tile(buf);
    const char* vt = v_tile(buf);
    const int row_last = wrow0 + WROWS - 1;
    const int low = window > 0 ? wrow0 - window + 1 : 0;
    const int high = min(row_last, lkv - 1);
    bool on[NS];
#pragma unroll
    for (int sub = 0; sub < NS; ++sub) {
      const int k0 = n0 + sub * 16;
      on[sub] = k0 <= high && (k0 + 15 >= low || k0 < sinks);
    }
    f32x4 s[NS][NR];
#pragma unroll
    for (int sub = 0; sub < NS; ++sub) {
      if (on[sub]) {
        vec8 kf[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          kf[ks] = __builtin_bit_cast(
              vec8, *reinterpret_cast<const u32x4*>(kt + swz_off<D>(sub * 16 + c, 4 * ks + g)));
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          s[sub][n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) s[sub][n] = TR::mfma16(kf[ks], qf[n][ks], s[sub][n]);
        }
        const int k0 = n0 + sub * 16;
        // (a group that every row of the wave sees in full needs no mask: 1 to 2 % on long prompts.  With one row
        //  tile per wave the branch costs registers that spill: 4 % on 8 x 1024, window 256)
        if (NR == 1 || !(k0 + 15 <= min(wrow0, lkv - 1) && (window == 0 || k0 > row_last - window || k0 + 15 < sinks))) {
#pragma unroll
          for (int n = 0; n < NR; ++n) {
            const int qrow = wrow0 + n * 16 + c;
            const int last = min(qrow, lkv - 1) - k0 - 4 * g;
            const int first = (window > 0 ? qrow - window + 1 : 0) - k0 - 4 * g;
            const int sink = sinks - k0 - 4 * g;
#pragma unroll
            for (int r = 0; r < 4; ++r)
              s[sub][n][r] = (int)(r <= last) & ((int)(r >= first) | (int)(r < sink)) ? s[sub][n][r] : -INFINITY;
          }
        }
      } else {
#pragma unroll
        for (int n = 0; n < NR; ++n) s[sub][n] = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      }
    }
    vec8 pf[NR][NS / 2];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      float mx = -INFINITY;
#pragma unroll
      for (int sub = 0; sub < NS; ++sub)
        if (on[sub]) {
#pragma unroll
          for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[sub][n][r]);
        }
      move_reference(n, max_xor_16_32(mx) * scale_log2e);
      float m_ref;
      const float factor = weight_factor(s, n, m_ref);
#pragma unroll
      for (int sub = 0; sub < NS; ++sub)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          pf[n][sub >> 1][(sub & 1) * 4 + r] =
              on[sub] ? (T)__builtin_amdgcn_exp2f(__builtin_fmaf(s[sub][n][r], factor, -m_ref)) : (T)0.f;
    }
#pragma unroll
    for (int k2 = 0; k2 < NS / 2; ++k2)
      if (on[2 * k2] || on[2 * k2 + 1]) pv_step(vt, k2, pf);
  };

  // ---- main loop: tiles every wave attends in full first (no mask code), then the diagonal /
  //      ragged tiles.  Tile t+1 streams into the other LDS buffer while tile t is computed. -----
  auto run_tiles = [&](int t_begin, int t_end, auto masked_tag) {
    constexpr bool MASKED = decltype(masked_tag)::value;
    for (int tile = t_begin; tile < t_end; ++tile) {
      const int buf = tile & 1;
      if (tile + 1 < n_tiles) stage(tile + 1, buf ^ 1);
      // wave-uniform: skip a tile that is fully masked for all of this wave's rows
      if (!MASKED || tile * BN <= wrow0 + WROWS - 1) compute(tile, buf, masked_tag);
      stage_wait();
      __syncthreads();
    }
  };
  if constexpr (WIN) {
    const int count = ns + max(0, n_tiles - tw);
    auto tile_at = [&](int i) { return i < ns ? i : tw + i - ns; };
    if (count > 0) {
      // the first two tiles together: where the first holds a few sinks, its arithmetic would not cover
      // the way of the second
      stage(tile_at(0), 0);
      if (count > 1) stage(tile_at(1), 1);
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qf[n][ks]));
      stage_wait();
      __syncthreads();
      const int wrow1 = wrow0 + WROWS - 1;  // last row of the wave
      for (int i = 0; i < count; ++i) {
        const int tile = tile_at(i), buf = i & 1;
        if (i > 0 && i + 1 < count) stage(tile_at(i + 1), buf ^ 1);
        const int k0 = tile * BN, k1 = k0 + BN - 1;
        // wave-uniform: some row sees some key / every row sees every key
        const bool some = k0 <= wrow1 && (window == 0 || k1 > wrow0 - window || k0 < sinks);
        const bool all = k1 <= wrow0 && k1 < lkv && (window == 0 || k0 > wrow1 - window || k1 < sinks);
        if (all) compute(tile, buf, std::false_type{});
        else if (some) compute_part(tile, buf);
        stage_wait();
        __syncthreads();
      }
    }
  } else if (n_tiles > 0) {
    const int n_full = min(min(m0, lkv) / BN, n_tiles);
    stage(0, 0);
    // Retire the Q loads here: an empty asm that "rewrites" the fragments makes the compiler wait
    // for them before the loop instead of carrying them as pending into its wait-count
    // bookkeeping of every iteration.
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qf[n][ks]));
    stage_wait();
    __syncthreads();
    run_tiles(0, n_full, std::false_type{});
    run_tiles(n_full, n_tiles, std::true_type{});
  }

  // WIN: rows whose sum is finite and whose output is not.  The matrix instructions multiply hidden
  // values by a weight of 0, and 0 * inf (or NaN) is NaN: such a row is computed again from the keys
  // it sees, below.  (A NaN in a visible score makes the sum NaN, and the row's result with it.)
  uint32_t again = 0;
  if constexpr (WIN) {
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      float worst = 0.f;  // 0 * x is NaN for an infinity or a NaN
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 4; ++r) worst += 0.f * acc[dt][n][r];
      uint64_t b = __builtin_amdgcn_ballot_w64(worst != 0.f && 0.f * acc_l[n][0] == 0.f);
      b |= b >> 32;
      b |= b >> 16;
      again |= (uint32_t)(b & 0xffffu) << (16 * n);
    }
  }

  // ---- epilogue: normalise, stage the wave's WROWS x D tile in LDS, store whole rows ---------
  // The 16 lanes of a group write 8 bytes each to 16 different rows: 8-byte unit u of row r goes
  // to unit u ^ (r & 15) so that they cover the 128-byte bank window once.
  char* o_lds = smem + wave * (WROWS * D * 2);
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const float l = acc_l[n][0];  // every output row of the ones-MFMA holds the column's sum
    const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      typename TR::vec4 o4;
#pragma unroll
      for (int r = 0; r < 4; ++r) o4[r] = (T)(acc[dt][n][r] * inv);
      *reinterpret_cast<typename TR::vec4*>(o_lds + (n * 16 + c) * (D * 2) + (((4 * dt + g) ^ c) << 3)) = o4;
    }
  }
  __syncthreads();
  typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
#pragma unroll
  for (int i = 0; i < WROWS * CPR / 64; ++i) {
    const int idx = lane + i * 64;
    const int row = idx / CPR, ch = idx % CPR;
    const int qrow = wrow0 + row;
    const int x = row & 15;
    const u32x2 lo = *reinterpret_cast<const u32x2*>(o_lds + row * (D * 2) + (((2 * ch) ^ x) << 3));
    const u32x2 hi = *reinterpret_cast<const u32x2*>(o_lds + row * (D * 2) + (((2 * ch + 1) ^ x) << 3));
    if (qrow < lq && ch < hchunks && !(WIN && (again >> row & 1u))) {
      *reinterpret_cast<u32x4*>(out + (int64_t)(q0 + qrow) * out_stride + (int64_t)head * head_size + ch * 8) =
          u32x4{lo[0], lo[1], hi[0], hi[1]};
    }
  }
  if constexpr (WIN) {
    // rows to compute again: the wave walks the visible keys one by one, a lane holds elements
    // lane + 64 t of the head (never taken with finite values)
    while (again) {  // wave-uniform
      const int row = __builtin_ctz(again);
      again &= again - 1;
      const int qrow = wrow0 + row;
      if (qrow >= lq) continue;
      constexpr int E = D / 64;
      float qe[E], o[E], m = NEG, l = 0.f;
#pragma unroll
      for (int t = 0; t < E; ++t) {
        const int d = lane + 64 * t;
        qe[t] = d < head_size ? to_f32(q[(int64_t)(q0 + qrow) * q_stride + (int64_t)head * head_size + d]) : 0.f;
        o[t] = 0.f;
      }
      const int last = min(qrow, lkv - 1), first = window > 0 ? max(0, qrow - window + 1) : 0;
      for (int j = sinks > 0 ? 0 : first; j <= last; ++j) {
#pragma clang fp contract(off)
        if (j >= sinks && j < first) {
          j = first;
          if (j > last) break;
        }
        const T* kp = k + (int64_t)(kv0 + j) * k_stride + (int64_t)kvh * head_size;
        const T* vp = v + (int64_t)(kv0 + j) * v_stride + (int64_t)kvh * head_size;
        float dot = 0.f;
#pragma unroll
        for (int t = 0; t < E; ++t)
          if (lane + 64 * t < head_size) dot += qe[t] * to_f32(kp[lane + 64 * t]);
        const float x = wave_sum(dot) * scale_log2e;
        const float m_new = fmaxf(m, x), f = __builtin_amdgcn_exp2f(m - m_new), p = __builtin_amdgcn_exp2f(x - m_new);
        m = m_new;
        l = l * f + p;
#pragma unroll
        for (int t = 0; t < E; ++t)
          if (lane + 64 * t < head_size) o[t] = o[t] * f + p * to_f32(vp[lane + 64 * t]);
      }
#pragma unroll
      for (int t = 0; t < E; ++t)
        if (lane + 64 * t < head_size)
          out[(int64_t)(q0 + qrow) * out_stride + (int64_t)head * head_size + lane + 64 * t] =
              from_f32<T>(l > 0.f ? o[t] / l : 0.f);
    }
  }
}

}  // namespace pe
