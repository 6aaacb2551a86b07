// igl_attend4.h - attention over the 4-bit key/value ring (igl_cache4.h) with a
// sliding window and first positions that stay visible, gfx950.
//
// For the query heads q of a lane at position p and the key/value head they
// share, over the visible positions t (t <= p and, with a window, t > p - window
// or t < sinks):
//     o = sum_t 2^(f q . k_t - m) v_t / sum_t 2^(f q . k_t - m),
// f the score scale, the key scale and log2 e, m a base near the peak.
#pragma once

#include "igl_cache4.h"

namespace igl {

struct Attend4Args {
  const uint8_t *key_code, *key_gain, *value_code, *value_gain;
  long long room;        // slots a gain row holds
  int span, sinks;
  int kv_width;          // values a row
  int share;             // query heads a key/value head
  const float *query;
  float *out;
  long long lane_stride;
  int place;             // of lane 0
  int newest;            // place of the last lane
  int newest_slot;       // and its slot, where it lies past the sinks
  int window;
  int rows;              // lanes * share
  int key_power;         // key scale, score scale, log2 e and 256: key_part 2^key_power
  float key_part;        // in [1/2, 1), or of a score scale below zero
  float value_scale;     // times 256
  int segments;          // of a row tile's blocks
  float *part_out;       // [segments][kv][rows][HEAD], with more than one segment
  float *part_base;      // [segments][kv][rows]
  float *part_total;
};

// The blocks of `block` slots that hold what lanes at positions first ..
// last see: blocks 0 .. low - 1, then mid .. mid + count - low - 1.  The visible
// slots are the sinks' and the ring's from the oldest position to the newest,
// cut in two where the ring wraps; the piece from slot sinks on joins the sinks.
struct Blocks4 {
  int low, mid, count;
  __host__ __device__ int at(int i) const { return i < low ? i : mid + i - low; }
};

__host__ __device__ __forceinline__ Blocks4 attend4_blocks(int block, int span, int sinks, int window, int first,
                                                               int last) {
  Blocks4 b = {0, 0, 0};
  const int kept = last < sinks ? last + 1 : sinks;
  int oldest = window > 0 && first >= window ? first + 1 - window : 0;
  if (oldest < sinks) oldest = sinks;
  int low_slots = kept, mid_first = 0, mid_last = -1;
  if (oldest <= last) {
    mid_first = cache4_slot(oldest, sinks, span);
    mid_last = cache4_slot(last, sinks, span);
    if (mid_first > mid_last) {
      low_slots = mid_last + 1;
      mid_last = span - 1;
    }
  }
  b.low = (low_slots + block - 1) / block;
  b.mid = mid_first / block;
  if (b.mid < b.low) b.mid = b.low;
  const int end = mid_last < 0 ? 0 : mid_last / block + 1;
  b.count = b.low + (end > b.mid ? end - b.mid : 0);
  return b;
}


// Segments a row's blocks are cut into, at most: the fold takes one a thread.
constexpr int kAttend4Segments = 256;

// The position whose row a slot holds once `newest` is laid; INT_MAX: none.
__device__ __forceinline__ int attend4_place(int slot, const Attend4Args &a) {
  int back = a.newest_slot - slot;
  if (back < 0) back += a.span - a.sinks;
  int place = a.newest - back;
  if (a.newest_slot < 0 || place < a.sinks) place = 0x7FFFFFFF;
  if (slot < a.sinks) place = slot;
  return slot < a.span ? place : 0x7FFFFFFF;
}

// ---- operands ---------------------------------------------------------------

// Two gain bytes at bits [0,8) and [16,24) as binary16 values of real8 / 256.
__device__ __forceinline__ half2_t gain_pair(uint32_t x) { return as_half2((x + (x & 0x00800080u)) << 7); }

__device__ __forceinline__ half2_t half_low(half2_t x) { return __builtin_shufflevector(x, x, 0, 0); }
__device__ __forceinline__ half2_t half_high(half2_t x) { return __builtin_shufflevector(x, x, 1, 1); }

// What turns 16 + c into (c - 8) g with one fma: -24 g, exact (g has four
// significant bits).  E2M1 codes are levels as they are decoded.
__device__ __forceinline__ half2_t gain_offset(half2_t g) { return g * half2_t{(_Float16)-24.0f, (_Float16)-24.0f}; }

// Element e of a key operand of eight dims is dim key_order<FMT>(e) of them: a
// dword's nibbles i and i + 4 lie 16 bits apart, the halves of one register; a
// byte's two are converted together.
template <int FMT>
__host__ __device__ constexpr int key_order(int e) {
  return FMT == IGL_CACHE4_INT4 ? (e >> 1) + 4 * (e & 1) : e;
}

// Eight codes of one row, times their gain (both halves of g; h its offset).
template <int FMT>
__device__ __forceinline__ half8_t key_operand(uint32_t w, half2_t g, half2_t h, uint32_t exp16) {
  half2_t p[4];
  if (FMT == IGL_CACHE4_INT4) {
    p[0] = __builtin_elementwise_fma(nibble_pair16<0>(w, exp16), g, h);
    p[1] = __builtin_elementwise_fma(nibble_pair16<1>(w, exp16), g, h);
    p[2] = __builtin_elementwise_fma(nibble_pair16<2>(w, exp16), g, h);
    p[3] = __builtin_elementwise_fma(nibble_pair16<3>(w, exp16), g, h);
  } else {
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 0) * g;
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 1) * g;
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 2) * g;
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 3) * g;
  }
  return __builtin_bit_cast(half8_t, p);
}

// Eight rows of DIMS (4 or 8) codes each, low nibble first, as DIMS operands of
// one dim and the eight rows, times the rows' gains (pairs of rows; h their
// offsets).
template <int FMT, int DIMS>
__device__ __forceinline__ void value_operands(const uint32_t (&x)[8], const half2_t (&g)[4], const half2_t (&h)[4],
                                               uint32_t exp16, half8_t (&out)[DIMS]) {
  half2_t p[DIMS][4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const uint32_t a = x[2 * q], b = x[2 * q + 1];
    if (FMT == IGL_CACHE4_INT4) {
#pragma unroll
      for (int half = 0; half < DIMS / 4; ++half) {
        const uint32_t t = __builtin_amdgcn_perm(b, a, half ? 0x07060302u : 0x05040100u);
        p[4 * half + 0][q] = __builtin_elementwise_fma(nibble_pair16<0>(t, exp16), g[q], h[q]);
        p[4 * half + 1][q] = __builtin_elementwise_fma(nibble_pair16<1>(t, exp16), g[q], h[q]);
        p[4 * half + 2][q] = __builtin_elementwise_fma(nibble_pair16<2>(t, exp16), g[q], h[q]);
        p[4 * half + 3][q] = __builtin_elementwise_fma(nibble_pair16<3>(t, exp16), g[q], h[q]);
      }
    } else {
      // bytes of both rows' nibbles: of the even dims, and of the odd ones
      const uint32_t even = (a & 0x0F0F0F0Fu) | ((b << 4) & 0xF0F0F0F0u);
      const uint32_t odd = ((a >> 4) & 0x0F0F0F0Fu) | (b & 0xF0F0F0F0u);
      p[0][q] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(even, 1.0f, 0) * g[q];
      p[1][q] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(odd, 1.0f, 0) * g[q];
      p[2][q] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(even, 1.0f, 1) * g[q];
      p[3][q] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(odd, 1.0f, 1) * g[q];
      if (DIMS == 8) {
        p[DIMS - 4][q] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(even, 1.0f, 2) * g[q];
        p[DIMS - 3][q] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(odd, 1.0f, 2) * g[q];
        p[DIMS - 2][q] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(even, 1.0f, 3) * g[q];
        p[DIMS - 1][q] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(odd, 1.0f, 3) * g[q];
      }
    }
  }
#pragma unroll
  for (int d = 0; d < DIMS; ++d) out[d] = __builtin_bit_cast(half8_t, p[d]);
}

// Largest and sum over the four lanes of a wave that differ by 16 and 32, the
// same in all four: each swap of two copies leaves the partners' values side by
// side (written out as xsum32 is).
__device__ __forceinline__ float xmax48(float v) {
  float a = v, b = v;
  asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
  a = b = fmaxf(a, b);
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
  return fmaxf(a, b);
}

__device__ __forceinline__ float xsum48(float v) {
  float a = v, b = v;
  asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
  a = b = a + b;
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
  return a + b;
}

// ---- the kernel ---------------------------------------------------------------

// Work.  A wave takes a tile of rows (a row is a lane's query head of one
// key/value head) through blocks of 32 U slots, everything in registers:
//   scores  S^T (slots x rows)  = K (slots x dims) . Q^T
//   blend   O^T (dims x rows)   = V^T (dims x slots) . P^T
// Transposed, a score's lane and register are where the blend's product wants
// its probability: lane 16 g + n of S^T holds row n's slots 4 g + r of a
// 16-slot tile, and of P^T row n's eight slots 8 g + e.  With slot 32 u + 8 g +
// 2 r + b as index 4 g + r of tile 2 u + b, e is 2 r + b, and nothing crosses
// lanes between the two products but a row's peak.  Keys are read as they lie,
// 16 bytes of a row (one gain's dims) a lane; values eight rows a lane, whose
// nibbles pair up by twos of rows.
//
// Rows keep 24 bits: queries (scaled by a power of two to their row's largest)
// and probabilities are two binary16 terms.  A tile of up to eight rows (PAIR)
// holds both terms in the 16 columns of one product; others take two products.
// DW waves split a head's dims (the partial scores meet in LDS), PS waves a
// segment's blocks (their blends meet in LDS at the end).
//
// A row's base m is a whole number, so every rescaling is exact; weights are
// 2^(score - m).  It moves, to 12 below the block's peak, when the peak is not 8
// to 14 above it: most blocks rescale nothing, a block's largest weight is in
// [2^8, 2^15), and weights down to 2^-32 of it keep a term of binary16 (against a
// base at the peak they end at 2^-24: one position that outweighs a block's
// others by that much, its own value small, would take them from the blend).
// The base stays within 58 of the largest so far, below which weights count for
// nothing: sums stay in range.
template <int HEAD, int FMT, int RB, bool PAIR, int DW, int PS, int U>
struct Attend4Shape {
  static constexpr int DH = HEAD / DW;            // dims a wave holds
  static constexpr int KL = DH >= 128 ? DH / 128 : 1;  // key chunks of a row a lane reads
  static constexpr int KW = DH >= 128 ? 4 : 2;    // dwords of a chunk
  static constexpr int DPL = DH / 16;             // value dims a lane
  static constexpr int ROWS = PAIR ? 8 : 16 * RB;
  static constexpr int TERMS = PAIR ? 1 : 2;      // products a term pair takes
  static constexpr int BLOCK = 32 * U;
  static constexpr int TREE = PS > 1 ? PS / 2 * DW * (DPL * RB * 1024 + RB * 512) : 0;
  static constexpr int SWAP = DW > 1 ? 2 * PS * DW * 2 * U * RB * 1024 : 0;
  static constexpr int LDS = TREE > SWAP ? TREE : SWAP;
};

template <int HEAD, int FMT, int RB, bool PAIR, int DW, int PS, int U>
__global__ __launch_bounds__(64 * DW * PS) void attend4_kernel(Attend4Args a) {
  using F = Attend4Shape<HEAD, FMT, RB, PAIR, DW, PS, U>;
  constexpr int DH = F::DH, KL = F::KL, KW = F::KW, DPL = F::DPL, ROWS = F::ROWS, TERMS = F::TERMS, BLOCK = F::BLOCK;
  constexpr int VD = DPL >= 8 ? 8 : 4;   // dims a value step takes
  constexpr int VW = DPL >= 8 ? DPL / 8 : 1;  // dwords of a value row a lane reads
  extern __shared__ __attribute__((aligned(16))) uint8_t lds4[];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int dw = DW > 1 ? wave % DW : 0, ps = wave / DW;
  const int g = lane >> 4, n = lane & 15;
  const int kv = blockIdx.z, seg = blockIdx.y;
  const int row0 = (int)(gridDim.x - 1 - blockIdx.x) * ROWS;  // a prompt's longest first
  const int row_last = min(row0 + ROWS, a.rows) - 1;
  const int place_low = a.place + row0 / a.share, place_high = a.place + row_last / a.share;
  const Blocks4 blocks = attend4_blocks(BLOCK, a.span, a.sinks, a.window, place_low, place_high);
  const int per = (blocks.count + a.segments - 1) / a.segments;
  const int first = seg * per + ps, end = min(blocks.count, seg * per + per);
  const uint32_t exp16 = 0x4C004C00u;
  const uint32_t row_bytes = (uint32_t)a.kv_width / 2;
  const size_t head_bytes = ((size_t)kv * HEAD + dw * DH) / 2;
  const size_t gain_row = ((size_t)kv * HEAD + dw * DH) / kCache4Group;

  // ---- the rows' queries, this wave's dims
  half8_t q[RB][TERMS][KL * KW];
  float factor[RB];
  int place[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int row = min(row0 + 16 * rb + (PAIR ? n & 7 : n), row_last);
    const int l = row / a.share;
    place[rb] = a.place + l;
    const float *src = a.query + (size_t)l * a.lane_stride + ((size_t)kv * a.share + (row - l * a.share)) * HEAD + dw * DH;
    const bool vec = (((uintptr_t)a.query | ((size_t)a.lane_stride * 4)) & 15u) == 0;  // uniform
    float x[KL * KW][8];
#pragma unroll
    for (int c = 0; c < KL; ++c)
#pragma unroll
      for (int s = 0; s < KW; ++s) {
        const float *p = src + (KW == 4 ? 32 * (4 * c + g) : 16 * g) + 8 * s;
        if (vec) {
          const float4_t u = *reinterpret_cast<const float4_t *>(p), v = *reinterpret_cast<const float4_t *>(p + 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[KW * c + s][e] = u[e], x[KW * c + s][4 + e] = v[e];
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[KW * c + s][e] = p[e];
        }
      }
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < KL * KW; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[i][e]));
    top = xmax48(top);
    // to [2^13, 2^14); an infinity or NaN stays one in its terms
    const int up = top > 0.0f && top < INFINITY ? 14 - __builtin_amdgcn_frexp_expf(top) : 0;
    const float sign = a.key_part < 0.0f ? -1.0f : 1.0f;  // a factor below zero turns the queries
    factor[rb] = __builtin_amdgcn_ldexpf(fabsf(a.key_part), a.key_power - up);
#pragma unroll
    for (int i = 0; i < KL * KW; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = __builtin_amdgcn_ldexpf(x[i][key_order<FMT>(e)] * sign, up);
        const _Float16 hi = (_Float16)v, lo = (_Float16)(v - (float)hi);
        if (PAIR) {
          q[rb][0][i][e] = n >= 8 ? lo : hi;
        } else {
          q[rb][0][i][e] = hi;
          q[rb][TERMS - 1][i][e] = lo;
        }
      }
  }

  // ---- what a block's rows are read into
  uint32_t kr[2 * U][KL][KW];
  uint32_t kg[U][KL];
  uint32_t vr[U][8][VW];
  uint2_t vg[U];
  const uint32_t k_lane = (uint32_t)(2 * n) * row_bytes + (KW == 4 ? 16 : 8) * g;
  const uint32_t v_lane = (uint32_t)(8 * g) * row_bytes + (uint32_t)(n * DPL / 2);
  const size_t k_gain_lane = (size_t)(KW == 4 ? g : g / 2) * a.room + 2 * n;
  const size_t v_gain_lane = (size_t)(n * DPL / kCache4Group) * a.room + 8 * g;
  auto rows_at = [&](const uint8_t *codes, int slot0) {
    return uniform_rows(codes + (size_t)slot0 * row_bytes + head_bytes);
  };
  auto load_keys = [&](int i) {
    const int slot0 = blocks.at(i) * BLOCK;
    const auto src = rows_at(a.key_code, slot0);
    const bool whole = slot0 + BLOCK <= a.span;
#pragma unroll
    for (int t = 0; t < 2 * U; ++t) {
      // slot 32 u + 2 n + b; past the ring's end its last row, which no row sees there
      const int at = 32 * (t >> 1) + (t & 1);
      const uint32_t off = whole ? k_lane
                                 : (uint32_t)min(at + 2 * n, a.span - 1 - slot0) * row_bytes + (KW == 4 ? 16 : 8) * g;
      const uint32_t base = whole ? (uint32_t)at * row_bytes : 0u;
#pragma unroll
      for (int c = 0; c < KL; ++c) {
        if constexpr (KW == 4) {
          const uint4_t w = __builtin_amdgcn_raw_buffer_load_b128(src, off + 64 * c, base, 0);
#pragma unroll
          for (int s = 0; s < 4; ++s) kr[t][c][s] = w[s];
        } else {
          const uint2_t w = __builtin_amdgcn_raw_buffer_load_b64(src, off, base, 0);
          kr[t][c][0] = w[0];
          kr[t][c][1] = w[1];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int c = 0; c < KL; ++c)
        kg[u][c] = *reinterpret_cast<const uint16_t *>(a.key_gain + (gain_row + 4 * c) * a.room + slot0 + 32 * u + k_gain_lane);
  };
  auto load_values = [&](int i) {
    const int slot0 = blocks.at(i) * BLOCK;
    const auto src = rows_at(a.value_code, slot0);
    const bool whole = slot0 + BLOCK <= a.span;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int at = 32 * u + e;
        const uint32_t off = whole ? v_lane
                                   : (uint32_t)min(at + 8 * g, a.span - 1 - slot0) * row_bytes + (uint32_t)(n * DPL / 2);
        const uint32_t base = whole ? (uint32_t)at * row_bytes : 0u;
        if constexpr (DPL == 4) {
          vr[u][e][0] = __builtin_amdgcn_raw_buffer_load_b16(src, off, base, 0);
        } else if constexpr (DPL == 8) {
          vr[u][e][0] = __builtin_amdgcn_raw_buffer_load_b32(src, off, base, 0);
        } else if constexpr (DPL == 16) {
          const uint2_t w = __builtin_amdgcn_raw_buffer_load_b64(src, off, base, 0);
          vr[u][e][0] = w[0];
          vr[u][e][VW - 1] = w[1];
        } else {
          const uint4_t w = __builtin_amdgcn_raw_buffer_load_b128(src, off, base, 0);
#pragma unroll
          for (int s = 0; s < VW; ++s) vr[u][e][s] = w[s];
        }
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
      vg[u] = *reinterpret_cast<const uint2_t *>(a.value_gain + gain_row * a.room + slot0 + 32 * u + v_gain_lane);
  };

  float4_t out[RB][DPL];
  float base[RB], top_base[RB], total[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    base[rb] = top_base[rb] = -INFINITY;
    total[rb] = 0.0f;
#pragma unroll
    for (int j = 0; j < DPL; ++j) out[rb][j] = float4_t{0, 0, 0, 0};
  }
  // waves that split dims walk the same blocks: they meet at each one's scores
  if (first < end) {
    load_keys(first);
    load_values(first);
  }
  int turn = 0;
  const int steps = DW > 1 && PS > 1 ? (end - (first - ps) + PS - 1) / PS : 0;  // of the workgroup's slowest wave
  for (int i = first, step = 0; DW > 1 && PS > 1 ? step < steps : i < end; i += PS, ++step) {
    const bool live = !(DW > 1 && PS > 1) || i < end;  // uniform; a wave past its blocks only meets the others
    float4_t s[RB][2 * U];
    if (live) {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int t = 0; t < 2 * U; ++t) s[rb][t] = float4_t{0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < KL; ++c)
#pragma unroll
        for (int t = 0; t < 2 * U; ++t) {
          const uint32_t two = kg[t >> 1][c];
          const half2_t pair = gain_pair((two & 0xFFu) | ((two & 0xFF00u) << 8));
          const half2_t gain = t & 1 ? half_high(pair) : half_low(pair), off = gain_offset(gain);
#pragma unroll
          for (int w = 0; w < KW; ++w) {
            const half8_t k = key_operand<FMT>(kr[t][c][w], gain, off, exp16);
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
#pragma unroll
              for (int m = TERMS - 1; m >= 0; --m)
                s[rb][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q[rb][m][KW * c + w], s[rb][t], 0, 0, 0);
          }
        }
      if (i + PS < end) load_keys(i + PS);
    }
    if constexpr (DW > 1) {
      // the waves' partial scores, each in its own factor, summed in wave order
      float4_t *room = reinterpret_cast<float4_t *>(lds4) + (size_t)turn * (PS * DW * 2 * U * RB * 64);
      if (live) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
          for (int t = 0; t < 2 * U; ++t) {
#pragma unroll
            for (int r = 0; r < 4; ++r) s[rb][t][r] *= factor[rb];
            room[((wave * RB + rb) * 2 * U + t) * 64 + lane] = s[rb][t];
          }
      }
      lds_barrier();
      if (live) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
          for (int t = 0; t < 2 * U; ++t) {
            float4_t sum = room[(((ps * DW) * RB + rb) * 2 * U + t) * 64 + lane];
#pragma unroll
            for (int w = 1; w < DW; ++w) sum += room[(((ps * DW + w) * RB + rb) * 2 * U + t) * 64 + lane];
            s[rb][t] = sum;
          }
      }
      turn ^= 1;
    }
    if (!live) continue;

    // ---- the rows' peaks and weights
    const int slot0 = blocks.at(i) * BLOCK;
    const int place0 = attend4_place(slot0, a);
    const bool all = slot0 >= a.sinks && slot0 + BLOCK <= a.span && place0 <= place_low - (BLOCK - 1) &&
                     attend4_place(slot0 + BLOCK - 1, a) == place0 + BLOCK - 1 &&
                     (a.window == 0 || place0 > place_high - a.window);  // uniform: every row sees every slot
    half8_t p[RB][TERMS][U];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const float f = DW > 1 ? 1.0f : factor[rb];
      if (PAIR) {
#pragma unroll
        for (int t = 0; t < 2 * U; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[rb][t][r] += dpp_move<0x128>(s[rb][t][r]);  // row n and n + 8
      }
      uint32_t seen = 0xFFFFFFFFu;
      if (!all) {
        seen = 0;
#pragma unroll
        for (int t = 0; t < 2 * U; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int at = attend4_place(slot0 + 32 * (t >> 1) + 8 * g + 2 * r + (t & 1), a);
            if (at <= place[rb] && (a.window == 0 || at > place[rb] - a.window || at < a.sinks)) seen |= 1u << (4 * t + r);
          }
      }
      float peak = -INFINITY;
#pragma unroll
      for (int t = 0; t < 2 * U; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (all)
            peak = fmaxf(peak, s[rb][t][r]);
          else
            peak = fmaxf(peak, seen >> (4 * t + r) & 1u ? s[rb][t][r] : -INFINITY);
      peak = xmax48(peak);
      if (peak != -INFINITY) peak *= f;
      const float low = floorf(peak);
      float m = base[rb];
      if (low != -INFINITY && !(low >= m + 8.0f && low <= m + 14.0f)) {
        top_base[rb] = fmaxf(top_base[rb], low - 12.0f);
        m = fmaxf(low - 12.0f, top_base[rb] - 58.0f);
      }
      if (__builtin_amdgcn_ballot_w64(m != base[rb])) {
        const float keep = base[rb] != -INFINITY ? __builtin_amdgcn_exp2f(base[rb] - m) : 0.0f;
        total[rb] *= keep;
#pragma unroll
        for (int j = 0; j < DPL; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) out[rb][j][r] *= keep;
        base[rb] = m;
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          half2_t hi, lo;
          float w[2];
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const int t = 2 * u + b;
            w[b] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rb][t][r], f, -m));
            if (!all) w[b] = seen >> (4 * t + r) & 1u ? w[b] : 0.0f;
            total[rb] += w[b];
            hi[b] = (_Float16)w[b];
            lo[b] = (_Float16)(w[b] - (float)hi[b]);
          }
          if (PAIR) {
            const half2_t mine = n >= 8 ? lo : hi;
            p[rb][0][u][2 * r] = mine[0];
            p[rb][0][u][2 * r + 1] = mine[1];
          } else {
            p[rb][0][u][2 * r] = hi[0];
            p[rb][0][u][2 * r + 1] = hi[1];
            p[rb][TERMS - 1][u][2 * r] = lo[0];
            p[rb][TERMS - 1][u][2 * r + 1] = lo[1];
          }
        }
    }

    // ---- the blend
#pragma unroll
    for (int u = 0; u < U; ++u) {
      half2_t gain[4], off[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        gain[k] = gain_pair(__builtin_amdgcn_perm(0u, vg[u][k >> 1], k & 1 ? 0x0C030C02u : 0x0C010C00u));
        off[k] = gain_offset(gain[k]);
      }
#pragma unroll
      for (int v = 0; v < VW; ++v) {
        uint32_t x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = vr[u][e][v];
        half8_t op[VD];
        value_operands<FMT, VD>(x, gain, off, exp16, op);
#pragma unroll
        for (int d = 0; d < VD; ++d)
#pragma unroll
          for (int rb = 0; rb < RB; ++rb)
#pragma unroll
            for (int t = TERMS - 1; t >= 0; --t)
              out[rb][VD * v + d] =
                  __builtin_amdgcn_mfma_f32_16x16x32_f16(op[d], p[rb][t][u], out[rb][VD * v + d], 0, 0, 0);
      }
    }
    if (i + PS < end) load_values(i + PS);
  }
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) total[rb] = xsum48(total[rb]);

  // ---- waves that took different blocks: halves of them fold into the others
  if constexpr (PS > 1) {
    constexpr int SIZE = DPL * RB * 64 + RB * 32;  // float4 of a wave's blend, then its bases and totals
#pragma unroll
    for (int half = PS / 2; half > 0; half >>= 1) {
      __syncthreads();
      float4_t *room = reinterpret_cast<float4_t *>(lds4) + (size_t)((ps % half) * DW + dw) * SIZE;
      float *stats = reinterpret_cast<float *>(room + DPL * RB * 64);
      if (ps >= half && ps < 2 * half) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
#pragma unroll
          for (int j = 0; j < DPL; ++j) room[(rb * DPL + j) * 64 + lane] = out[rb][j];
          stats[128 * rb + lane] = base[rb];
          stats[128 * rb + 64 + lane] = total[rb];
        }
      }
      __syncthreads();
      if (ps < half) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
          const float theirs = stats[128 * rb + lane];
          const float m = fmaxf(base[rb], theirs);
          const float mine = base[rb] != -INFINITY ? __builtin_amdgcn_exp2f(base[rb] - m) : 0.0f;
          const float part = theirs != -INFINITY ? __builtin_amdgcn_exp2f(theirs - m) : 0.0f;
          base[rb] = m;
          total[rb] = total[rb] * mine + stats[128 * rb + 64 + lane] * part;
#pragma unroll
          for (int j = 0; j < DPL; ++j) {
            const float4_t o = room[(rb * DPL + j) * 64 + lane];
#pragma unroll
            for (int r = 0; r < 4; ++r) out[rb][j][r] = out[rb][j][r] * mine + o[r] * part;
          }
        }
      }
    }
    if (ps > 0) return;
  }

  // ---- the rows' blends, or this segment's share of them: dims (4 g + r) DPL + j
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    if (PAIR) {
#pragma unroll
      for (int j = 0; j < DPL; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) out[rb][j][r] += dpp_move<0x128>(out[rb][j][r]);
    }
    const int row = row0 + 16 * rb + (PAIR ? n & 7 : n);
    if (row > row_last) continue;
    const bool split = a.segments > 1;
    const int l = row / a.share;
    float *dst = a.out + (size_t)l * a.lane_stride + ((size_t)kv * a.share + (row - l * a.share)) * HEAD;
    float mul = a.value_scale;
    bool vec = (((uintptr_t)a.out | ((size_t)a.lane_stride * 4)) & 15u) == 0;
    if (split) {
      const size_t at = ((size_t)seg * gridDim.z + kv) * a.rows + row;
      dst = a.part_out + at * HEAD;
      vec = true;
      if (g == 0 && dw == 0 && (!PAIR || n < 8)) {
        a.part_base[at] = base[rb];
        a.part_total[at] = total[rb];
      }
    } else {
      mul *= 1.0f / total[rb];
    }
    dst += dw * DH;
    // PAIR: both halves of the columns hold the sums; each writes half of them
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (PAIR && (r >= 2) != (n >= 8)) continue;
#pragma unroll
      for (int j = 0; j < DPL; j += 4) {
        float *to = dst + (4 * g + r) * DPL + j;
        const float4_t o = {out[rb][j][r] * mul, out[rb][j + 1][r] * mul, out[rb][j + 2][r] * mul, out[rb][j + 3][r] * mul};
        if (vec) {
          *reinterpret_cast<float4_t *>(to) = o;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) to[e] = o[e];
        }
      }
    }
  }
}

// Folds the segments of a row: a workgroup a row and DIMS of its dims, thread
// (c, s) of four dims c and the segments s, s + SL, ...  Every segment's base
// and total go through LDS as its weight and weighted total.
template <int DIMS>
__global__ __launch_bounds__(256) void attend4_fold_kernel(Attend4Args a, int head_size) {
  constexpr int COLS = DIMS / 4, SL = 256 / COLS;
  __shared__ float weight[kAttend4Segments];
  __shared__ float share[kAttend4Segments];
  __shared__ float4_t part[SL][COLS];
  const int tid = threadIdx.x, c = tid % COLS, sl = tid / COLS;
  const int row = blockIdx.x, kv = blockIdx.y, kv_count = gridDim.y;
  const size_t step = (size_t)kv_count * a.rows, at = (size_t)kv * a.rows + row;
  const int d0 = blockIdx.z * DIMS + 4 * c;
  constexpr int AHEAD = 4;
  float4_t first[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) {
    const int s = min(sl + i * SL, a.segments - 1);
    first[i] = *reinterpret_cast<const float4_t *>(a.part_out + (at + s * step) * head_size + d0);
  }
  // base of segment tid (there are no more than 256)
  const float mine = tid < a.segments ? a.part_base[at + tid * step] : -INFINITY;
  const float sum = tid < a.segments ? a.part_total[at + tid * step] : 0.0f;
  share[tid] = mine;
  __syncthreads();
  float m = -INFINITY;
  for (int s = 0; s < a.segments; ++s) m = fmaxf(m, share[s]);
  const float w = mine != -INFINITY ? __builtin_amdgcn_exp2f(mine - m) : 0.0f;
  __syncthreads();
  weight[tid] = w;
  share[tid] = w * sum;
  __syncthreads();
  float4_t acc = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) {
    const int s = sl + i * SL;
    if (s < a.segments) acc += first[i] * weight[s];
  }
  for (int s = sl + AHEAD * SL; s < a.segments; s += SL)
    acc += *reinterpret_cast<const float4_t *>(a.part_out + (at + s * step) * head_size + d0) * weight[s];
  part[sl][c] = acc;
  __syncthreads();
  if (sl) return;
  float total = 0.0f;
  for (int s = 0; s < a.segments; ++s) total += share[s];
  for (int s = 1; s < SL; ++s) acc += part[s][c];
  const int l = row / a.share;
  float *to = a.out + (size_t)l * a.lane_stride + ((size_t)kv * a.share + (row - l * a.share)) * head_size + d0;
  const float mul = 1.0f / total;
#pragma unroll
  for (int e = 0; e < 4; ++e) to[e] = acc[e] * mul;
}

}  // namespace igl

using namespace igl;

// Which form a launch takes.
struct Attend4Plan {
  int pair, rb, dw, ps;  // attend4_kernel's
  int tiles, segments;
};

static Attend4Plan attend4_plan(int head, int span, int sinks, int kv_count, int share, int place, int window, int lanes) {
  Attend4Plan p = {0, 1, 1, 4, 1, 1};
  const long long rows = (long long)lanes * share;
  const long long tiles32 = (rows + 31) / 32;
  if (rows <= 8) {
    p.pair = 1;
  } else if (tiles32 * kv_count >= 256) {
    p.rb = 2;
    p.ps = 1;
    p.dw = head == 512 ? 2 : 1;
  } else if (head == 512) {
    p.dw = 2;
    p.ps = 2;
  }
  const int each = p.pair ? 8 : 16 * p.rb;
  p.tiles = (int)((rows + each - 1) / each);
  // a tile's blocks, the last one's
  const int first = place + (int)(((long long)(p.tiles - 1) * each) / share), last = place + lanes - 1;
  const int blocks = attend4_blocks(64, span, sinks, window, first, last).count;
  long long s = p.ps == 1 ? 1 : 256 / ((long long)p.tiles * kv_count);
  const long long room = (long long)IGL_ATTEND_FIXED_FLOATS / (rows * kv_count * (head + 2));
  if (s > (blocks + p.ps - 1) / p.ps) s = (blocks + p.ps - 1) / p.ps;
  if (s > room) s = room;
  if (s > kAttend4Segments) s = kAttend4Segments;
  if (s < 1) s = 1;
  p.segments = (int)s;
  return p;
}

template <int HEAD, int FMT, int RB, bool PAIR, int DW, int PS, int U>
static hipError_t attend4_launch(const Attend4Args &a, const Attend4Plan &p, int kv_count, hipStream_t stream) {
  constexpr int size = Attend4Shape<HEAD, FMT, RB, PAIR, DW, PS, U>::LDS;
  const void *kernel = reinterpret_cast<const void *>(&attend4_kernel<HEAD, FMT, RB, PAIR, DW, PS, U>);
  if (size > 65536) {  // granted once a device; granting again changes nothing
    const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, size);
    if (e != hipSuccess) return e;
  }
  const dim3 grid(p.tiles, p.segments, kv_count);
  hipLaunchKernelGGL((attend4_kernel<HEAD, FMT, RB, PAIR, DW, PS, U>), grid, dim3(64 * DW * PS), (size_t)size, stream, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.segments == 1) return e;
  const int dims = a.rows <= 64 ? 16 : 64;
  const dim3 fgrid(a.rows, kv_count, HEAD / dims);
  if (dims == 16)
    hipLaunchKernelGGL((attend4_fold_kernel<16>), fgrid, dim3(256), 0, stream, a, HEAD);
  else
    hipLaunchKernelGGL((attend4_fold_kernel<64>), fgrid, dim3(256), 0, stream, a, HEAD);
  return hipGetLastError();
}

template <int HEAD, int FMT>
static hipError_t attend4_launch_head(const Attend4Args &a, const Attend4Plan &p, int kv_count, hipStream_t stream) {
  constexpr int DW = HEAD == 512 ? 2 : 1;
  if (p.pair) return attend4_launch<HEAD, FMT, 1, true, 1, 4, 2>(a, p, kv_count, stream);
  if (p.rb == 2) return attend4_launch<HEAD, FMT, 2, false, DW, 1, 2>(a, p, kv_count, stream);
  return attend4_launch<HEAD, FMT, 1, false, DW, 4 / DW, 2>(a, p, kv_count, stream);
}

template <int HEAD>
static hipError_t attend4_launch_format(const Attend4Args &a, const Attend4Plan &p, int format, int kv_count,
                                        hipStream_t stream) {
  if (format == IGL_CACHE4_INT4) return attend4_launch_head<HEAD, IGL_CACHE4_INT4>(a, p, kv_count, stream);
  return attend4_launch_head<HEAD, IGL_CACHE4_E2M1>(a, p, kv_count, stream);
}

extern "C" hipError_t igl_launch_attend4(const igl_cache4 *store, int group_share, const float *query, int lane_stride,
                                         int place_first, int window, int lanes, float score_scale, float *blend_out,
                                         float *work, hipStream_t stream) {
  Attend4Args a = {};
  const long long rows = (long long)lanes * group_share;
  if (rows > 0x7FFFFFFF - 64) return hipErrorInvalidValue;
  const Attend4Plan p = attend4_plan(store->head_size, store->cache_span, store->sink_count, store->kv_count, group_share,
                                     place_first, window, lanes);
  a.key_code = store->key_code;
  a.key_gain = store->key_gain;
  a.value_code = store->value_code;
  a.value_gain = store->value_gain;
  a.room = (long long)igl_cache4_room(store->cache_span);
  a.span = store->cache_span;
  a.sinks = store->sink_count;
  a.kv_width = store->kv_count * store->head_size;
  a.share = group_share;
  a.query = query;
  a.out = blend_out;
  a.lane_stride = lane_stride;
  a.place = place_first;
  a.newest = place_first + lanes - 1;
  a.newest_slot = a.newest < a.sinks ? -1 : cache4_slot(a.newest, a.sinks, a.span);
  a.window = window;
  a.rows = (int)rows;
  // log2 e, and the 256 that a gain is divided by
  const double factor = (double)store->key_scale * score_scale * 1.4426950408889634 * 256.0;
  a.key_part = (float)frexp(factor, &a.key_power);
  a.value_scale = store->value_scale * 256.0f;
  a.segments = p.segments;
  a.part_out = work;
  a.part_base = work + (size_t)p.segments * store->kv_count * rows * store->head_size;
  a.part_total = a.part_base + (size_t)p.segments * store->kv_count * rows;
  switch (store->head_size) {
    case 64: return attend4_launch_format<64>(a, p, store->format, store->kv_count, stream);
    case 128: return attend4_launch_format<128>(a, p, store->format, store->kv_count, stream);
    case 256: return attend4_launch_format<256>(a, p, store->format, store->kv_count, stream);
    case 512: return attend4_launch_format<512>(a, p, store->format, store->kv_count, stream);
    default: return hipErrorInvalidValue;
  }
}
