// igl_attend4.h - attention over the 4-bit key/value ring (igl_cache4.h) with a
// sliding window and first positions that stay visible, gfx950.
//
// For the query heads q of a lane at position p and the key/value head they
// share, over the visible positions t (t <= p and, with a window, t > p - window
// or t < sinks):
//     o = sum_t 2^(f q . k_t - m) v_t / sum_t 2^(f q . k_t - m),
// f the score scale, the key scale and log2 e, m a base near the peak.
//
// On the matrix cores, in binary16 with fp32 sums.  A key or value is level * gain:
// eight significant bits at most, exact in binary16 with the gain over 256 (their
// scales are multiplied in afterwards).  Queries and weights are two binary16 terms
// each, high and low, 2^-22 of themselves: one term would leave 2^-11, two products
// leave blends as near their 64-bit value as fp32 sums do (2.7e-7 to 5.5e-7 of them).
// Products are taken transposed, S^T = K Q^T and O^T = V^T P^T, so that a lane that
// decodes codes holds a row's eight dims, or a dim's eight rows, as one operand, and a
// query row's scores lie along lanes as its weights are wanted.
//
// A row's base is a whole number about twelve below the block's peak, moved only
// where a peak leaves it by a few: most blocks rescale nothing, a block's largest
// weight is 2^8 to 2^15, and its small ones are held to half of binary16's last
// step, 2^-25.  That is 2^-33 of the largest: of a weight 26 powers of two below it
// in its own block 2^-7 is left, of one 33 below nothing, in other blocks 2^-22.  A
// third term would hold them, for half as many products again.  Bases follow peaks
// down too, to 58 below the highest, so that positions far below others keep what
// fp32 sums keep of them.
//
// Times below are of runs of some ten launches, before the card's clocks have risen:
// after some hundred, what computes takes a tenth less.
#pragma once

#include <float.h>
#include <math.h>

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
  uint32_t share_mul;    // row / share = row * share_mul >> share_shift
  int share_shift;
  int key_power;         // key scale, score scale, log2 e and 256: key_part 2^key_power
  float key_part;        // in [1/2, 1), or of a score scale below zero, or NaN
  float value_scale;
  int segments;          // of a row tile's blocks, each `per` of them and the last what is left
  int per;
  int part_row0;         // first row whose blocks are cut
  float *part_out;       // [segments][kv][rows - part_row0][HEAD], with more than one segment
  float *part_base;      // [segments][kv][rows - part_row0]
  float *part_total;
};

// The blocks of `block` slots that hold what lanes at positions first .. last
// see: blocks 0 .. low - 1, then mid .. mid + count - low - 1.  The visible slots
// are the sinks' and the ring's from the oldest position to the newest, cut in
// two where the ring wraps; the piece from slot sinks on joins the sinks.
struct Blocks4 {
  int low, mid, count;
  int low_ahead, mid_ahead;  // a ring slot's position less the slot, in the two runs
  __host__ __device__ int at(int i) const { return i < low ? i : mid + i - low; }
};

__host__ __device__ inline Blocks4 attend4_blocks(int block, int first, int last, const Attend4Args &a) {
  Blocks4 b = {0, 0, 0, 0, 0};
  int low_slots = last < a.sinks ? last + 1 : a.sinks;
  int oldest = a.window > 0 && first >= a.window ? first + 1 - a.window : 0;
  if (oldest < a.sinks) oldest = a.sinks;
  int mid_first = 0, mid_last = -1;
  if (oldest <= last) {  // all of them within a turn of the ring before the newest
    mid_first = a.newest_slot - (a.newest - oldest);
    if (mid_first < a.sinks) mid_first += a.span - a.sinks;
    mid_last = a.newest_slot - (a.newest - last);
    if (mid_last < a.sinks) mid_last += a.span - a.sinks;
    if (mid_first > mid_last) {
      low_slots = mid_last + 1;
      mid_last = a.span - 1;
    }
  }
  b.low = (low_slots + block - 1) / block;
  b.mid = mid_first / block;
  if (b.mid < b.low) b.mid = b.low;
  const int end = mid_last < 0 ? 0 : mid_last / block + 1;
  b.count = b.low + (end > b.mid ? end - b.mid : 0);
  // slots past the newest position's hold a turn before
  b.low_ahead = a.newest - a.newest_slot;
  b.mid_ahead = b.low_ahead - (mid_first > a.newest_slot ? a.span - a.sinks : 0);
  return b;
}

// The lane of a row of a key/value head.
__host__ __device__ __forceinline__ int attend4_lane(int row, const Attend4Args &a) {
  return (int)(((uint64_t)(uint32_t)row * a.share_mul) >> a.share_shift);
}

// Segments a row's blocks are cut into, at most: the fold takes one a thread.
constexpr int kAttend4Segments = 256;

// The position whose row a slot holds once `newest` is laid, INT_MAX for none; a
// first position is its slot's before it is laid too.
__host__ __device__ __forceinline__ int attend4_place(int slot, const Attend4Args &a) {
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

// Nibbles I of both halves of a dword as 64 + c: moved to bits 4 .. 7 of the
// halves, where they count whole numbers under binary16's exponent of 64.
constexpr uint32_t kNibble64 = 0x54005400u;

template <int I>
__device__ __forceinline__ half2_t nibble_pair64(uint32_t d, uint32_t exp64) {
  const uint32_t moved = I == 0 ? d << 4 : d >> (I == 0 ? 0 : 4 * I - 4);
  return as_half2(and_or_b32(moved, 0x00F000F0u, exp64));
}

// What turns 64 + c into (c - 8) g with one fma: -72 g, exact (72 and g have four
// significant bits each).  E2M1 codes are levels as they are decoded.
__device__ __forceinline__ half2_t gain_offset(half2_t g) { return g * half2_t{(_Float16)-72.0f, (_Float16)-72.0f}; }

// Element e of a key operand of eight dims is dim key_order<FMT>(e) of them: a
// dword's nibbles i and i + 4 lie 16 bits apart, the halves of one register; a
// byte's two are converted together.
template <int FMT>
__host__ __device__ constexpr int key_order(int e) {
  return FMT == IGL_CACHE4_INT4 ? (e >> 1) + 4 * (e & 1) : e;
}

// Eight codes of one row, times their gain (both halves of g; h its offset).
template <int FMT>
__device__ __forceinline__ half8_t key_operand(uint32_t w, half2_t g, half2_t h, uint32_t exp64) {
  half2_t p[4];
  if (FMT == IGL_CACHE4_INT4) {
    p[0] = __builtin_elementwise_fma(nibble_pair64<0>(w, exp64), g, h);
    p[1] = __builtin_elementwise_fma(nibble_pair64<1>(w, exp64), g, h);
    p[2] = __builtin_elementwise_fma(nibble_pair64<2>(w, exp64), g, h);
    p[3] = __builtin_elementwise_fma(nibble_pair64<3>(w, exp64), g, h);
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
                                               uint32_t exp64, half8_t (&out)[DIMS]) {
  half2_t p[DIMS][4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const uint32_t a = x[2 * q], b = x[2 * q + 1];
    if (FMT == IGL_CACHE4_INT4) {
#pragma unroll
      for (int half = 0; half < DIMS / 4; ++half) {
        const uint32_t t = __builtin_amdgcn_perm(b, a, half ? 0x07060302u : 0x05040100u);
        p[4 * half + 0][q] = __builtin_elementwise_fma(nibble_pair64<0>(t, exp64), g[q], h[q]);
        p[4 * half + 1][q] = __builtin_elementwise_fma(nibble_pair64<1>(t, exp64), g[q], h[q]);
        p[4 * half + 2][q] = __builtin_elementwise_fma(nibble_pair64<2>(t, exp64), g[q], h[q]);
        p[4 * half + 3][q] = __builtin_elementwise_fma(nibble_pair64<3>(t, exp64), g[q], h[q]);
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

// The same for four dims, one half (`high`, uniform) of eight rows' dwords.
template <int FMT>
__device__ __forceinline__ void value_operands_half(const uint32_t (&x)[8], bool high, const half2_t (&g)[4],
                                                    const half2_t (&h)[4], uint32_t exp64, half8_t (&out)[4]) {
  const uint32_t pick = high ? 0x07060302u : 0x05040100u;
  half2_t p[4][4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const uint32_t t = __builtin_amdgcn_perm(x[2 * q + 1], x[2 * q], pick);  // the rows' four codes each
    if (FMT == IGL_CACHE4_INT4) {
      p[0][q] = __builtin_elementwise_fma(nibble_pair64<0>(t, exp64), g[q], h[q]);
      p[1][q] = __builtin_elementwise_fma(nibble_pair64<1>(t, exp64), g[q], h[q]);
      p[2][q] = __builtin_elementwise_fma(nibble_pair64<2>(t, exp64), g[q], h[q]);
      p[3][q] = __builtin_elementwise_fma(nibble_pair64<3>(t, exp64), g[q], h[q]);
    } else {
      const uint32_t even = (t & 0x0F0Fu) | ((t >> 12) & 0xF0F0u);         // bytes of both rows: dims 0, 2
      const uint32_t odd = ((t >> 4) & 0x0F0Fu) | ((t >> 16) & 0xF0F0u);   // and 1, 3
      p[0][q] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(even, 1.0f, 0) * g[q];
      p[1][q] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(odd, 1.0f, 0) * g[q];
      p[2][q] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(even, 1.0f, 1) * g[q];
      p[3][q] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(odd, 1.0f, 1) * g[q];
    }
  }
#pragma unroll
  for (int d = 0; d < 4; ++d) out[d] = __builtin_bit_cast(half8_t, p[d]);
}

// The largest over groups of N neighbouring lanes, in each of them.
template <int N>
__device__ __forceinline__ float group_max(float v) {
  v = fmaxf(v, dpp_move<0xB1>(v));
  v = fmaxf(v, dpp_move<0x4E>(v));
  v = fmaxf(v, dpp_move<0x141>(v));
  if (N >= 16) v = fmaxf(v, dpp_move<0x140>(v));
  if (N >= 32) {
    float a = v, b = v;
    asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
    v = fmaxf(a, b);
  }
  if (N >= 64) {
    float a = v, b = v;
    asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
    v = fmaxf(a, b);
  }
  return v;
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

// LDS only: rows requested ahead stay in flight.
__device__ __forceinline__ void attend4_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xC07F);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// A buffer over the rows at a uniform address: scalar registers and a 32-bit
// lane offset.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t attend4_rows(const uint8_t *rows) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(rows), 0, 0xFFFFFFFF, 0x00020000);
}

// Bytes to a row of a block: both factors are below 2^24.
__device__ __forceinline__ uint32_t row_at(int row, uint32_t row_bytes) {
  return ((uint32_t)row & 0xFFFFFFu) * (row_bytes & 0xFFFFFFu);
}

// A row's queries as two binary16 terms: times the score factor's significand and a
// power of two that brings the row's largest, `top`, to [2^12, 2^14) (or as far up as a
// float reaches, then without the significand), so that no query is too large or too
// small for them.  The power of two that is left is the scores' factor: their products
// with it are exact, so that a base lies below a peak by what it should however large
// scores are.  It is never zero, so that it leaves a hidden score's -infinity one.  A
// score factor below zero turns the queries instead.  A NaN or an infinity stays one
// in its terms.
__device__ __forceinline__ float query_factor(const Attend4Args &a, float top, float &scale) {
  const int want = top > 0.0f && top < INFINITY ? 14 - __builtin_amdgcn_frexp_expf(top) : 0;
  const int up = want > 126 ? 126 : want;
  const bool apart = want > 126 || a.key_part == 0.0f;
  const float part = fabsf(a.key_part);
  scale = __builtin_amdgcn_ldexpf(__builtin_copysignf(apart ? 1.0f : part, a.key_part), up);
  const float factor = __builtin_amdgcn_ldexpf(apart ? part : 1.0f, a.key_power - up);
  return factor < FLT_MIN ? FLT_MIN : factor > 0x1p127f ? 0x1p127f : factor;  // nor too large for a score of zero
}

typedef float float2_t __attribute__((ext_vector_type(2)));

// Two values as two binary16 terms each, x = hi + lo to 2^-22 of itself.
__device__ __forceinline__ void two_terms(float x, float y, half2_t &hi, half2_t &lo) {
  hi = __builtin_convertvector((float2_t){x, y}, half2_t);
  lo = __builtin_convertvector(((float2_t){__builtin_fmaf((float)hi[0], -1.0f, x), __builtin_fmaf((float)hi[1], -1.0f, y)}),
                               half2_t);
}

// Eight queries in the key operands' order.
template <int FMT>
__device__ __forceinline__ void query_operands(const float (&x)[8], float scale, half8_t &hi, half8_t &lo) {
  half2_t h[4], l[4];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    two_terms(x[key_order<FMT>(2 * e)] * scale, x[key_order<FMT>(2 * e + 1)] * scale, h[e], l[e]);
  hi = __builtin_bit_cast(half8_t, h);
  lo = __builtin_bit_cast(half8_t, l);
}

// Floats from the queries' (and the blends') start to a row of a key/value head.
__device__ __forceinline__ size_t attend4_row(int row, int kv, int head, const Attend4Args &a) {
  const int l = attend4_lane(row, a);
  return (size_t)l * a.lane_stride + ((size_t)kv * a.share + (row - l * a.share)) * head;
}

// A tile's rows as terms in LDS, a thread eight dims: row r at `to` + r (HEAD + 8),
// its second term `second` halves on, its factor at factors[r].  Rows past the last
// are the last again.
template <int HEAD, int FMT, int ROWS, int THREADS>
struct QueryLoad {
  static constexpr int PIECES = HEAD / 8, ITEMS = ROWS * PIECES, PER = (ITEMS + THREADS - 1) / THREADS;
  float x[PER][8];
  __device__ __forceinline__ void load(const Attend4Args &a, int kv, int row0, int row_last, int tid) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int item = min(tid + THREADS * i, ITEMS - 1);
      const float *src = a.query + attend4_row(min(row0 + item / PIECES, row_last), kv, HEAD, a) + 8 * (item % PIECES);
      const float4_t u = *reinterpret_cast<const float4a_t *>(src), v = *reinterpret_cast<const float4a_t *>(src + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[i][e] = u[e], x[i][4 + e] = v[e];
    }
  }
  __device__ __forceinline__ void store(const Attend4Args &a, int tid, _Float16 *to, int second, float *factors) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int item = tid + THREADS * i;
      if (ITEMS % THREADS != 0 && item >= ITEMS) break;  // whole waves
      float top = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[i][e]));
      top = group_max<PIECES>(top);
      float scale;
      const float factor = query_factor(a, top, scale);
      half8_t hi, lo;
      query_operands<FMT>(x[i], scale, hi, lo);
      const int row = item / PIECES;
      _Float16 *at = to + row * (HEAD + 8) + 8 * (item % PIECES);
      *reinterpret_cast<half8_t *>(at) = hi;
      *reinterpret_cast<half8_t *>(at + second) = lo;
      if (item % PIECES == 0) factors[row] = factor;
    }
  }
};

// Whether a lane at `place` sees a slot's position.
__host__ __device__ __forceinline__ bool attend4_seen(int slot, int place, const Attend4Args &a) {
  const int at = attend4_place(slot, a);
  return at <= place && (a.window == 0 || at > place - a.window || at < a.sinks);
}

// Whether every lane from place_low to place_high sees all of a run's `count` slots
// from slot0 on: all past the sinks, and from the oldest position that the last
// lane sees to the first lane's own (a slot of another turn would lie outside).
__host__ __device__ __forceinline__ bool attend4_all(int slot0, int count, int ahead, int place_low, int place_high,
                                                     const Attend4Args &a) {
  const int place0 = slot0 + ahead;
  return slot0 >= a.sinks && slot0 <= a.span - count && place0 <= place_low - (count - 1) &&
         (a.window == 0 || place0 > place_high - a.window);
}

// Whether a row's base stays after a block with this peak (before its factor).
__device__ __forceinline__ bool attend4_stays(float peak, float factor, float base) {
  const float above = peak * factor - base;
  return (above >= 8.0f && above < 15.0f) || peak == -INFINITY;
}

// The row's base after such a block.
__device__ __forceinline__ float attend4_base(float peak, float factor, float base, float &top_base) {
  if (attend4_stays(peak, factor, base)) return base;
  const float at = peak * factor;
  const float low = fabsf(at) < 0x1p23f ? floorf(at) - 12.0f : at;  // where a float holds whole numbers
  top_base = fmaxf(top_base, low);
  return fmaxf(low, top_base - 58.0f);
}

// What is added to a score (times its factor) below a base; a row that has seen
// nothing yet has none, and only hidden scores.
__device__ __forceinline__ float attend4_from(float base) { return base != -INFINITY ? -base : 0.0f; }

// Writes a row's dims from dim0 + (4 g + r) DPL + j of out[j][r] on: the blend, or
// a segment's share of it (with its base and total where `stats`).  PAIR: columns
// n and n + 8 hold a row's two terms, and each writes half of their sums.
template <int HEAD, int DPL, bool PAIR>
__device__ __forceinline__ void attend4_store(const Attend4Args &a, float4_t (&out)[DPL], float base, float total, int row,
                                              int row_last, int seg, int kv, int dim0, bool stats, int g, int n) {
  if (PAIR) {
#pragma unroll
    for (int j = 0; j < DPL; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) out[j][r] += dpp_move<0x128>(out[j][r]);
  }
  if (row > row_last) return;
  const int l = attend4_lane(row, a);
  float *dst = a.out + (size_t)l * a.lane_stride + ((size_t)kv * a.share + (row - l * a.share)) * HEAD;
  float mul = 1.0f, scale = 1.0f;
  if (a.segments > 1) {
    const size_t at = ((size_t)seg * gridDim.z + kv) * a.rows + row;
    dst = a.part_out + at * HEAD;
    if (stats && g == 0 && (!PAIR || n < 8)) {
      a.part_base[at] = base;
      a.part_total[at] = total;
    }
  } else {
    // the 256 that a gain is divided by; the scale apart, as a total may be past 2^70
    // and a float not hold their product
    mul = 256.0f / total;
    scale = a.value_scale;
  }
  dst += dim0 + 4 * g * DPL;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    if (PAIR && (r >= 2) != (n >= 8)) continue;
#pragma unroll
    for (int j = 0; j < DPL; j += 4) {
      *reinterpret_cast<float4a_t *>(dst + r * DPL + j) =
          float4_t{out[j][r] * mul * scale, out[j + 1][r] * mul * scale, out[j + 2][r] * mul * scale,
                   out[j + 3][r] * mul * scale};
    }
  }
}

// ---- few rows -----------------------------------------------------------------

// Steps and blocks of a few lanes.  Four waves take a block of 64 T slots, the
// scores divided by slots (a wave T tiles of 16, every dim), the blend by dims
// (VD ways) and then by slots (VS ways): so a wave's chain from one barrier to
// the next is a quarter of the block's work.  Weights cross between the two
// divisions through LDS, against a base that the four waves agree on.  The next
// block's codes are on their way while this one's are used.  Up to eight rows
// (PAIR) put both terms of a row into the sixteen columns of one product.
//
// A short context is bound by its chain, about 1.5 us a block, so it is cut over as
// many workgroups as it has blocks: a 512 window of 256-dim heads 5.6 us and 3.7 for
// the fold (one wave a block took 16.9 in all), 16384 positions 6.2 + 3.6.  A long
// one is bound by its bytes and their decoding (16 us of vector issue a CU and 3 of
// matrix): 131072 positions of eight 128-dim heads, 143 MB, in 34.4 us, 4.1 TB/s
// (out of caches 41, 3.5; int4's 37.6 and 45).
//
// Blocks of 512 slots fill the registers of a wave of two a SIMD, which those of
// 128-dim heads ask for: one register more of int4's halved the workgroups a CU, 52 us
// for 37.6.  Those of 64-dim heads have them anyhow, and asking took 0.4 us of 29.
template <int HEAD, bool PAIR, int T>
struct Step4Shape {
  static constexpr int KL = HEAD >= 128 ? HEAD / 128 : 1;  // key chunks of a row a lane reads
  static constexpr int KW = HEAD >= 128 ? 4 : 2;           // dwords of a chunk
  static constexpr int ROWS = PAIR ? 8 : 16;
  static constexpr int TERMS = PAIR ? 1 : 2;
  static constexpr int BLOCK = 64 * T;
  static constexpr int VD = HEAD >= 128 ? HEAD / 128 : 1, VS = 4 / VD;
  static constexpr int DB = HEAD / VD, DPL = DB / 16;      // a wave's dims of the blend, a lane's
  static constexpr int UB = BLOCK / VS / 32;               // its steps of 32 slots
  static constexpr int QP = HEAD + 8, PP = BLOCK + 8;      // pitches in halves
  static constexpr int Q = 0;                              // [TERMS][16][QP]
  static constexpr int P = Q + TERMS * 16 * QP * 2;        // [TERMS][16][PP]
  static constexpr int PEAK = P + TERMS * 16 * PP * 2;     // [4][16]
  static constexpr int FACTOR = PEAK + 4 * 16 * 4;         // [16]
  static constexpr int LOOP = FACTOR + 16 * 4;
  static constexpr int MERGE = (VS - 1) * VD * DPL * 1024;  // the blends of waves that took other slots
  static constexpr int LDS = LOOP > MERGE ? LOOP : MERGE;
  static_assert(UB >= 1, "a blend step takes 32 slots");
  static_assert(BLOCK <= IGL_ATTEND4_BLOCK_MOST, "slots are counted to a block's end");
};

template <int HEAD, int FMT, bool PAIR, int T>
__global__ __launch_bounds__(256, T > 4 && HEAD > 64 ? 2 : 1) void attend4_step_kernel(Attend4Args a) {
  using F = Step4Shape<HEAD, PAIR, T>;
  constexpr int KL = F::KL, KW = F::KW, ROWS = F::ROWS, TERMS = F::TERMS, BLOCK = F::BLOCK;
  constexpr int VD = F::VD, VS = F::VS, DB = F::DB, DPL = F::DPL, UB = F::UB, QP = F::QP, PP = F::PP;
  __shared__ __attribute__((aligned(16))) uint8_t lds[F::LDS];
  _Float16 *qs = reinterpret_cast<_Float16 *>(lds + F::Q), *ws = reinterpret_cast<_Float16 *>(lds + F::P);
  float *peaks = reinterpret_cast<float *>(lds + F::PEAK), *factors = reinterpret_cast<float *>(lds + F::FACTOR);

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int vd = wave % VD, vs = wave / VD;
  const int g = lane >> 4, n = lane & 15;
  const int kv = blockIdx.z, seg = blockIdx.y;
  const int row0 = (int)blockIdx.x * ROWS;
  const int row_last = min(row0 + ROWS, a.rows) - 1;
  const int place_low = a.place + attend4_lane(row0, a), place_high = a.place + attend4_lane(row_last, a);
  const Blocks4 blocks = attend4_blocks(BLOCK, place_low, place_high, a);
  const int first = min(blocks.count, seg * a.per);
  const int end = seg == a.segments - 1 ? blocks.count : min(blocks.count, first + a.per);
  const uint32_t exp64 = kNibble64;
  const uint32_t row_bytes = (uint32_t)a.kv_width / 2;
  const size_t head_bytes = (size_t)kv * HEAD / 2;
  const size_t gain_row = (size_t)kv * HEAD / kCache4Group;

  uint32_t kr[T][KL][KW], kg[T][KL], vr[UB][8];
  uint2_t vg[UB];
  const uint32_t k_lane = (uint32_t)n * row_bytes + (KW == 4 ? 16 : 8) * g;
  const uint32_t v_lane = (uint32_t)(8 * g) * row_bytes + (uint32_t)((vd * DB + n * DPL) / 2);
  const size_t k_gain_lane = (size_t)(KW == 4 ? g : g / 2) * a.room + n;
  const size_t v_gain_lane = (size_t)((vd * DB + n * DPL) / kCache4Group) * a.room + 8 * g;
  auto load_keys = [&](int i) {
    const int slot0 = blocks.at(i) * BLOCK;
    const auto src = attend4_rows(a.key_code + (size_t)slot0 * row_bytes + head_bytes);
    const bool whole = slot0 <= a.span - BLOCK;
#pragma unroll
    for (int j = 0; j < T; ++j) {
      const int at = 16 * (T * wave + j);
      const uint32_t off = whole ? k_lane : row_at(min(at + n, a.span - 1 - slot0), row_bytes) + (KW == 4 ? 16 : 8) * g;
      const uint32_t base = whole ? (uint32_t)at * row_bytes : 0u;
#pragma unroll
      for (int c = 0; c < KL; ++c) {
        if constexpr (KW == 4) {
          const uint4_t w = __builtin_amdgcn_raw_buffer_load_b128(src, off + 64 * c, base, 0);
#pragma unroll
          for (int s = 0; s < 4; ++s) kr[j][c][s] = w[s];
        } else {
          const uint2_t w = __builtin_amdgcn_raw_buffer_load_b64(src, off, base, 0);
          kr[j][c][0] = w[0];
          kr[j][c][1] = w[1];
        }
      }
      // gain rows end on a block: past the ring's end lies their padding
#pragma unroll
      for (int c = 0; c < KL; ++c)
        kg[j][c] = a.key_gain[(gain_row + 4 * c) * a.room + min(slot0 + at, (int)a.room - 16) + k_gain_lane];
    }
  };
  auto load_values = [&](int i) {
    const int slot0 = blocks.at(i) * BLOCK;
    const auto src = attend4_rows(a.value_code + (size_t)slot0 * row_bytes + head_bytes);
    const bool whole = slot0 <= a.span - BLOCK;
#pragma unroll
    for (int u = 0; u < UB; ++u) {
      const int at = 32 * (UB * vs + u);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t off = whole ? v_lane
                                   : row_at(min(at + 8 * g + e, a.span - 1 - slot0), row_bytes) +
                                         (uint32_t)((vd * DB + n * DPL) / 2);
        const uint32_t base = whole ? (uint32_t)(at + e) * row_bytes : 0u;
        if constexpr (DPL == 4)
          vr[u][e] = __builtin_amdgcn_raw_buffer_load_b16(src, off, base, 0);
        else
          vr[u][e] = __builtin_amdgcn_raw_buffer_load_b32(src, off, base, 0);
      }
      vg[u] = *reinterpret_cast<const uint2_t *>(a.value_gain + gain_row * a.room + min(slot0 + at, (int)a.room - 32) +
                                                 v_gain_lane);
    }
  };

  // ---- the rows' queries to LDS; PAIR: a row's second term in column n + 8
  QueryLoad<HEAD, FMT, ROWS, 256> queries;
  queries.load(a, kv, row0, row_last, tid);
  if (first < end) {
    load_keys(first);
    load_values(first);
  }
  queries.store(a, tid, qs, (PAIR ? 8 : 16) * QP, factors);
  attend4_barrier();
  const int row = PAIR ? n & 7 : n;
  const int place = a.place + attend4_lane(min(row0 + row, row_last), a);
  const float factor = factors[row];
  auto query_at = [&](int m, int i) {  // key step i = KW c + w
    const int d = KW == 4 ? 32 * (4 * (i / 4) + g) + 8 * (i % 4) : 16 * g + 8 * i;
    return *reinterpret_cast<const half8_t *>(qs + (size_t)(m * 16 + n) * QP + d);
  };
  constexpr bool KEEP = KL * KW * TERMS <= 16;  // in registers through the loop
  half8_t q[TERMS][KL * KW];
  if (KEEP) {
#pragma unroll
    for (int m = 0; m < TERMS; ++m)
#pragma unroll
      for (int i = 0; i < KL * KW; ++i) q[m][i] = query_at(m, i);
  }

  float4_t out[DPL];
  float base = -INFINITY, top_base = -INFINITY, total = 0.0f;
#pragma unroll
  for (int j = 0; j < DPL; ++j) out[j] = float4_t{0, 0, 0, 0};
  for (int i = first; i < end; ++i) {
    float4_t s[T];
#pragma unroll
    for (int j = 0; j < T; ++j) s[j] = float4_t{0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < KL; ++c) {
      half2_t gain[T], off[T];
#pragma unroll
      for (int j = 0; j < T; ++j) {
        gain[j] = half_low(gain_pair(kg[j][c]));
        off[j] = gain_offset(gain[j]);
      }
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        half8_t k[T];
#pragma unroll
        for (int j = 0; j < T; ++j) k[j] = key_operand<FMT>(kr[j][c][w], gain[j], off[j], exp64);
#pragma unroll
        for (int m = TERMS - 1; m >= 0; --m) {
          const half8_t op = KEEP ? q[m][KW * c + w] : query_at(m, KW * c + w);
#pragma unroll
          for (int j = 0; j < T; ++j) s[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[j], op, s[j], 0, 0, 0);
        }
      }
    }
    if (i + 1 < end) load_keys(i + 1);

    // ---- the block's peaks
    const int slot0 = blocks.at(i) * BLOCK;
    const bool all =
        attend4_all(slot0, BLOCK, i < blocks.low ? blocks.low_ahead : blocks.mid_ahead, place_low, place_high, a);  // uniform
    if (PAIR) {
#pragma unroll
      for (int j = 0; j < T; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[j][r] += dpp_move<0x128>(s[j][r]);  // row n and n + 8
    }
    if (!all) {
#pragma unroll
      for (int j = 0; j < T; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (!attend4_seen(slot0 + 16 * (T * wave + j) + 4 * g + r, place, a)) s[j][r] = -INFINITY;
    }
    float peak = -INFINITY;
#pragma unroll
    for (int j = 0; j < T; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) peak = fmaxf(peak, s[j][r]);
    peak = xmax48(peak);
    if (g == 0) peaks[wave * 16 + n] = peak;
    attend4_barrier();
    // ---- the base, the same in every wave, and the weights
#pragma unroll
    for (int w = 0; w < 4; ++w) peak = fmaxf(peak, peaks[w * 16 + n]);
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(!attend4_stays(peak, factor, base)) != 0, 0)) {
      const float m = attend4_base(peak, factor, base, top_base);
      const float keep = base != -INFINITY ? __builtin_amdgcn_exp2f(base - m) : 0.0f;
      total *= keep;
#pragma unroll
      for (int j = 0; j < DPL; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) out[j][r] *= keep;
      base = m;
    }
    const float from = attend4_from(base);
#pragma unroll
    for (int j = 0; j < T; ++j) {
      half2_t hi[2], lo[2];
#pragma unroll
      for (int r = 0; r < 4; r += 2) {
        const float w0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j][r], factor, from));
        const float w1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j][r + 1], factor, from));
        total += w0 + w1;
        two_terms(w0, w1, hi[r / 2], lo[r / 2]);
        if (PAIR && n >= 8) hi[r / 2] = lo[r / 2];
      }
      _Float16 *to = ws + n * PP + 16 * (T * wave + j) + 4 * g;
      __builtin_memcpy(__builtin_assume_aligned(to, 8), hi, sizeof(hi));
      if (!PAIR) __builtin_memcpy(__builtin_assume_aligned(to + 16 * PP, 8), lo, sizeof(lo));
    }
    attend4_barrier();
    // ---- the blend of the wave's dims over its slots
#pragma unroll
    for (int u = 0; u < UB; ++u) {
      half8_t p[TERMS];
#pragma unroll
      for (int m = 0; m < TERMS; ++m)
        p[m] = *reinterpret_cast<const half8_t *>(ws + (size_t)(m * 16 + n) * PP +
                                                      32 * (UB * vs + u) + 8 * g);
      half2_t gain[4], off[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        gain[k] = gain_pair(__builtin_amdgcn_perm(0u, vg[u][k >> 1], k & 1 ? 0x0C030C02u : 0x0C010C00u));
        off[k] = gain_offset(gain[k]);
      }
      half8_t op[DPL];
      value_operands<FMT, DPL>(vr[u], gain, off, exp64, op);
#pragma unroll
      for (int m = TERMS - 1; m >= 0; --m)
#pragma unroll
        for (int d = 0; d < DPL; ++d)
          out[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(op[d], p[m], out[d], 0, 0, 0);
    }
    if (i + 1 < end) load_values(i + 1);
  }

  // ---- the waves' totals and, of waves that took other slots, blends
  attend4_barrier();
  total = xsum48(total);
  if (g == 0) peaks[wave * 16 + n] = total;
  attend4_barrier();
  total = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; ++w) total += peaks[w * 16 + n];
  if constexpr (VS > 1) {
    attend4_barrier();
    float4_t *room = reinterpret_cast<float4_t *>(lds) + lane;
    if (vs > 0) {
#pragma unroll
      for (int j = 0; j < DPL; ++j) room[(((vs - 1) * VD + vd) * DPL + j) * 64] = out[j];
    }
    attend4_barrier();
    if (vs > 0) return;
#pragma unroll
    for (int w = 1; w < VS; ++w)
#pragma unroll
      for (int j = 0; j < DPL; ++j) out[j] += room[(((w - 1) * VD + vd) * DPL + j) * 64];
  }
  attend4_store<HEAD, DPL, PAIR>(a, out, base, total, row0 + row, row_last, seg, kv, vd * DB, vd == 0, g, n);
}

// ---- many rows ----------------------------------------------------------------

// Prompts.  A workgroup of eight waves takes four tiles of 16 rows through blocks
// of slots, whose codes its waves decode together into LDS as binary16 operands,
// once for all its rows and a block ahead of the products.  Two waves share a
// tile's products: of 512-dim heads each takes half the dims (their partial scores
// meet in LDS), of others half the block's slots (their blends meet in LDS at the
// end).  Transposed, scores stay where the blend wants them: lane 16 g + n of S^T
// (slots x rows) holds row n's slots 4 g + r of 16-slot tile b, and of P^T, with slot
// 16 b + 4 g + r as element 4 b + r of lane group g's eight, the same.
//
// A wave decodes the next block while it multiplies this one's keys: an item of 32
// dims of a key and one of four dims of a lane group's eight slots of values a
// thread, in straight code that the scheduler is told to lay between the products.
// Blends leave through LDS as whole rows (scattered dwords were 4 us of a window's 41).
//
// 2047 lanes of 512-dim heads 121 us, 34 GFLOP before the second terms; of a 512 window
// of 256-dim heads 36 us.  No unit is full: of 207k busy cycles a CU vector work, half
// of it decoding, issues in 100k a SIMD, products in 67k, LDS serves in 81k.  A block's
// scores, exchange, weights and blend follow one another, and two waves a SIMD, which
// is what 250 registers leave, cover for each other only in part: a wave waits for data
// or barriers in a third of its cycles and for its turn to issue in three tenths.  64
// rows a workgroup halve the decoding of 32 (156 and 41 us).
//
// LDS.  Keys: a slot's dims in 16-byte pieces, piece s of chunk c (dims 32 c + 8 s ..
// + 7, a dword of codes) at s HEAD / 32 + c, xor the slot's low bits.  Values: a dim's
// 32 slots in four pieces, one a lane group; dim 8 d + i is row i HEAD / 8 + d, its
// piece for g at g xor the row's bits 1 and 2.  So the eight lanes that one cycle
// writes or reads lie in distinct banks, with no padding.
template <int HEAD>
struct Tile4Shape {
  static constexpr int RT = 4, WAVES = 8;
  static constexpr int DW = HEAD == 512 ? 2 : 1, SH = 2 / DW;
  static constexpr int BLOCK = HEAD == 512 ? 32 : 64;
  static constexpr int DH = HEAD / DW;                     // dims a wave multiplies
  static constexpr int KS = DH / 32;                       // its key steps
  static constexpr int DPL = DH / 16;                      // its tiles of 16 dims of the blend
  static constexpr int KITEMS = BLOCK * HEAD / 32;         // chunks of 32 dims, a thread each: all or half of the 512
  static constexpr int VITEMS = BLOCK / 32 * 4 * HEAD / 8; // (lane group, 8 dims) of the block's 32s of slots
  static constexpr int V = BLOCK * HEAD * 2;               // bytes of a block's keys, and of its values
  static constexpr int X = 4 * V;                          // partial scores: [WAVES][2][64] float4
  static constexpr int LOOP = X + (DW > 1 ? WAVES * 2048 : 0);
  static constexpr int QUERY = 2 * 16 * RT * (HEAD + 8) * 2;     // [2][16 RT][HEAD + 8] halves, before the loop
  static constexpr int ROWS = SH * 16 * RT * HEAD * 4;           // [SH][16 RT][HEAD] floats, after it
  static constexpr int STATS = LOOP > QUERY ? (LOOP > ROWS ? LOOP : ROWS) : (QUERY > ROWS ? QUERY : ROWS);
  static constexpr int LDS = STATS + WAVES * 32 * 4;
  static_assert(KITEMS <= 512 && VITEMS <= 256, "an item of each a thread");
};

template <int HEAD, int FMT>
__global__ __launch_bounds__(512, 2) void attend4_tile_kernel(Attend4Args a) {
  using F = Tile4Shape<HEAD>;
  constexpr int RT = F::RT, DW = F::DW, SH = F::SH, THREADS = 512, BLOCK = F::BLOCK, DH = F::DH, KS = F::KS;
  constexpr int DPL = F::DPL, TC = DH / 128;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds4[];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rt = wave >> 1, dw = DW > 1 ? wave & 1 : 0, sh = SH > 1 ? wave & 1 : 0;
  const int g = lane >> 4, n = lane & 15;
  const int kv = blockIdx.z, seg = blockIdx.y;
  const int row0 = (int)(gridDim.x - 1 - blockIdx.x) * 16 * RT;  // a prompt's longest first
  const int row_last = min(row0 + 16 * RT, a.rows) - 1;
  const bool split = a.segments > 1 && row0 >= a.part_row0;
  if (seg > 0 && !split) return;
  const int place_low = a.place + attend4_lane(row0, a), place_high = a.place + attend4_lane(row_last, a);
  const Blocks4 blocks = attend4_blocks(BLOCK, place_low, place_high, a);
  const int first = min(blocks.count, seg * a.per);
  const int end = !split || seg == a.segments - 1 ? blocks.count : min(blocks.count, first + a.per);
  const uint32_t exp64 = kNibble64;
  const uint32_t row_bytes = (uint32_t)a.kv_width / 2;
  const size_t head_bytes = (size_t)kv * HEAD / 2;
  const size_t gain_row = (size_t)kv * HEAD / kCache4Group;

  // ---- a thread's items of a block: where there are fewer than threads, two write
  // the same
  const int k_item = tid % F::KITEMS, k_slot = k_item / (HEAD / 32), k_chunk = k_item % (HEAD / 32);
  const int v_item = (tid & 255) % F::VITEMS, v_dims = v_item % (HEAD / 8), v_of = v_item / (HEAD / 8) % 4;
  const int v_group = v_item / (HEAD / 2), v_slot = 32 * v_group + 4 * v_of;
  const bool v_high = wave >= 4;  // which four of the eight dims
  uint4_t kr;
  uint32_t kg, vr[8], vg[2];
  const uint8_t *const k_gain = a.key_gain + (gain_row + k_chunk) * a.room + k_slot;
  const uint8_t *const v_gain = a.value_gain + (gain_row + v_dims / 4) * a.room + v_slot;
  const uint32_t k_lane = row_at(k_slot, row_bytes) + 16 * k_chunk, v_lane = row_at(v_slot, row_bytes) + 4 * v_dims;
  auto load = [&](int i) {
    const int slot0 = blocks.at(i) * BLOCK;
    const auto keys = attend4_rows(a.key_code + (size_t)slot0 * row_bytes + head_bytes);
    const auto values = attend4_rows(a.value_code + (size_t)slot0 * row_bytes + head_bytes);
    if (slot0 <= a.span - BLOCK) {  // uniform: rows at scalar distances
      kr = __builtin_amdgcn_raw_buffer_load_b128(keys, k_lane, 0, 0);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        vr[e] = __builtin_amdgcn_raw_buffer_load_b32(values, v_lane, (16 * (e >> 2) + (e & 3)) * row_bytes, 0);
    } else {
      const int left = a.span - 1 - slot0;  // rows past the ring's last slot are read from it
      kr = __builtin_amdgcn_raw_buffer_load_b128(keys, row_at(min(k_slot, left), row_bytes) + 16 * k_chunk, 0, 0);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int slot = v_slot + 16 * (e >> 2) + (e & 3);
        vr[e] = __builtin_amdgcn_raw_buffer_load_b32(values, row_at(min(slot, left), row_bytes) + 4 * v_dims, 0, 0);
      }
    }
    kg = k_gain[slot0];
#pragma unroll
    for (int b = 0; b < 2; ++b) vg[b] = *reinterpret_cast<const uint32_t *>(v_gain + slot0 + 16 * b);
  };
  auto decode = [&](uint8_t *room) {
    {
      const half2_t gain = half_low(gain_pair(kg)), off = gain_offset(gain);
      half8_t *to = reinterpret_cast<half8_t *>(room) + k_slot * (HEAD / 8);
#pragma unroll
      for (int s = 0; s < 4; ++s)
        to[(s * (HEAD / 32) + k_chunk) ^ (k_slot & 7)] = key_operand<FMT>(kr[s], gain, off, exp64);
    }
    half2_t gain[4], off[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      gain[k] = gain_pair(__builtin_amdgcn_perm(0u, vg[k >> 1], k & 1 ? 0x0C030C02u : 0x0C010C00u));
      off[k] = gain_offset(gain[k]);
    }
    half8_t op[4];
    value_operands_half<FMT>(vr, v_high, gain, off, exp64, op);
    half8_t *to = reinterpret_cast<half8_t *>(room + F::V) + v_group * (HEAD * 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = (i + (v_high ? 4 : 0)) * (HEAD / 8) + v_dims;
      to[row * 4 + (v_of ^ (row >> 1 & 3))] = op[i];
    }
  };
  QueryLoad<HEAD, FMT, 16 * RT, THREADS> queries;
  queries.load(a, kv, row0, row_last, tid);
  if (first < end) load(first);

  // ---- the rows' queries: their terms through LDS, a thread eight dims, to the
  // waves' operands
  half8_t q[2][KS];
  float *stats = reinterpret_cast<float *>(lds4 + F::STATS);
  constexpr int QP = HEAD + 8;  // pitch in halves
  _Float16 *qs = reinterpret_cast<_Float16 *>(lds4);
  queries.store(a, tid, qs, 16 * RT * QP, stats);
  attend4_barrier();
  const int row = min(row0 + 16 * rt + n, row_last);
  const int place = a.place + attend4_lane(row, a);
  const float factor = stats[16 * rt + n];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int k = 0; k < KS; ++k) {  // step 4 c + s is dword s of chunk 4 c + g
      const int d = DH * dw + 32 * (4 * (k / 4) + g) + 8 * (k % 4);
      q[m][k] = *reinterpret_cast<const half8_t *>(qs + m * (16 * RT * QP) + (16 * rt + n) * QP + d);
    }
  attend4_barrier();

  float4_t out[DPL];
  float base = -INFINITY, top_base = -INFINITY, total = 0.0f;
#pragma unroll
  for (int j = 0; j < DPL; ++j) out[j] = float4_t{0, 0, 0, 0};
  uint8_t *now = lds4, *next = lds4 + 2 * F::V;
  if (first < end) {
    decode(now);
    load(min(first + 1, end - 1));
    attend4_barrier();
  }
  for (int i = first; i < end; ++i) {
    // ---- scores, and the next block's operands
    const half8_t *keys = reinterpret_cast<const half8_t *>(now) + 32 * sh * (HEAD / 8);
    float4_t s[2] = {float4_t{0, 0, 0, 0}, float4_t{0, 0, 0, 0}}, low[2] = {s[0], s[1]};
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const int piece = (k % 4) * (HEAD / 32) + (DH / 32) * dw + 4 * (k / 4) + g;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int slot = 16 * b + n;
        const half8_t op = keys[slot * (HEAD / 8) + (piece ^ (slot & 7))];
        low[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(op, q[1][k], low[b], 0, 0, 0);
        s[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(op, q[0][k], s[b], 0, 0, 0);
      }
    }
    decode(next);
    // two products, the next one's operand, and their share of the decoding
    __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
#pragma unroll
    for (int k = 0; k < 2 * KS; ++k) {
      __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 128 / (2 * KS), 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      if (k % (KS / 4) == 0) __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);
    }
    load(min(i + 2, end - 1));
    s[0] += low[0];
    s[1] += low[1];
    if constexpr (DW > 1) {
      float4_t *room = reinterpret_cast<float4_t *>(lds4 + F::X);
#pragma unroll
      for (int b = 0; b < 2; ++b) room[(wave * 2 + b) * 64 + lane] = s[b];
      attend4_barrier();
#pragma unroll
      for (int b = 0; b < 2; ++b) s[b] = room[((wave & ~1) * 2 + b) * 64 + lane] + room[((wave | 1) * 2 + b) * 64 + lane];
    }
    // ---- the rows' weights
    const int slot0 = blocks.at(i) * BLOCK + 32 * sh;
    const bool all =
        attend4_all(slot0, 32, i < blocks.low ? blocks.low_ahead : blocks.mid_ahead, place_low, place_high, a);  // uniform
    if (!all) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (!attend4_seen(slot0 + 16 * b + 4 * g + r, place, a)) s[b][r] = -INFINITY;
    }
    float peak = -INFINITY;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) peak = fmaxf(peak, s[b][r]);
    peak = xmax48(peak);
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(!attend4_stays(peak, factor, base)) != 0, 0)) {
      const float m = attend4_base(peak, factor, base, top_base);
      const float keep = base != -INFINITY ? __builtin_amdgcn_exp2f(base - m) : 0.0f;
      total *= keep;
#pragma unroll
      for (int j = 0; j < DPL; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) out[j][r] *= keep;
      base = m;
    }
    half8_t p[2];
    {
      half2_t hi[4], lo[4];
      const float from = attend4_from(base);
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
          const float w0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][r], factor, from));
          const float w1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][r + 1], factor, from));
          total += w0 + w1;
          two_terms(w0, w1, hi[2 * b + r / 2], lo[2 * b + r / 2]);
        }
      p[0] = __builtin_bit_cast(half8_t, hi);
      p[1] = __builtin_bit_cast(half8_t, lo);
    }
    // ---- the blend: tile j is rows (j / TC) HEAD / 8 + 16 (j % TC) + .. of the wave's
    const half8_t *values = reinterpret_cast<const half8_t *>(now + F::V) + sh * (HEAD * 4);
#pragma unroll
    for (int j = 0; j < DPL; ++j) {
      const int at = (j / TC) * (HEAD / 8) + dw * (DH / 8) + 16 * (j % TC) + n;
      const half8_t op = values[at * 4 + (g ^ (at >> 1 & 3))];
#pragma unroll
      for (int k = 1; k >= 0; --k) out[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(op, p[k], out[j], 0, 0, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 1);
#pragma unroll
    for (int j = 0; j < DPL; ++j) {
      __builtin_amdgcn_sched_group_barrier(0x008, 2, 1);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 1);
    }
    uint8_t *const was = now;
    now = next;
    next = was;
    attend4_barrier();
  }
  total = xsum48(total);

  // ---- blends through LDS, which the waves' halves of the slots meet in, to whole
  // rows: 16-byte piece p of row r at p ^ r % 8
  if (g == 0) {
    stats[wave * 32 + n] = base;
    stats[wave * 32 + 16 + n] = total;
  }
  attend4_barrier();
  float mul = 1.0f;
  if constexpr (SH > 1) {
    const float theirs = stats[(wave ^ 1) * 32 + n], m = fmaxf(base, theirs);
    const float mine = base != -INFINITY ? __builtin_amdgcn_exp2f(base - m) : 0.0f;
    const float part = theirs != -INFINITY ? __builtin_amdgcn_exp2f(theirs - m) : 0.0f;
    base = m;
    total = total * mine + stats[(wave ^ 1) * 32 + 16 + n] * part;
    mul *= mine;
  }
  if (!split) mul *= 256.0f / total;  // the value scale after it, as attend4_store has them
  const float scale = split ? 1.0f : a.value_scale;
  float *rows = reinterpret_cast<float *>(lds4) + sh * (16 * RT * HEAD) + (16 * rt + n) * HEAD;
#pragma unroll
  for (int t = 0; t < TC; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int h = 0; h < 8; h += 4) {  // the tiles t, t + TC, .. are its dims
        const int piece = dw * (DH / 4) + 2 * (16 * t + 4 * g + r) + h / 4;
        *reinterpret_cast<float4_t *>(rows + 4 * (piece ^ (n & 7))) =
            float4_t{out[TC * h + t][r] * mul, out[TC * (h + 1) + t][r] * mul, out[TC * (h + 2) + t][r] * mul,
                     out[TC * (h + 3) + t][r] * mul};
      }
  attend4_barrier();
  const int count = row_last - row0 + 1;
  const size_t part0 = ((size_t)seg * gridDim.z + kv) * (a.rows - a.part_row0) + (row0 - a.part_row0);
  for (int i = tid; i < count * (HEAD / 4); i += THREADS) {
    const int r = i / (HEAD / 4), piece = i % (HEAD / 4);
    const float *from = reinterpret_cast<const float *>(lds4) + r * HEAD + 4 * (piece ^ (r & 7));
    float4_t o = *reinterpret_cast<const float4_t *>(from);
    if (SH > 1) o += *reinterpret_cast<const float4_t *>(from + 16 * RT * HEAD);
    float *to = (split ? a.part_out + (part0 + r) * HEAD : a.out + attend4_row(row0 + r, kv, HEAD, a)) + 4 * piece;
    *reinterpret_cast<float4a_t *>(to) = o * scale;
  }
  if (split && g == 0 && dw == 0 && sh == 0 && 16 * rt + n < count) {
    a.part_base[part0 + 16 * rt + n] = base;
    a.part_total[part0 + 16 * rt + n] = total;
  }
}

// Folds the segments of a row: a workgroup a row and DIMS of its dims, thread
// (c, s) of four dims c and the segments s, s + SL, ...  Thread t finds segment
// t's weight; the blends are requested before.  Segments are added in the same
// order every time.  Few rows are cut by dims to fill the card, bound by the chain
// of three loads (3.6 us at 9 and at 256 segments); many rows are taken whole, so
// that statistics are read once (7928 rows of two segments, 512 dims, 12 us, 4.1
// TB/s; by 64 dims 60).
template <int DIMS>
__global__ __launch_bounds__(256) void attend4_fold_kernel(Attend4Args a, int head_size) {
  constexpr int COLS = DIMS / 4, SL = 256 / COLS;
  constexpr int AHEAD = 4;
  __shared__ float weight[kAttend4Segments], red[8];
  __shared__ float4_t part[SL][COLS];
  const int tid = threadIdx.x, c = tid % COLS, sl = tid / COLS;
  const int wave = tid >> 6;
  const int row = a.part_row0 + (int)blockIdx.x, kv = blockIdx.y, kv_count = gridDim.y;
  const size_t step = (size_t)kv_count * gridDim.x, at = (size_t)kv * gridDim.x + blockIdx.x;
  const int d0 = blockIdx.z * DIMS + 4 * c;
  const float mine = tid < a.segments ? a.part_base[at + tid * step] : -INFINITY;
  const float sum = tid < a.segments ? a.part_total[at + tid * step] : 0.0f;
  float4_t first[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) {
    const int s = min(sl + i * SL, a.segments - 1);
    first[i] = *reinterpret_cast<const float4_t *>(a.part_out + (at + s * step) * head_size + d0);
  }
  const float top = group_max<64>(mine);
  if ((tid & 63) == 0) red[wave] = top;
  attend4_barrier();
  const float m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float w = mine != -INFINITY ? __builtin_amdgcn_exp2f(mine - m) : 0.0f;
  weight[tid] = w;
  const float part_total = wave_sum_to_last(w * sum);
  if ((tid & 63) == 63) red[4 + wave] = part_total;
  attend4_barrier();
  float4_t acc = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) {
    const int s = sl + i * SL;
    if (s < a.segments) acc += first[i] * weight[s];
  }
  for (int s = sl + AHEAD * SL; s < a.segments; s += SL)
    acc += *reinterpret_cast<const float4_t *>(a.part_out + (at + s * step) * head_size + d0) * weight[s];
  part[sl][c] = acc;
  // the slices by halves, in the same order every time
#pragma unroll
  for (int half = SL / 2; half > 0; half >>= 1) {
    attend4_barrier();
    if (sl < half) {
      acc += part[sl + half][c];
      part[sl][c] = acc;
    }
  }
  if (sl) return;
  const float mul = 256.0f / (red[4] + red[5] + red[6] + red[7]);
  *reinterpret_cast<float4a_t *>(a.out + attend4_row(row, kv, head_size, a) + d0) = acc * mul * a.value_scale;
}

}  // namespace igl

using namespace igl;

// How a launch is cut: tiles of up to eight rows (`pair`) or sixteen on
// attend4_step_kernel, or of 64 on attend4_tile_kernel; blocks of `block` slots.
struct Attend4Plan {
  bool step, pair;
  int deep;                // times the slots of a step's block, 2 or 4, or 0
  int block, each, tiles;  // rows a tile
  int blocks;              // of the tile with most, or a bound of it
  long long all;           // of all tiles
};

// Counts a form's blocks.  Without a window the last tile has most; with one, as
// many as any alignment of a tile's span and the sinks' can touch.
static int attend4_tile_blocks(const Attend4Plan &p, int tile, const Attend4Args &a) {
  const int low = tile * p.each, high = a.rows - low < p.each ? a.rows - 1 : low + p.each - 1;
  return attend4_blocks(p.block, a.place + low / a.share, a.place + high / a.share, a).count;
}

static void attend4_count(Attend4Plan &p, const Attend4Args &a) {
  p.tiles = (int)(((long long)a.rows + p.each - 1) / p.each);
  p.blocks = attend4_tile_blocks(p, p.tiles - 1, a);
  p.all = (long long)p.blocks * p.tiles;
  if (a.window > 0) {
    const long long reach = (long long)a.window + (p.each + a.share - 2) / a.share;
    const long long most = (reach + p.block - 2) / p.block + 1 + (a.sinks + p.block - 1) / p.block + 1;
    const int whole = attend4_blocks(p.block, a.place, a.newest, a).count;
    p.blocks = most < whole ? (int)most : whole;
    p.all = (long long)p.blocks * p.tiles;
  } else if (p.tiles > 1) {  // between the first tile's and the last's, evenly
    p.all = ((long long)attend4_tile_blocks(p, 0, a) + p.blocks) * p.tiles / 2;
  }
}

// `room`: floats there are for partials.
static Attend4Plan attend4_plan(Attend4Args &a, int head, int kv_count, long long room = IGL_ATTEND4_FLOATS) {
  const long long cus = 256;
  Attend4Plan p = {};
  // Tiles of 64 rows, where they give every CU more than six blocks of 64 slots:
  // 2047 lanes of a 512 window, 256-dim heads, 36 us (step form 49), of 512-dim heads
  // 64 (76), a prompt of as many 62 + 10 (100) and 122 + 12 (168), 100 lanes at 15000
  // 40 + 6 (53 + 6); but 1000 lanes, 4.6 blocks, 27 + 10 (25).  64-dim heads decode so
  // little that they never do: 45 + 10 (37).
  p.block = head == 512 ? 32 : 64;
  p.each = 64;
  p.step = true;
  if (a.rows > 48 && head >= 128) {
    attend4_count(p, a);
    p.step = p.all * kv_count * p.block <= 6 * 64 * cus;
  }
  if (p.step) {
    p.pair = a.rows <= 8;
    p.each = p.pair ? 8 : 16;
    p.block = head < 256 ? 128 : 64;
    // Four times the slots between barriers, and on their way, where every workgroup
    // still has two such blocks: 131072 positions of eight 128-dim heads in caches 40.7 ->
    // 34.6 us (35.9 by twice), int4's 44.2 -> 37.4 (39.3); out of them 50.2 -> 40.7 and
    // 51.2 -> 44.2; and no more than an eighth more slots than in small blocks, by which
    // it waits for its last: 200000 of eight 77.8 -> 73.2 (3584 for 3200), but 40000 of
    // sixteen 28.4 -> 35.0 (25.3 by twice), 66000 of eight 29.7 -> 34.4, 105000 35.9 ->
    // 41.5.  Of 64-dim heads a fifth: 200000 61.0 -> 46.0, but 80000 of eight 27.4 -> 29.8,
    // 40000 of sixteen 24.0 -> 29.7 (20.0 by twice), 66000 25.7 -> 28.6.  Else twice the
    // slots, where it has two of those and no more slots than in small blocks: 131072 of
    // two 64-dim heads 12.4 -> 10.0 us (int4) and 10.8 -> 9.6, 128-dim 15.6 -> 13.8 and
    // 15.0 -> 13.2, 32768 of eight 15.2 -> 13.6 and 14.6 -> 12.9, 80000 30.9 -> 29.8; but
    // 33000, 768 slots for 640, 19.0 -> 20.2.  Not of wide heads, whose rows already fill
    // the registers: two 512-dim heads by twice the slots 32.9 -> 42.8.
    if (p.pair && head < 256) {
      const auto blocks = [&](int times) {
        return (long long)attend4_blocks(times * p.block, a.place, a.newest, a).count * kv_count;
      };
      const auto slots = [&](int times) {  // of a workgroup, in small blocks
        return (blocks(times) + 2 * cus - 1) / (2 * cus) * times;
      };
      const int part = head == 64 ? 5 : 8;
      if (blocks(4) >= 2 * 2 * cus && slots(4) * part <= slots(1) * (part + 1))
        p.deep = 4;
      else if (blocks(2) >= 2 * 2 * cus && slots(2) <= slots(1))
        p.deep = 2;
      if (p.deep) p.block *= p.deep;
    }
    attend4_count(p, a);
  }

  // Segments: as many as fill the card, two step workgroups a CU (each taken for the
  // longest: a cut of all rows costs a fold) or one of the tiles'.
  const auto floats = [&](long long segments) { return segments * kv_count * (a.rows - a.part_row0) * (head + 2); };
  const int per_least = (p.blocks + kAttend4Segments - 1) / kAttend4Segments;
  const long long at_once = p.step ? 2 * cus : cus;
  long long per = ((p.step ? (long long)p.blocks * p.tiles : p.all) * kv_count + at_once - 1) / at_once;
  a.part_row0 = 0;
  // One step workgroup a CU where it then has four blocks at most and partials are
  // many and wide: five lanes at 16000, 512-dim heads 16.4 + 4.7 -> 16.2 + 4.1 us,
  // eight 17.7 + 6.2 -> 18.7 + 4.4, five of four 256-dim at 4000 11.8 -> 10.3; but of
  // 64-dim heads 6.0 -> 6.7, and twelve lanes, six blocks, 22.6 + 5.0 -> 24.2 + 4.0.
  if (p.step && !p.pair && head >= 256) {
    const long long one = ((long long)p.blocks * p.tiles * kv_count + cus - 1) / cus;
    if (one <= 4) per = one;
  }
  if (!p.step && (a.window > 0 || 4 * attend4_tile_blocks(p, 0, a) > 3 * p.blocks)) {
    // Tiles alike: the cheapest number of whole turns of the card, a workgroup's start
    // and end taken for one block and a share of 2^20 partial floats for another
    // (160 lanes at 15000, 512-dim heads: 13 segments of 20 tiles, two turns, 165 us;
    // 12, one turn, 117).
    double least = 0.0;
    for (int n = 1; n <= p.blocks && n <= kAttend4Segments; ++n) {
      const long long size = (p.blocks + n - 1) / n, used = (p.blocks + size - 1) / size;
      if (used > 1 && floats(used) > room) break;
      const double cost = (double)((used * p.tiles * kv_count + cus - 1) / cus) * (double)(size + 1) +
                          (used > 1 ? 1.0 + (double)floats(used) / (1 << 20) : 0.0);
      if (n == 1 || cost < least) least = cost, per = size;
    }
  }
  for (;;) {
    if (per < per_least) per = per_least;
    if (per < 1) per = 1;
    if (per > p.blocks) per = p.blocks;
    a.per = (int)per;
    a.segments = (int)((p.blocks + per - 1) / per);
    if (a.segments == 1) break;
    if (!p.step && a.window == 0) {  // only the rows of more blocks than a share
      int low = 0, high = p.tiles - 1;  // the first tile of more
      while (low < high) {
        const int mid = (low + high) / 2;
        if (attend4_tile_blocks(p, mid, a) > per)
          high = mid;
        else
          low = mid + 1;
      }
      a.part_row0 = low * p.each;
    }
    if (floats(a.segments) <= room) break;
    per += (per + 7) / 8;
  }
  return p;
}

template <int HEAD, int FMT>
static hipError_t attend4_launch(const Attend4Args &a, const Attend4Plan &p, int kv_count, hipStream_t stream) {
  constexpr int T = HEAD >= 256 ? 1 : 2;
  const dim3 grid(p.tiles, a.segments, kv_count);
  if (!p.step) {
    if constexpr (HEAD >= 128) {
      constexpr int size = Tile4Shape<HEAD>::LDS;
      static_assert(size > 65536 && size <= 163840, "a granted size");
      const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(&attend4_tile_kernel<HEAD, FMT>),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, size);  // again: no change
      if (e != hipSuccess) return e;
      hipLaunchKernelGGL((attend4_tile_kernel<HEAD, FMT>), grid, dim3(512), (size_t)size, stream, a);
    }
  } else if (p.deep) {
    if constexpr (HEAD < 256) {
      if (p.deep == 4)
        hipLaunchKernelGGL((attend4_step_kernel<HEAD, FMT, true, 4 * T>), grid, dim3(256), 0, stream, a);
      else
        hipLaunchKernelGGL((attend4_step_kernel<HEAD, FMT, true, 2 * T>), grid, dim3(256), 0, stream, a);
    }
  } else if (p.pair) {
    hipLaunchKernelGGL((attend4_step_kernel<HEAD, FMT, true, T>), grid, dim3(256), 0, stream, a);
  } else {
    hipLaunchKernelGGL((attend4_step_kernel<HEAD, FMT, false, T>), grid, dim3(256), 0, stream, a);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.segments == 1) return e;
  const int rows = a.rows - a.part_row0, dims = rows <= 64 ? 16 : rows <= 1024 ? 64 : HEAD;
  const dim3 fgrid(rows, kv_count, HEAD / dims);
  if (dims == 16)
    hipLaunchKernelGGL((attend4_fold_kernel<16>), fgrid, dim3(256), 0, stream, a, HEAD);
  else if (dims == 64)
    hipLaunchKernelGGL((attend4_fold_kernel<64>), fgrid, dim3(256), 0, stream, a, HEAD);
  else
    hipLaunchKernelGGL((attend4_fold_kernel<HEAD>), fgrid, dim3(256), 0, stream, a, HEAD);
  return hipGetLastError();
}

template <int HEAD>
static hipError_t attend4_launch_format(const Attend4Args &a, const Attend4Plan &p, int format, int kv_count,
                                        hipStream_t stream) {
  if (format == IGL_CACHE4_INT4) return attend4_launch<HEAD, IGL_CACHE4_INT4>(a, p, kv_count, stream);
  return attend4_launch<HEAD, IGL_CACHE4_E2M1>(a, p, kv_count, stream);
}

static Attend4Args attend4_args(const igl_cache4 *store, int group_share, const float *query, int lane_stride,
                                int place_first, int window, int lanes, float score_scale, float *blend_out) {
  Attend4Args a = {};
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
  a.rows = lanes * group_share;
  // rows below 2^31: a multiplier that is less than share / 2^shift too large, 2^shift >= 2^31 share
  a.share_shift = 31;
  while ((1 << (a.share_shift - 31)) < group_share) ++a.share_shift;
  a.share_mul = (uint32_t)(((1ull << a.share_shift) + group_share - 1) / group_share);
  // log2 e, and the 256 that a gain is divided by
  const double factor = (double)store->key_scale * score_scale * 1.4426950408889634 * 256.0;
  a.key_part = isfinite(factor) ? (float)frexp(factor, &a.key_power) : NAN;
  a.value_scale = store->value_scale;
  return a;
}

extern "C" hipError_t igl_launch_attend4(const igl_cache4 *store, int group_share, const float *query, int lane_stride,
                                         int place_first, int window, int lanes, float score_scale, float *blend_out,
                                         float *work, hipStream_t stream) {
  Attend4Args a =
      attend4_args(store, group_share, query, lane_stride, place_first, window, lanes, score_scale, blend_out);
  const Attend4Plan p = attend4_plan(a, store->head_size, store->kv_count, work ? IGL_ATTEND4_FLOATS : 0);
  if (a.segments > 1) {
    const size_t parts = (size_t)a.segments * store->kv_count * (size_t)(a.rows - a.part_row0);
    a.part_out = work;
    a.part_base = work + parts * store->head_size;
    a.part_total = a.part_base + parts;
  }
  switch (store->head_size) {
    case 64: return attend4_launch_format<64>(a, p, store->format, store->kv_count, stream);
    case 128: return attend4_launch_format<128>(a, p, store->format, store->kv_count, stream);
    case 256: return attend4_launch_format<256>(a, p, store->format, store->kv_count, stream);
    case 512: return attend4_launch_format<512>(a, p, store->format, store->kv_count, stream);
    default: return hipErrorInvalidValue;
  }
}
