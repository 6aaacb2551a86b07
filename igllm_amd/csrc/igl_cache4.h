// igl_cache4.h - the 4-bit key/value ring: its slots, its codes, and the
// kernels that lay rows into it and read them back, gfx950.
//
// Every 32 values x of a head share a gain g, an e4m3 byte b, and a layer's
// side a scale s:
//     b = e4m3(amax |x| / (top s)),  level = nearest(x / (real8(b) s)),
//     value = level real8(b) s
// with top 7 (INT4: levels -7 .. 7, code level + 8) or 6 (E2M1).  A level has
// at most 4 significant bits and an e4m3 value 4, so level * g is exact in
// binary16 and fp32, and a reader rounds once, by the scale.
//
// Both decisions are those of real arithmetic: the quotients are formed in
// double, where a 24-bit x over a 28-bit step (or over the 27-bit top s) lies
// further from a border than the quotient's rounding unless it lies on it.
#pragma once

#include "igl_device.h"
#include "igl_launch.h"

namespace igl {

constexpr int kCache4Group = 32;  // values that share a gain
constexpr int kCache4Block = 64;  // slots the gain rows are padded to

// real8 of a gain byte: e4m3 as the byte ring reads it (0x7F 480, no NaN).
__device__ __forceinline__ float cache4_gain(uint32_t byte) {
  const uint32_t h = ((byte + (byte & 0x80u)) << 7) & 0xFFFFu;  // binary16 of real8 / 256
  return (float)__builtin_bit_cast(_Float16, (uint16_t)h) * 256.0f;
}

// The level a code stands for.
template <int FMT>
__device__ __forceinline__ float cache4_level(uint32_t code) {
  if (FMT == IGL_CACHE4_INT4) return (float)((int)code - 8);
  const uint32_t h = ((code & 8u) << 12) | ((code & 7u) << 9);  // binary16 of level / 2^14
  return (float)__builtin_bit_cast(_Float16, (uint16_t)h) * 16384.0f;
}

// The slot of a position (cache4's ring with its first positions kept).
__host__ __device__ __forceinline__ int cache4_slot(int place, int sinks, int span) {
  return place < sinks ? place : sinks + (place - sinks) % (span - sinks);
}

// e4m3 byte of a quotient >= 0 (or infinite): nearest, ties to even, 448 at most.
__device__ __forceinline__ uint32_t cache4_gain_byte(double q) {
  if (!(q < 448.0)) return 0x7Eu;
  if (q < 0.015625) return (uint32_t)__builtin_rint(q * 512.0);  // 2^-9 steps; 8 is 2^-6's byte
  uint64_t u = __builtin_bit_cast(uint64_t, q);
  u += 0xFFFFFFFFFFFFull + ((u >> 49) & 1u);  // to three bits of mantissa
  return (uint32_t)(u >> 49) - (1016u << 3);
}

// The level index of |q| = |x| / step, in single precision or exactly: INT4 q
// itself; E2M1 2 q below 2, 2 + q below 4, 4 + q / 2 from there (its tables' steps
// are 1/2, 1 and 2), to the nearest whole number, ties to even.
template <int FMT, typename F>
__device__ __forceinline__ F cache4_index(F q) {
  if (FMT == IGL_CACHE4_INT4) return q;
  return q < (F)2 ? (F)2 * q : q < (F)4 ? (F)2 + q : (F)4 + (F)0.5 * q;
}

// What decides a group's codes: its step, real8(b) s, and in single precision the
// step's reciprocal (0 where a float does not hold it in full: then every code is
// decided exactly).
struct Cache4Step {
  double step;
  float inverse;
};

__device__ __forceinline__ Cache4Step cache4_step(double step) {
  const bool held = step > 1e-30 && step < 1e30;
  return Cache4Step{step, held ? 1.0f / (float)step : 0.0f};
}

// The code of x; x NaN or step 0: zero.  The single-precision index is off by less
// than 2^-20 of itself, at most 14 where it counts, so it decides unless it lies
// within 2^-15 of halfway; there the exact quotient does.
template <int FMT>
__device__ __forceinline__ uint32_t cache4_code(float x, const Cache4Step &t) {
  const float m = fabsf(x);
  const float at = cache4_index<FMT>(m * t.inverse);
  float index = __builtin_rintf(at);
  if (!(fabsf(at - index) < 0.5f - 3.1e-5f) || t.inverse == 0.0f) {  // and a NaN, an infinity, a number past 2^23
    if (at <= 16.0f || t.inverse == 0.0f) {
      double exact = t.step > 0.0 ? cache4_index<FMT, double>((double)m / t.step) : 0.0;
      exact = __builtin_rint(exact);
      index = exact < 7.0 ? (float)exact : 7.0f;
    }
  }
  if (!(index <= 7.0f)) index = 7.0f;
  const uint32_t level = m == m ? (uint32_t)index : 0u;
  if (FMT == IGL_CACHE4_INT4) return x < 0.0f ? 8u - level : 8u + level;
  return level && x < 0.0f ? level | 8u : level;
}

// Four floats at any address of a float: rows need no alignment.
typedef float float4a_t __attribute__((ext_vector_type(4), aligned(4)));

struct Cache4Args {
  uint8_t *code[2];    // key, value: [span][width / 2]
  uint8_t *gain[2];    // [width / 32][room]
  float scale[2];
  const float *in[2];  // rows to lay
  float *out[2];       // rows to read, or NULL
  long long room;      // slots a gain row holds
  int width;           // values a row
  int span, sinks;
  int row_stride;
  int place;
  int lanes;
};

// A thread eight values, a dword of codes, and four threads a group, whose largest
// value meets by two lane moves; blockIdx.y the side.  Streams: 16384 rows of 1024
// values a side, 152 MB, in 31.4 us, 4.9 TB/s (a large copy: 5.0); 41.8 with every
// code decided by a division in double.  A step's row takes 2.8, its launch.
template <int FMT>
__global__ __launch_bounds__(256) void cache4_lay_kernel(Cache4Args a) {
  const int per = a.width / 8;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  const int lane = (int)(i / per);
  if (lane >= a.lanes) return;  // whole groups: `per` is a multiple of eight
  const int d0 = 8 * (int)(i - (long long)lane * per);
  const int side = blockIdx.y;
  const float *src = a.in[side] + (size_t)lane * a.row_stride + d0;
  const float4_t u = *reinterpret_cast<const float4a_t *>(src), v = *reinterpret_cast<const float4a_t *>(src + 4);
  const float x[8] = {u[0], u[1], u[2], u[3], v[0], v[1], v[2], v[3]};
  float top = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[e]));  // a NaN is passed over
  top = fmaxf(top, dpp_move<0xB1>(top));
  top = fmaxf(top, dpp_move<0x4E>(top));
  const double scale = (double)a.scale[side];
  const uint32_t byte = cache4_gain_byte((double)top / ((FMT == IGL_CACHE4_INT4 ? 7.0 : 6.0) * scale));
  const Cache4Step step = cache4_step((double)cache4_gain(byte) * scale);
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) w |= cache4_code<FMT>(x[e], step) << (4 * e);
  const size_t slot = (size_t)cache4_slot(a.place + lane, a.sinks, a.span);
  *reinterpret_cast<uint32_t *>(a.code[side] + slot * (size_t)(a.width / 2) + d0 / 2) = w;
  if ((threadIdx.x & 3) == 0) a.gain[side][(size_t)(d0 / kCache4Group) * a.room + slot] = (uint8_t)byte;
}

// A thread eight values; blockIdx.y the side (one where only one is wanted).
// Streams: 131071 rows of 512 values a side, 608 MB, in 137 us, 4.5 TB/s, seven in
// eight of them written.
template <int FMT>
__global__ __launch_bounds__(256) void cache4_read_kernel(Cache4Args a, int side0) {
  const int per = a.width / 8;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  const int lane = (int)(i / per);
  if (lane >= a.lanes) return;
  const int d0 = 8 * (int)(i - (long long)lane * per);
  const int side = side0 + blockIdx.y;
  const size_t slot = (size_t)cache4_slot(a.place + lane, a.sinks, a.span);
  const uint32_t w = *reinterpret_cast<const uint32_t *>(a.code[side] + slot * (size_t)(a.width / 2) + d0 / 2);
  const float gain = cache4_gain(a.gain[side][(size_t)(d0 / kCache4Group) * a.room + slot]);
  const float scale = a.scale[side];
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = cache4_level<FMT>((w >> (4 * e)) & 15u) * gain * scale;
  float *dst = a.out[side] + (size_t)lane * a.row_stride + d0;
  *reinterpret_cast<float4a_t *>(dst) = float4_t{y[0], y[1], y[2], y[3]};
  *reinterpret_cast<float4a_t *>(dst + 4) = float4_t{y[4], y[5], y[6], y[7]};
}

}  // namespace igl
