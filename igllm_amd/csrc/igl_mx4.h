// igl_mx4.h - microscaled 4-bit rows (MX, e2m1 codes under a power of two every 32
// values): rows put into the form and read back, and products with them, gfx950.
//
// Every 32 values x of a row share a byte b; a value is level * 2^(b - 127), its
// level one of 0, 1/2, 1, 3/2, 2, 3, 4, 6 or their negatives.  Written rows take
//     b = floor(log2(max |x|)) - 2 + 127 (0 at least),
//     level = nearest(x / 2^(b - 127)), ties to the even code, 6 at most.
// A power of two changes no digits, so single precision decides both exactly.
//
// The product takes the codes as they lie: the scaled matrix instruction reads
// e2m1 operands with a scale byte for every 32 of them.  Its other operand is the
// lanes, microscaled rows as they lie too, or floats cut into terms:
//     x = 2^(s - 127) (t_0 + t_1 / 32 + t_2 / 32^2 + ..),
// s a byte for the group, t_j e2m3 numbers.  The group's largest is at most 3.75
// under its scale, so t_0 is off by 1/8 at most, thirty-two times what is left is 4
// at most, off by 1/8 again, and so on: T terms hold a value to 2^(-3 - 5 (T - 1))
// where the group's largest is more than 1.875, so to 2^(1 - 5 T) of the largest:
// 2^-24 with five (fp32 lanes), 2^-14 with three (bf16 lanes, whose outputs are
// rounded to 2^-8).  e2m3 against e2m1 runs at twice e4m3's rate (8.8 to 4.7
// PFLOP/s, all of a card's SIMDs), so five terms are 1.8 PFLOP/s of fp32 lanes and
// three 2.9 of bf16 ones, and no code is ever decoded.
#pragma once

#include "igl_device.h"
#include "igl_launch.h"

namespace igl {

typedef int int8v_t __attribute__((ext_vector_type(8)));
typedef uint32_t uint6_t __attribute__((ext_vector_type(6)));
typedef float float32_t __attribute__((ext_vector_type(32)));

constexpr int kMx4Group = 32;

// ---- rows ---------------------------------------------------------------------

struct __attribute__((packed)) Mx4Quad {
  float v[4];
};
struct __attribute__((packed)) Mx4Half8 {
  uint16_t v[8];
};

__device__ __forceinline__ float bf16_float(uint16_t b) { return __builtin_bit_cast(float, (uint32_t)b << 16); }

// bf16 of a float, nearest, ties to even; a NaN stays one.
__device__ __forceinline__ uint16_t float_bf16(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  if ((u & 0x7FFFFFFFu) > 0x7F800000u) return (uint16_t)((u >> 16) | 0x40u);
  return (uint16_t)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
}

// Eight values of a row, at any alignment that their type allows.
template <bool BF16>
__device__ __forceinline__ void mx4_load8(const void *row, size_t at, float (&x)[8]) {
  if (BF16) {
    const Mx4Half8 h = *reinterpret_cast<const Mx4Half8 *>(static_cast<const uint16_t *>(row) + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = bf16_float(h.v[i]);
  } else {
    const float *p = static_cast<const float *>(row) + at;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const Mx4Quad f = *reinterpret_cast<const Mx4Quad *>(p + 4 * q);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * q + i] = f.v[i];
    }
  }
}

// The bits of a magnitude order as it does; infinities and NaNs lie above all.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7FFFFFFFu; }

constexpr uint32_t kInfBits = 0x7F800000u;

// One thread for eight values, four threads a group: loads and stores stay whole
// and neighbouring.
template <bool BF16>
__global__ __launch_bounds__(256) void mx4_lay_kernel(const void *src, long long src_stride, int eighths, int rows,
                                                      uint8_t *code, size_t code_stride, uint8_t *scale,
                                                      size_t scale_stride) {
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long row = id / eighths;
  const int at = (int)(id - row * eighths);
  if (row >= rows) return;  // a group's four threads leave or stay together: eighths is a multiple of four
  float x[8];
  mx4_load8<BF16>(static_cast<const uint8_t *>(src) + (size_t)row * (size_t)src_stride * (BF16 ? 2 : 4), 8 * (size_t)at,
                  x);
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, abs_bits(x[i]));
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xF, 0xF, true));  // quad_perm [1,0,3,2]
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xF, 0xF, true));  // quad_perm [2,3,0,1]
  // floor(log2) of a float's magnitude: its exponent field; below 2^-125 the byte is 0
  const int field = (int)(top >> 23);
  const int byte = top >= kInfBits ? 255 : max(field - 2, 0);
  uint32_t codes = 0;
  if (byte != 255) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float m = __builtin_ldexpf(fabsf(x[i]), 127 - byte);
      // steps of 1/2, 1 and 2; m times a power of two is rounded, not a sum that has lost m's last digit
      const float index = m < 2.0f   ? __builtin_rintf(2.0f * m)
                          : m < 4.0f ? 2.0f + __builtin_rintf(m)
                                     : 4.0f + __builtin_rintf(0.5f * m);
      const uint32_t level = (uint32_t)fminf(index, 7.0f);
      codes |= (level | (__builtin_bit_cast(uint32_t, x[i]) >> 31 << 3)) << (4 * i);
    }
  }
  *reinterpret_cast<uint32_t *>(code + (size_t)row * code_stride + 4 * (size_t)at) = codes;
  if ((at & 3) == 0) scale[(size_t)row * scale_stride + (at >> 2)] = (uint8_t)byte;
}

// Eight values a thread.  A level times its power of two is exact (a NaN scale gives NaN); rounded to bf16
// none is lost either, but below 2^-126, where bf16's digits end.
template <bool BF16>
__global__ __launch_bounds__(256) void mx4_read_kernel(const uint8_t *code, size_t code_stride, const uint8_t *scale,
                                                       size_t scale_stride, int eighths, int rows, void *dst,
                                                       long long dst_stride) {
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long row = id / eighths;
  const int at = (int)(id - row * eighths);
  if (row >= rows) return;
  const uint32_t codes = *reinterpret_cast<const uint32_t *>(code + (size_t)row * code_stride + 4 * (size_t)at);
  const int byte = scale[(size_t)row * scale_stride + (at >> 2)];
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t c = codes >> (4 * i);
    // binary16 of level / 2^14: e2m1's fields at the bottom of its own
    const float level = (float)__builtin_bit_cast(_Float16, (uint16_t)(((c & 8u) << 12) | ((c & 7u) << 9)));
    x[i] = byte == 255 ? __builtin_nanf("") : __builtin_ldexpf(level, byte - 127 + 14);
  }
  uint8_t *out = static_cast<uint8_t *>(dst) + ((size_t)row * (size_t)dst_stride + 8 * (size_t)at) * (BF16 ? 2 : 4);
  if (BF16) {
    Mx4Half8 h;
#pragma unroll
    for (int i = 0; i < 8; ++i) h.v[i] = float_bf16(x[i]);
    *reinterpret_cast<Mx4Half8 *>(out) = h;
  } else {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      Mx4Quad f;
#pragma unroll
      for (int i = 0; i < 4; ++i) f.v[i] = x[4 * q + i];
      *reinterpret_cast<Mx4Quad *>(out + 16 * q) = f;
    }
  }
}

// ---- lanes of floats as terms ---------------------------------------------------

// A group of a lane in T terms: six dwords a term, then the scale bytes of the first
// four (s, s - 5, ..), and of the fifth; whole chunks of sixteen bytes.
template <int T>
struct TermForm {
  static constexpr int kDwords = T == 5 ? 32 : 20;
  static constexpr int kBytes = 4 * kDwords;
  static constexpr int kScale = 6 * T;  // the dword of the scales
  static_assert(6 * T + (T + 3) / 4 <= kDwords, "room");
};

// The terms of a group.  s is 20 at least, so that s - 5 j stays a byte (five terms
// then end at 2^-130, three at 2^-120); an infinity or a NaN makes the scale a NaN, so that
// every output of its lane is one.
template <int T>
__device__ __forceinline__ void mx4_terms(float (&x)[32], uint32_t (&rec)[TermForm<T>::kDwords]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) top = max(top, abs_bits(x[i]));
  int s = (int)(top >> 23) - ((top & 0x7FFFFFu) <= 0x700000u ? 1 : 0);  // top / 2^(s - 127) <= 3.75
  s = max(s, 20);
  const bool none = top >= kInfBits;
#pragma unroll
  for (int i = 0; i < 32; ++i) x[i] = none ? 0.0f : __builtin_ldexpf(x[i], 127 - s);
#pragma unroll
  for (int t = 0; t < T; ++t) {
    float16_t even, odd;  // the conversion takes a group's even and odd values apart
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      even[i] = x[2 * i];
      odd[i] = x[2 * i + 1];
    }
    const uint6_t w = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(even, odd, 1.0f);
#pragma unroll
    for (int i = 0; i < 6; ++i) rec[6 * t + i] = w[i];
    if (t + 1 < T) {
      const float32_t back = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(w, 32.0f);
#pragma unroll
      for (int i = 0; i < 32; ++i) x[i] = __builtin_fmaf(x[i], 32.0f, -back[i]);
    }
  }
  if (none) s = 255;
  rec[TermForm<T>::kScale] = (uint32_t)s * 0x01010101u - 0x0F0A0500u;
  if (T == 5) rec[TermForm<T>::kScale + 1] = (uint32_t)(s - 20);
#pragma unroll
  for (int i = TermForm<T>::kScale + (T + 3) / 4; i < TermForm<T>::kDwords; ++i) rec[i] = 0;
}

// The operand of term t of a record, and its scale.
template <int T>
__device__ __forceinline__ int8v_t term_operand(const uint32_t (&rec)[TermForm<T>::kDwords], int t) {
  return int8v_t{(int)rec[6 * t],     (int)rec[6 * t + 1], (int)rec[6 * t + 2], (int)rec[6 * t + 3],
                 (int)rec[6 * t + 4], (int)rec[6 * t + 5], 0,                   0};
}

// A thread a group: lanes of floats to records [lane][groups].
template <int T, bool BF16>
__global__ __launch_bounds__(256) void mx4_terms_kernel(const void *act, long long act_stride, int groups, int lanes,
                                                        uint32_t *terms) {
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long lane = id / groups;
  const int g = (int)(id - lane * groups);
  if (lane >= lanes) return;
  const void *row = static_cast<const uint8_t *>(act) + (size_t)lane * (size_t)act_stride * (BF16 ? 2 : 4);
  float x[32];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float part[8];
    mx4_load8<BF16>(row, 32 * (size_t)g + 8 * e, part);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[8 * e + i] = part[i];
  }
  uint32_t rec[TermForm<T>::kDwords];
  mx4_terms<T>(x, rec);
  uint4_t *dst = reinterpret_cast<uint4_t *>(terms + (size_t)id * TermForm<T>::kDwords);
#pragma unroll
  for (int i = 0; i < TermForm<T>::kDwords / 4; ++i)
    dst[i] = uint4_t{rec[4 * i], rec[4 * i + 1], rec[4 * i + 2], rec[4 * i + 3]};
}

// ---- the product ------------------------------------------------------------------

// Rows of a microscaled weight; in a batch of experts expert e's rows begin at
// row e * rows_each.
struct Mx4View {
  const uint8_t *code;
  size_t code_stride;
  const uint8_t *scale;
  size_t scale_stride;
};

// Which lanes a tile of a grouped product takes: places `first` .. first + count - 1
// of its expert's list.
struct Mx4Tile {
  int expert, first, count;
};

struct Mx4Args {
  Mx4View w;
  int rows, groups;         // rows of a sheet (an expert's), groups of a row
  const uint32_t *terms;    // records [lane][groups], lanes of floats
  Mx4View act;              // or microscaled lanes
  int lanes;
  // grouped: the tiles, how many there are, and the lane of every place (NULL: the place)
  const Mx4Tile *tiles;
  const int *tile_count;
  const int *lane_of;
  void *out;                // [lane or place][out_stride]
  long long out_stride;
};

// The codes and scale byte of group g of a row; behind the row's last group zeros.
__device__ __forceinline__ int8v_t mx4_group(const Mx4View &v, size_t row, int g, int groups, int &scale) {
  if (g >= groups) {
    scale = 0;
    return int8v_t{0, 0, 0, 0, 0, 0, 0, 0};
  }
  const uint4_t c = *reinterpret_cast<const uint4_t *>(v.code + row * v.code_stride + 16 * (size_t)g);
  scale = v.scale[row * v.scale_stride + g];
  return int8v_t{(int)c[0], (int)c[1], (int)c[2], (int)c[3], 0, 0, 0, 0};
}

// A wave takes 16 rows and 16 lanes, 128 columns a step: lane l of the wave holds
// group l / 16 of row and lane l % 16.  T terms, 0: microscaled lanes.
template <int T, bool OUT_BF16>
__global__ __launch_bounds__(256) void mx4_wave_kernel(Mx4Args g) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n0 = (blockIdx.x * 4 + wave) * 16;
  if (n0 >= g.rows) return;
  int first = blockIdx.y * 16, count = min(16, g.lanes - first);
  size_t row0 = 0;
  if (g.tiles) {
    if ((int)blockIdx.y >= *g.tile_count) return;
    const Mx4Tile t = g.tiles[blockIdx.y];
    first = t.first;
    count = t.count;
    row0 = (size_t)t.expert * (size_t)g.rows;
  }
  const int part = lane >> 4, at = lane & 15;
  const size_t row = row0 + (size_t)min(n0 + at, g.rows - 1);
  const int place = first + min(at, count - 1);
  const size_t from = (size_t)(g.lane_of ? g.lane_of[place] : place);
  float4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int g0 = 0; g0 < g.groups; g0 += 4) {
    int ws, as;
    const int8v_t w = mx4_group(g.w, row, g0 + part, g.groups, ws);
    if constexpr (T == 0) {
      const int8v_t a = mx4_group(g.act, from, g0 + part, g.groups, as);
      acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, acc, 4, 4, 0, ws, 0, as);
    } else {
      uint32_t rec[TermForm<T>::kDwords];
      const uint4_t *src = reinterpret_cast<const uint4_t *>(
          g.terms + (from * (size_t)g.groups + (size_t)min(g0 + part, g.groups - 1)) * TermForm<T>::kDwords);
#pragma unroll
      for (int i = 0; i < TermForm<T>::kDwords / 4; ++i) {
        const uint4_t c = g0 + part < g.groups ? src[i] : uint4_t{0, 0, 0, 0};
        rec[4 * i] = c[0], rec[4 * i + 1] = c[1], rec[4 * i + 2] = c[2], rec[4 * i + 3] = c[3];
      }
#pragma unroll
      for (int t = 0; t < T; ++t) {
        as = t < 4 ? (int)(rec[TermForm<T>::kScale] >> (8 * t)) : (int)rec[TermForm<T>::kScale + 1];
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, term_operand<T>(rec, t), acc, 4, 2, 0, ws, 0, as);
      }
    }
  }
  // the weight is the first operand: this wave lane holds rows 4 (l / 16) .. + 3 of lane l % 16
  if (at >= count) return;
  const size_t out = (size_t)(first + at) * (size_t)g.out_stride;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int n = n0 + 4 * part + r;
    if (n >= g.rows) continue;
    if (OUT_BF16)
      static_cast<uint16_t *>(g.out)[out + n] = float_bf16(acc[r]);
    else
      static_cast<float *>(g.out)[out + n] = acc[r];
  }
}

// ---- the experts' feed-forward ------------------------------------------------------

// Places: the slots (lane, choice) in the order of their experts.  One workgroup
// counts them, sets every expert's range and tiles, and lists the slots; a slot whose
// expert is none (out of range) has no place.
constexpr int kPlaceThreads = 1024;

struct PlaceArgs {
  const int32_t *pick;
  int slots, top, experts, tile;  // places a tile
  int *lane_of;                   // [slots] lane of a place
  int *place_of;                  // [slots] place of a slot, or -1
  Mx4Tile *tiles;
  int *tile_count;
  int *count;                     // [experts] scratch
};

__global__ __launch_bounds__(kPlaceThreads) void expert_place_kernel(PlaceArgs a) {
  for (int e = threadIdx.x; e < a.experts; e += kPlaceThreads) a.count[e] = 0;
  __syncthreads();
  for (int s = threadIdx.x; s < a.slots; s += kPlaceThreads) {
    const int e = a.pick[s];
    if (e >= 0 && e < a.experts) atomicAdd(&a.count[e], 1);
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int place = 0, tile = 0;
    for (int e = 0; e < a.experts; ++e) {
      const int n = a.count[e];
      a.count[e] = place;
      for (int i = 0; i < n; i += a.tile) a.tiles[tile++] = Mx4Tile{e, place + i, min(a.tile, n - i)};
      place += n;
    }
    *a.tile_count = tile;
  }
  __syncthreads();
  for (int s = threadIdx.x; s < a.slots; s += kPlaceThreads) {
    const int e = a.pick[s];
    int place = -1;
    if (e >= 0 && e < a.experts) {
      place = atomicAdd(&a.count[e], 1);
      a.lane_of[place] = s / a.top;
    }
    a.place_of[s] = place;
  }
}

// silu(x) = x / (1 + e^-x)
__device__ __forceinline__ float silu_near(float x) {
  if (!(x > -87.0f)) return x * 0.0f;
  return x / (1.0f + exp_near(x > 87.0f ? -87.0f : -x));
}

// gate(g) * u of gate_up rows [place][2 inner] -> [place][inner]
__global__ __launch_bounds__(256) void expert_gate_kernel(const float *both, int inner, int places, int silu, float *h) {
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long place = id / inner;
  if (place >= places) return;
  const int n = (int)(id - place * inner);
  const float g = both[(size_t)place * 2 * inner + n], u = both[(size_t)place * 2 * inner + inner + n];
  h[id] = (silu ? silu_near(g) : gelu_near(g)) * u;
}

// out[lane] = sum over its choices, in their order, of weight * row of the slot's place
template <bool BF16>
__global__ __launch_bounds__(256) void expert_join_kernel(const float *rows, const int *place_of, const float *weight,
                                                          int top, int hidden, int lanes, void *out, long long out_stride) {
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long lane = id / hidden;
  if (lane >= lanes) return;
  const int n = (int)(id - lane * hidden);
  float sum = 0.0f;
  for (int j = 0; j < top; ++j) {
    const int place = place_of[lane * top + j];
    if (place >= 0) sum = __builtin_fmaf(weight[lane * top + j], rows[(size_t)place * hidden + n], sum);
  }
  if (BF16)
    static_cast<uint16_t *>(out)[(size_t)lane * out_stride + n] = float_bf16(sum);
  else
    static_cast<float *>(out)[(size_t)lane * out_stride + n] = sum;
}

}  // namespace igl

// ---- launchers ----------------------------------------------------------------------

using namespace igl;

static Mx4View mx4_view(const igl_mx4 *s, int row_first) {
  return Mx4View{s->code + (size_t)row_first * s->code_stride, s->code_stride,
                 s->scale + (size_t)row_first * s->scale_stride, s->scale_stride};
}

extern "C" hipError_t igl_launch_mx4_lay(const igl_mx4 *store, int row_first, int rows, const void *src, int bf16,
                                         int src_stride, hipStream_t stream) {
  const Mx4View v = mx4_view(store, row_first);
  const int eighths = store->col_count / 8;
  const unsigned blocks = (unsigned)(((long long)rows * eighths + 255) / 256);
  if (bf16)
    hipLaunchKernelGGL((mx4_lay_kernel<true>), dim3(blocks), dim3(256), 0, stream, src, src_stride, eighths, rows,
                       (uint8_t *)v.code, v.code_stride, (uint8_t *)v.scale, v.scale_stride);
  else
    hipLaunchKernelGGL((mx4_lay_kernel<false>), dim3(blocks), dim3(256), 0, stream, src, src_stride, eighths, rows,
                       (uint8_t *)v.code, v.code_stride, (uint8_t *)v.scale, v.scale_stride);
  return hipGetLastError();
}

extern "C" hipError_t igl_launch_mx4_read(const igl_mx4 *store, int row_first, int rows, void *dst, int bf16,
                                          int dst_stride, hipStream_t stream) {
  const Mx4View v = mx4_view(store, row_first);
  const int eighths = store->col_count / 8;
  const unsigned blocks = (unsigned)(((long long)rows * eighths + 255) / 256);
  if (bf16)
    hipLaunchKernelGGL((mx4_read_kernel<true>), dim3(blocks), dim3(256), 0, stream, v.code, v.code_stride, v.scale,
                       v.scale_stride, eighths, rows, dst, dst_stride);
  else
    hipLaunchKernelGGL((mx4_read_kernel<false>), dim3(blocks), dim3(256), 0, stream, v.code, v.code_stride, v.scale,
                       v.scale_stride, eighths, rows, dst, dst_stride);
  return hipGetLastError();
}

static size_t mx4_up(size_t bytes) { return (bytes + 255) & ~(size_t)255; }

static size_t terms_bytes(int lanes, int cols, int bf16) {
  return mx4_up((size_t)lanes * (cols / kMx4Group) * (bf16 ? TermForm<3>::kBytes : TermForm<5>::kBytes));
}

static hipError_t launch_terms(const void *act, int bf16, long long act_stride, int lanes, int cols, uint32_t *terms,
                               hipStream_t stream) {
  const int groups = cols / kMx4Group;
  const unsigned blocks = (unsigned)(((long long)lanes * groups + 255) / 256);
  if (bf16)
    hipLaunchKernelGGL((mx4_terms_kernel<3, true>), dim3(blocks), dim3(256), 0, stream, act, act_stride, groups, lanes,
                       terms);
  else
    hipLaunchKernelGGL((mx4_terms_kernel<5, false>), dim3(blocks), dim3(256), 0, stream, act, act_stride, groups, lanes,
                       terms);
  return hipGetLastError();
}

// tiles: lane tiles of the grid.  terms 0: microscaled lanes.
static hipError_t launch_product(const Mx4Args &a, int terms, int out_bf16, int tiles, hipStream_t stream) {
  const dim3 grid((a.rows + 63) / 64, tiles);
  if (terms == 0 && out_bf16)
    hipLaunchKernelGGL((mx4_wave_kernel<0, true>), grid, dim3(256), 0, stream, a);
  else if (terms == 0)
    hipLaunchKernelGGL((mx4_wave_kernel<0, false>), grid, dim3(256), 0, stream, a);
  else if (terms == 3 && out_bf16)
    hipLaunchKernelGGL((mx4_wave_kernel<3, true>), grid, dim3(256), 0, stream, a);
  else if (terms == 3)
    hipLaunchKernelGGL((mx4_wave_kernel<3, false>), grid, dim3(256), 0, stream, a);
  else if (out_bf16)
    hipLaunchKernelGGL((mx4_wave_kernel<5, true>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((mx4_wave_kernel<5, false>), grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}

extern "C" size_t igl_mx4_work_bytes(int rows, int cols, int lanes, int act_bf16) {
  (void)rows;
  return terms_bytes(lanes, cols, act_bf16);
}

extern "C" hipError_t igl_launch_mx4_mat_mat(const igl_mx4 *sheet, const void *act, int act_bf16, int act_stride,
                                             int lanes, void *out, int out_bf16, int out_stride, void *work,
                                             hipStream_t stream) {
  const hipError_t e =
      launch_terms(act, act_bf16, act_stride, lanes, sheet->col_count, static_cast<uint32_t *>(work), stream);
  if (e != hipSuccess) return e;
  Mx4Args a = {};
  a.w = mx4_view(sheet, 0);
  a.rows = sheet->row_count;
  a.groups = sheet->col_count / kMx4Group;
  a.terms = static_cast<const uint32_t *>(work);
  a.lanes = lanes;
  a.out = out;
  a.out_stride = out_stride;
  return launch_product(a, act_bf16 ? 3 : 5, out_bf16, (lanes + 15) / 16, stream);
}

extern "C" hipError_t igl_launch_mx4_mat_mx4(const igl_mx4 *sheet, const igl_mx4 *act, int lane_first, int lanes,
                                             void *out, int out_bf16, int out_stride, hipStream_t stream) {
  Mx4Args a = {};
  a.w = mx4_view(sheet, 0);
  a.rows = sheet->row_count;
  a.groups = sheet->col_count / kMx4Group;
  a.act = mx4_view(act, lane_first);
  a.lanes = lanes;
  a.out = out;
  a.out_stride = out_stride;
  return launch_product(a, 0, out_bf16, (lanes + 15) / 16, stream);
}

namespace igl {

// The places of a call's experts, its intermediate rows and their terms.
struct ExpertRoom {
  size_t lane_of, place_of, tiles, tile_count, count, x, both, h, h_terms, rows, end;
};

static int expert_tiles(int slots, int experts, int tile) {
  return slots / tile + (slots < experts ? slots : experts);
}

static ExpertRoom expert_room(const igl_experts *x, int lanes, int top, int bf16) {
  const size_t slots = (size_t)lanes * top;
  ExpertRoom r;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += mx4_up(bytes);
    return here;
  };
  r.lane_of = take(slots * sizeof(int));
  r.place_of = take(slots * sizeof(int));
  r.tiles = take((size_t)expert_tiles((int)slots, x->expert_count, 16) * sizeof(Mx4Tile));
  r.tile_count = take(sizeof(int));
  r.count = take((size_t)x->expert_count * sizeof(int));
  r.x = take(terms_bytes(lanes, x->hidden, bf16));
  r.both = take(slots * 2 * x->inner * sizeof(float));
  r.h = take(slots * x->inner * sizeof(float));
  r.h_terms = take(terms_bytes((int)slots, x->inner, 0));
  r.rows = take(slots * x->hidden * sizeof(float));
  r.end = at;
  return r;
}

}  // namespace igl

extern "C" size_t igl_experts_work_bytes(const igl_experts *x, int lanes, int top, int act_bf16) {
  return expert_room(x, lanes, top, act_bf16).end;
}

extern "C" hipError_t igl_launch_experts(const igl_experts *x, const void *act, int act_bf16, int act_stride, int lanes,
                                         const int32_t *pick, const float *weight, int top, void *out, int out_bf16,
                                         int out_stride, void *work, hipStream_t stream) {
  const ExpertRoom r = expert_room(x, lanes, top, act_bf16);
  uint8_t *base = static_cast<uint8_t *>(work);
  const int slots = lanes * top, tiles = expert_tiles(slots, x->expert_count, 16);
  hipError_t e;
  PlaceArgs p = {pick, slots, top, x->expert_count, 16, (int *)(base + r.lane_of), (int *)(base + r.place_of),
                 (Mx4Tile *)(base + r.tiles), (int *)(base + r.tile_count), (int *)(base + r.count)};
  hipLaunchKernelGGL(expert_place_kernel, dim3(1), dim3(kPlaceThreads), 0, stream, p);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  if ((e = launch_terms(act, act_bf16, act_stride, lanes, x->hidden, (uint32_t *)(base + r.x), stream)) != hipSuccess)
    return e;
  Mx4Args a = {};
  a.w = mx4_view(&x->gate_up, 0);
  a.rows = 2 * x->inner;
  a.groups = x->hidden / kMx4Group;
  a.terms = (const uint32_t *)(base + r.x);
  a.tiles = p.tiles;
  a.tile_count = p.tile_count;
  a.lane_of = p.lane_of;
  a.out = base + r.both;
  a.out_stride = 2 * x->inner;
  if ((e = launch_product(a, act_bf16 ? 3 : 5, 0, tiles, stream)) != hipSuccess) return e;
  hipLaunchKernelGGL(expert_gate_kernel, dim3((unsigned)(((long long)slots * x->inner + 255) / 256)), dim3(256), 0,
                     stream, (const float *)(base + r.both), x->inner, slots, x->gate == IGL_GATE_SILU,
                     (float *)(base + r.h));
  if ((e = hipGetLastError()) != hipSuccess) return e;
  if ((e = launch_terms(base + r.h, 0, x->inner, slots, x->inner, (uint32_t *)(base + r.h_terms), stream)) != hipSuccess)
    return e;
  a.w = mx4_view(&x->down, 0);
  a.rows = x->hidden;
  a.groups = x->inner / kMx4Group;
  a.terms = (const uint32_t *)(base + r.h_terms);
  a.lane_of = nullptr;
  a.out = base + r.rows;
  a.out_stride = x->hidden;
  if ((e = launch_product(a, 5, 0, tiles, stream)) != hipSuccess) return e;
  const unsigned blocks = (unsigned)(((long long)lanes * x->hidden + 255) / 256);
  if (out_bf16)
    hipLaunchKernelGGL((expert_join_kernel<true>), dim3(blocks), dim3(256), 0, stream, (const float *)(base + r.rows),
                       p.place_of, weight, top, x->hidden, lanes, out, out_stride);
  else
    hipLaunchKernelGGL((expert_join_kernel<false>), dim3(blocks), dim3(256), 0, stream, (const float *)(base + r.rows),
                       p.place_of, weight, top, x->hidden, lanes, out, out_stride);
  return hipGetLastError();
}
