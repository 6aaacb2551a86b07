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
// of the group's scale, whose largest is more than 1.875: to 2^-23.9 of the largest with
// five, exactly if it has bf16's eight digits and is 2^-16 of the largest or more.  A term
// less would be 2^-18.9, where fp32 has 2^-24.  e2m3 against e2m1 runs at 8.8 PFLOP/s (all
// of a card's SIMDs), so five terms are 1.8.  e4m3 terms, of which two hold bf16's digits, run at 4.7,
// but an instruction of them keeps only 13 bits below its largest product; e2m3's products, and
// the groups' sums, are added in single precision.
//
// bf16 lanes in tiles need no terms: codes become bf16 numbers in registers, exactly,
// and products are bf16's (2.5 PFLOP/s of them), exact too and added in single precision.
#pragma once

#include "igl_device.h"
#include "igl_launch.h"

namespace igl {

typedef int int8v_t __attribute__((ext_vector_type(8)));
typedef uint32_t uint6_t __attribute__((ext_vector_type(6)));
typedef float float32_t __attribute__((ext_vector_type(32)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

constexpr int kMx4Group = 32;

// A step of a product is four groups of a row, one for each sixteen lanes of a wave
// (its parts); two steps are a cache line of codes, and steps are taken in pairs.
__host__ __device__ constexpr int mx4_steps(int groups) { return (groups + 7) / 8 * 2; }

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
  return __builtin_bit_cast(uint16_t, static_cast<__bf16>(x));
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

// Eight values a thread.  A level times its power of two is exact (a NaN scale gives NaN) below 2^128; rounded to
// bf16 none is lost either, but below 2^-126, where bf16's digits end.
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

// Four groups of a lane (a step of a product) in T terms of six dwords, as pieces of 64
// bytes, sixteen a group: the first four dwords of every term, then the last two, two terms'
// side by side; the scales as if a term's last two: the bytes of the first four terms
// (s, s - 5, ..) and of the fifth.  Two pieces of a lane lie side by side, a step's lanes
// behind each other, then the next two pieces (a last one of an odd count by itself): a
// cache looks up a line of 128 bytes as fast as half of one, and at that rate the tiles of
// a product are brought.
template <int T>
struct TermForm {
  static constexpr int kStep = T * 96 + 32;  // bytes: 512 of five
  static constexpr int kChunks = kStep / 64; // pieces
};

// bf16 lanes of a tile as they are, in T's place: piece c holds values 8 c .. 8 c + 7 of a group.
constexpr int kTerms = 5, kPlain = 16;
template <>
struct TermForm<kPlain> {
  static constexpr int kStep = 256;
  static constexpr int kChunks = kStep / 64;
};

// Where group `part` of piece c begins in a step of `lanes` lanes.
template <int T>
__host__ __device__ __forceinline__ size_t term_piece(size_t lane, size_t lanes, int c, int part) {
  constexpr int kChunks = TermForm<T>::kChunks;
  return (size_t)(c / 2) * lanes * 128 + (c + 1 < kChunks || c % 2 ? lane * 128 + 64 * (c % 2) : lane * 64) + 16 * part;
}

// The terms of a group.  s is 20 at least, so that s - 5 j stays a byte (five terms
// then end at 2^-130); an infinity or a NaN makes the scale a NaN, so that
// every output of its lane is one.
template <int T, typename Put, typename Scales>
__device__ __forceinline__ void mx4_cut(float (&x)[32], Put put, Scales scales) {
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
    put(t, w);
    if (t + 1 < T) {
      const float32_t back = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(w, 32.0f);
#pragma unroll
      for (int i = 0; i < 32; ++i) x[i] = __builtin_fmaf(x[i], 32.0f, -back[i]);
    }
  }
  if (none) s = 255;
  scales(uint2_t{(uint32_t)s * 0x01010101u - 0x0F0A0500u, (uint32_t)(s - 20)});
}

// A group's terms into its step.
template <int T>
__device__ __forceinline__ void mx4_terms(float (&x)[32], uint8_t *step, size_t lane, size_t lanes, int part) {
  uint2_t high[T + 1];
  mx4_cut<T>(
      x,
      [&](int t, const uint6_t &w) {
        *reinterpret_cast<uint4_t *>(step + term_piece<T>(lane, lanes, t, part)) = uint4_t{w[0], w[1], w[2], w[3]};
        high[t] = uint2_t{w[4], w[5]};
      },
      [&](const uint2_t &s) { high[T] = s; });
#pragma unroll
  for (int t = 0; t <= T; t += 2)
    *reinterpret_cast<uint4_t *>(step + term_piece<T>(lane, lanes, T + t / 2, part)) =
        uint4_t{high[t][0], high[t][1], high[t + 1][0], high[t + 1][1]};
}

// And into a record of its own, a term behind the other.
__device__ __forceinline__ void mx4_terms_record(float (&x)[32], uint8_t *record) {
  mx4_cut<kTerms>(
      x,
      [&](int t, const uint6_t &w) {
        uint2_t *to = reinterpret_cast<uint2_t *>(record + 24 * t);
        to[0] = uint2_t{w[0], w[1]};
        to[1] = uint2_t{w[2], w[3]};
        to[2] = uint2_t{w[4], w[5]};
      },
      [&](const uint2_t &s) { *reinterpret_cast<uint2_t *>(record + 24 * kTerms) = s; });
}

// The operand of term t of a group, and its scales.
template <int T>
__device__ __forceinline__ int8v_t term_operand(const uint8_t *step, size_t lane, size_t lanes, int t, int part) {
  const uint4_t a = *reinterpret_cast<const uint4_t *>(step + term_piece<T>(lane, lanes, t, part));
  const uint2_t b = *reinterpret_cast<const uint2_t *>(step + term_piece<T>(lane, lanes, T + t / 2, part) + 8 * (t % 2));
  return int8v_t{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], 0, 0};
}

template <int T>
__device__ __forceinline__ uint2_t term_scales(const uint8_t *step, size_t lane, size_t lanes, int part) {
  return *reinterpret_cast<const uint2_t *>(step + term_piece<T>(lane, lanes, T + T / 2, part) + 8);
}

// A group of bf16 values as pieces; an infinity or a NaN makes all of them NaNs, as it does terms.
__device__ __forceinline__ void mx4_plain(const uint16_t *row, bool in, uint8_t *step, size_t lane, size_t lanes, int part) {
  uint4_t v[4];
  bool none = false;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    Mx4Half8 h = {};
    if (in) h = *reinterpret_cast<const Mx4Half8 *>(row + 8 * c);
    v[c] = __builtin_bit_cast(uint4_t, h);
#pragma unroll
    for (int i = 0; i < 8; ++i) none |= (h.v[i] & 0x7F80u) == 0x7F80u;
  }
#pragma unroll
  for (int c = 0; c < 4; ++c)
    *reinterpret_cast<uint4_t *>(step + term_piece<kPlain>(lane, lanes, c, part)) =
        none ? uint4_t{0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u} : v[c];
}

// A thread for group id of the lanes' groups: floats to its terms, or bf16 numbers to pieces.
template <int T, bool BF16>
__device__ __forceinline__ void mx4_terms_group(const void *act, long long act_stride, int groups, int lanes,
                                                uint8_t *terms, long long id) {
  const int padded = 4 * mx4_steps(groups);
  const long long lane = id / padded;
  const int g = (int)(id - lane * padded);
  if (lane >= lanes) return;
  const void *row = static_cast<const uint8_t *>(act) + (size_t)lane * (size_t)act_stride * (BF16 ? 2 : 4);
  uint8_t *const step = terms + (size_t)(g >> 2) * (size_t)lanes * TermForm<T>::kStep;
  if constexpr (T == kPlain) {
    static_assert(BF16, "bf16 lanes");
    mx4_plain(static_cast<const uint16_t *>(row) + 32 * (size_t)g, g < groups, step, (size_t)lane, (size_t)lanes, g & 3);
  } else {
    float x[32];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float part[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};  // groups behind the last are zeros
      if (g < groups) mx4_load8<BF16>(row, 32 * (size_t)g + 8 * e, part);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[8 * e + i] = part[i];
    }
    mx4_terms<T>(x, step, (size_t)lane, (size_t)lanes, g & 3);
  }
}

template <bool BF16>
__global__ __launch_bounds__(256) void mx4_terms_kernel(const void *act, long long act_stride, int groups, int lanes,
                                                        uint8_t *terms) {
  mx4_terms_group<kTerms, BF16>(act, act_stride, groups, lanes, terms, (long long)blockIdx.x * 256 + threadIdx.x);
}

// ---- the product ------------------------------------------------------------------

// What becomes of sums: rows of floats, or the gated products of row pairs (the experts'
// hidden values; from tiles as terms for the product behind).
enum { kOutF32 = 0, kOutBf16 = 1, kOutGate = 2 };

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
  const uint8_t *terms;     // or pieces of bf16, of term_lanes lanes of floats
  int term_lanes;
  Mx4View act;              // or microscaled lanes
  int lanes;
  // grouped: the tiles, how many there are, and the lane of every place (NULL: the place)
  const Mx4Tile *tiles;
  int tile_count;
  const int *lane_of;
  const uint8_t *row_scales;    // packed (mx4_prepare_kernel), for the tile kernel
  const uint32_t *lane_scales;
  void *out;                // [lane or place][out_stride]; the experts' gate: terms of out_stride places
  int slice;                // steps of a slice of the columns (blockIdx.z), whose sums lie slice_out outputs apart
  size_t slice_out;
  int silu;                 // the experts' gate
  // a few lanes' own floats, and a token's experts (lane_of: the picks)
  const void *act_rows;
  long long act_stride;
  int experts, top;
  long long out_stride;
};

// silu(x) = x / (1 + e^-x)
__device__ __forceinline__ float silu_near(float x) {
  if (!(x > -87.0f)) return x * 0.0f;
  return x / (1.0f + exp_near(x > 87.0f ? -87.0f : -x));
}

// ---- experts' places ----------------------------------------------------------------

// Places: the slots (lane, choice) in the order of their experts; tiles: pieces of an
// expert's places.  A slot whose expert is none (out of range) has no place.  Expert e's
// tiles begin at tile (places before e) / tile + e: no more than that many lie before, and
// every expert finds its own without the others.  Tiles left over have no places.
constexpr int kPrepareThreads = 256;
constexpr int kPlaceRound = 16, kPlaceRounds = 4;  // slots of a lane on their way; rounds kept in registers

struct PlaceArgs {
  const int32_t *pick;
  int slots, experts, tile;       // places a tile
  uint32_t top_inverse;           // 2^32 / top and up to one more, for slot / top (slots below 2^20); 0: top is 1
  int *lane_of;                   // [slots] lane of a place
  int *place_of;                  // [slots] place of a slot, or -1
  Mx4Tile *tiles;                 // [slots / tile + experts]
};

__host__ __device__ __forceinline__ uint32_t place_inverse(int top) {
  return top == 1 ? 0u : (uint32_t)((1ull << 32) / (uint32_t)top) + 1;
}

__host__ __device__ __forceinline__ int place_lane(int slot, uint32_t inverse) {
  return inverse ? (int)((uint64_t)(uint32_t)slot * inverse >> 32) : slot;
}

// A workgroup lists one expert's slots, in an order of their own that is always the same:
// it reads every pick (from the L2 but once), counts its own and those of experts before,
// and gives its own their numbers.  One workgroup for all of them, counting with atomics,
// took 33 us for 16376 slots.
__device__ __forceinline__ void expert_place(const PlaceArgs &a, int expert) {
  __shared__ int sums[2][kPrepareThreads / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  constexpr int kWaves = kPrepareThreads / 64;
  const int each = (a.slots + kWaves - 1) / kWaves;
  const int first = wave * each, end = min(first + each, a.slots);
  auto round = [&](int s0, int (&e)[kPlaceRound]) {  // no branch, so that all are on their way at once
#pragma unroll
    for (int i = 0; i < kPlaceRound; ++i) e[i] = a.pick[min(s0 + 64 * i + lane, a.slots - 1)];
#pragma unroll
    for (int i = 0; i < kPlaceRound; ++i) e[i] = s0 + 64 * i + lane < end ? e[i] : -1;
  };
  // up to 16384 slots are read once: all rounds on their way, and kept for the numbers
  constexpr int kSpan = 64 * kPlaceRound, kHeld = kSpan * kPlaceRounds;
  int held[kPlaceRounds][kPlaceRound];
  int mine = 0, before = 0;
  for (int s0 = first; s0 < end; s0 += kHeld) {
#pragma unroll
    for (int r = 0; r < kPlaceRounds; ++r)
      if (s0 + kSpan * r < end) round(s0 + kSpan * r, held[r]);
#pragma unroll
    for (int r = 0; r < kPlaceRounds; ++r)
      if (s0 + kSpan * r < end)
#pragma unroll
        for (int i = 0; i < kPlaceRound; ++i) {
          mine += held[r][i] == expert;
          before += (uint32_t)held[r][i] < (uint32_t)expert;
        }
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    mine += __shfl_xor(mine, d);
    before += __shfl_xor(before, d);
  }
  if (lane == 0) sums[0][wave] = mine, sums[1][wave] = before;
  __syncthreads();
  int base = 0, total = 0, next = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    base += sums[1][w];
    total += sums[0][w];
    if (w < wave) next += sums[0][w];
  }
  next += base;
  for (int s0 = first; s0 < end; s0 += kHeld) {
#pragma unroll
    for (int r = 0; r < kPlaceRounds; ++r) {
      if (s0 + kSpan * r >= end) break;
      if (end - first > kHeld) round(s0 + kSpan * r, held[r]);
#pragma unroll
      for (int i = 0; i < kPlaceRound; ++i) {
        const int e = held[r][i], s = s0 + kSpan * r + 64 * i + lane;
        const uint64_t own = __ballot(e == expert);
        const int place = (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(own >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)own, (uint32_t)next));
        next += __builtin_popcountll(own);
        if (e == expert) {
          a.place_of[s] = place;
          a.lane_of[place] = place_lane(s, a.top_inverse);
        }
        if (expert == 0 && s < end && (uint32_t)e >= (uint32_t)a.experts) a.place_of[s] = -1;
      }
    }
  }
  // this expert's tiles and those left over between it and the next's, or the end
  const int tile0 = base / a.tile + expert;
  const int tile1 = expert + 1 < a.experts ? (base + total) / a.tile + expert + 1 : a.slots / a.tile + a.experts;
  for (int i = tile0 + (int)threadIdx.x; i < tile1; i += kPrepareThreads) {
    const int from = (i - tile0) * a.tile;
    a.tiles[i] = Mx4Tile{expert, base + min(from, total), max(0, min(a.tile, total - from))};
  }
}

// The product of many lanes: WM x WN waves of 16 MT lanes x 16 NT rows, 128 columns a
// step, both operands through LDS in ST stages.  2047 bf16 lanes of 8192 x 2048 take 55
// us of the GPU (1.25 PFLOP/s of bf16 products, where a large library product has 1.39), 2048
// microscaled ones 29.
//   * Stages are written only by global_load_lds, ST - 1 steps ahead.  A load to registers
//     in the loop costs more than it brings: with such loads and these in flight the
//     compiler waits for all of either.
//   * The 16-byte pieces of a row's codes and of a lane's terms are xored by a key of the
//     row (tile_key, pair_key), so that no bank meets twice.
//   * Scale bytes were put in the order of their reading by the launch before
//     (mx4_prepare_kernel): as they lie, a byte a lane and row, they would take the
//     cache as long as the codes do.
template <int T, int MT, int NT, int WM, int WN, int ST>
struct TileForm {
  static_assert(NT % 4 == 0 && ST >= 2, "words of scale bytes");
  static constexpr int kWaves = WM * WN;
  static constexpr int kLanes = 16 * MT * WM;
  static constexpr int kWaveRows = 16 * NT;
  static constexpr int kRows = kWaveRows * WN;
  static constexpr int kChunks = T == 0 ? 1 : TermForm<T == 0 ? kTerms : T>::kChunks;  // of 1 KB, a tile of lanes
  static constexpr int kLaneLoads = MT * WM * kChunks;              // DMA instructions of a step: lanes,
  static constexpr int kRowLoads = NT * WN;                         // codes,
  static constexpr int kScaleLoads = (kRows * 4 + 1023) / 1024;     // their scales,
  static constexpr int kLaneScales = T == 0 ? (kLanes * 4 + 1023) / 1024 : 0;  // and microscaled lanes'
  static constexpr int kAll = kLaneLoads + kRowLoads + kScaleLoads + kLaneScales;
  static constexpr int kLoads = (kAll + kWaves - 1) / kWaves;       // of a wave
  static constexpr int kRowsAt = kLaneLoads * 1024, kScalesAt = kRowsAt + kRowLoads * 1024;
  static constexpr int kLaneScalesAt = kScalesAt + kScaleLoads * 1024;
  static constexpr int kStage = kAll * 1024;
  static constexpr int kOut = kWaves * 16 * (kWaveRows + 4) * 4;    // a tile of lanes' outputs of every wave
  static constexpr int kGate = kWaves * 16 * MT * (kWaveRows / 2 + 4) * 4;  // all hidden values
  static constexpr __host__ __device__ bool pair(int c) { return T != 0 && (c + 1 < kChunks || c % 2); }  // as in term_piece
  static constexpr int most(int a, int b) { return a > b ? a : b; }
  static constexpr int lds(bool gate) { return most(ST * kStage, gate ? kGate : kOut); }
  static constexpr bool kAhead = MT * NT < 32;  // two lane tiles' operands in registers
  static constexpr bool kSpread = !kAhead;
  static constexpr int kLds = lds(true);
  static_assert(kLds <= 160 * 1024, "LDS");
};

// A row's sixteen-byte piece c of a step lies at c ^ key, so that lanes that are read
// together meet all banks: these are not sixteen in a row but 0-3, 12-15 and 20-27, and
// 4-11, 16-19 and 28-31 (keys 0, 1, 2, 3 cost four cycles more a read, by the counter of
// bank conflicts).
__host__ __device__ __forceinline__ int tile_key(int row) { return 0x78 >> (row >> 1 & 6) & 3; }

// The same of a lane's two pieces of terms, 128 bytes.
__host__ __device__ __forceinline__ int pair_key(int lane) { return lane >> 1 & 7; }

// Row of tile j of a wave's block of 16 NT rows, of `rows` in all (clamped).
template <int NT, bool PAIR>
__device__ __forceinline__ int tile_row(int block, int j, int at, int rows) {
  if (!PAIR) return min(block * 16 * NT + 16 * j + at, rows - 1);
  // half the tiles rows of the gate, half the same rows of what it gates, behind all of the gate's
  const int half = rows / 2, r = min(block * 8 * NT + 16 * (j % (NT / 2)) + at, half - 1);
  return j < NT / 2 ? r : half + r;
}

template <int NT, bool PAIR>
__host__ __device__ __forceinline__ int tile_blocks(int rows) {
  return PAIR ? (rows / 2 + 8 * NT - 1) / (8 * NT) : (rows + 16 * NT - 1) / (16 * NT);
}

// Scale bytes in the order a wave reads them: [block][step][wave lane][tile], zeros
// behind a row's last group.
struct PackArgs {
  Mx4View w;
  int rows, groups, experts, first_block;  // `rows` of each expert
  uint8_t *dst;
};

// Sixteen scale bytes of a row from group g on, zeros behind its last; nothing behind the
// row is read.
__device__ __forceinline__ uint4_t mx4_scales16(const uint8_t *row, int g, int groups) {
  struct __attribute__((packed)) Word {
    uint32_t w;
  };
  struct __attribute__((packed)) Words {
    uint32_t w[4];
  };
  if (g + 16 <= groups) {
    const Words b = *reinterpret_cast<const Words *>(row + g);
    return uint4_t{b.w[0], b.w[1], b.w[2], b.w[3]};
  }
  uint4_t out = {0, 0, 0, 0};
  if (groups >= 4) {  // words that end with the row, moved down to where they belong
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = reinterpret_cast<const Word *>(row + min(g + 4 * i, groups - 4))->w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int late = g + 4 * i - min(g + 4 * i, groups - 4);
      out[i] = late < 4 ? w[i] >> (8 * late) : 0u;
    }
  } else if (g == 0) {
    const uint32_t a = row[0], b = row[min(1, groups - 1)], c = row[groups - 1];
    out[0] = a | (groups > 1 ? b << 8 : 0u) | (groups > 2 ? c << 16 : 0u);
  }
  return out;
}

// A thread takes row `at` of four tiles of a block and sixteen groups, four steps: a turn of
// four rows' bytes in registers.
template <int NT, bool PAIR>
__device__ __forceinline__ void mx4_pack_scales(const PackArgs &a, long long id) {
  const int steps = mx4_steps(a.groups), blocks = tile_blocks<NT, PAIR>(a.rows), fours = (steps + 3) / 4;
  const int at = (int)(id & 15), q = (int)(id / 16 % (NT / 4));
  id /= 16 * (NT / 4);
  const int four = (int)(id % fours);
  const long long block = id / fours;
  const int e = (int)(block / blocks);
  if (e >= a.experts) return;
  uint4_t v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const size_t row = (size_t)e * a.rows + tile_row<NT, PAIR>((int)(block % blocks), 4 * q + j, at, a.rows);
    v[j] = mx4_scales16(a.w.scale + row * a.w.scale_stride, 16 * four, a.groups);
  }
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    if (4 * four + s >= steps) break;
    uint32_t *const dst =
        reinterpret_cast<uint32_t *>(a.dst) + (((size_t)block * steps + 4 * four + s) * 64 + at) * (NT / 4) + q;
    // bytes 0 .. 3 of four rows: pairs of rows, then pairs of pairs
    const uint32_t r0 = v[0][s], r1 = v[1][s], r2 = v[2][s], r3 = v[3][s];
    const uint32_t lo01 = __builtin_amdgcn_perm(r1, r0, 0x05010400u), hi01 = __builtin_amdgcn_perm(r1, r0, 0x07030602u);
    const uint32_t lo23 = __builtin_amdgcn_perm(r3, r2, 0x05010400u), hi23 = __builtin_amdgcn_perm(r3, r2, 0x07030602u);
    dst[0] = __builtin_amdgcn_perm(lo23, lo01, 0x05040100u);
    dst[16 * (NT / 4)] = __builtin_amdgcn_perm(lo23, lo01, 0x07060302u);
    dst[32 * (NT / 4)] = __builtin_amdgcn_perm(hi23, hi01, 0x05040100u);
    dst[48 * (NT / 4)] = __builtin_amdgcn_perm(hi23, hi01, 0x07060302u);
  }
}

// What products of many lanes need first, in one launch: lanes as terms, a sheet's scales
// packed (as pairs of blocks for the experts' gate), then another's; of microscaled lanes
// theirs, four tiles a block, in the first's place.  Experts' places in front (a
// workgroup each; place.experts 0: none).
struct PrepareArgs {
  const void *act;
  long long act_stride;
  int groups, lanes;
  uint8_t *terms;
  PlaceArgs place;
  PackArgs pairs, rows;  // first_block: the workgroup they begin with
  int lane_block;        // the terms' first, or the lane scales'
  PackArgs lane_scales;
};

template <int T, int NT, bool BF16>
__global__ __launch_bounds__(kPrepareThreads) void mx4_prepare_kernel(PrepareArgs a) {
  const int block = blockIdx.x;
  if (block >= a.rows.first_block) {
    mx4_pack_scales<NT, false>(a.rows, (long long)(block - a.rows.first_block) * kPrepareThreads + threadIdx.x);
  } else if (block >= a.pairs.first_block) {
    mx4_pack_scales<NT, true>(a.pairs, (long long)(block - a.pairs.first_block) * kPrepareThreads + threadIdx.x);
  } else if (block >= a.lane_block) {
    const long long id = (long long)(block - a.lane_block) * kPrepareThreads + threadIdx.x;
    if constexpr (T == 0)
      mx4_pack_scales<4, false>(a.lane_scales, id);
    else
      mx4_terms_group<T, BF16>(a.act, a.act_stride, a.groups, a.lanes, a.terms, id);
  } else {
    expert_place(a.place, block);
  }
}


template <bool V>
struct Choice {
  static constexpr bool value = V;
};
template <int V>
struct Count {
  static constexpr int value = V;
};

// Eight codes under their group's scale (a float whose exponent field is the scale byte) as bf16 numbers.
__device__ __forceinline__ bf16x8_t mx4_bf16(uint32_t codes, float scale) {
  typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
  const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0);
  const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
  const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2);
  const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
  return bf16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

template <int T, int MT, int NT, int WM, int WN, int ST, int OUT>
__global__ __launch_bounds__(64 * WM * WN, 2) void mx4_tile_kernel(Mx4Args g) {
  using F = TileForm<T, MT, NT, WM, WN, ST>;
  constexpr bool PAIR = OUT == kOutGate;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds_x[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int part = lane >> 4, at = lane & 15, wm = wave / WN, wn = wave % WN;
  const int blocks = tile_blocks<NT, PAIR>(g.rows);
  int tile_x, tile_y, first, count, expert = 0;
  if (!g.tiles) {
    xcd_tile(tile_x, tile_y);
    first = tile_y * F::kLanes;
    count = min(F::kLanes, g.lanes - first);
  } else {
    // workgroups go to the eight XCDs in turn: each takes a run of tiles, all rows of one
    // after another, so that its L2 serves a tile's lanes and its expert's rows again
    const int gx = (blocks + WN - 1) / WN, total = gx * g.tile_count, id = (int)blockIdx.x;
    const int run = (total + 7) / 8, at = (id & 7) * run + (id >> 3);
    if (at >= total) return;
    tile_x = at % gx;
    tile_y = at / gx;
    const Mx4Tile t = g.tiles[tile_y];
    first = t.first;
    count = t.count;
    expert = t.expert;
    if (count == 0) return;
  }
  const size_t row0 = (size_t)expert * (size_t)g.rows;
  const int block0 = tile_x * WN;  // blocks behind the last hold its rows, and are not stored
  const int steps = mx4_steps(g.groups);

  // ---- what this wave brings each step: sixteen bytes a lane, from base[i] + step * by[i] + off[i], and of codes
  // (walks[i] all ones) a step's piece, to a row's last at most.  By number: lanes' chunks, rows' codes, packed
  // scales.  The last wave may bring one twice.  What is the wave's is uniform and what is a lane's fits 32 bits
  // (sixteen rows' codes, all lanes' terms), so that a load takes two or three instructions of the lanes'.
  const uint8_t *base[F::kLoads];
  uint32_t by[F::kLoads], off[F::kLoads], walks[F::kLoads];
  int from[F::kLoads];  // the lanes, all on their way at once
#pragma unroll
  for (int i = 0; i < F::kLoads; ++i) {
    const int c = (wave * F::kLoads + i) % F::kChunks, of = 16 * ((wave * F::kLoads + i) / F::kChunks);
    from[i] = first + min(of + (F::pair(c) ? 8 * (c % 2) + lane / 8 : lane / 4), count - 1);
  }
  if (g.lane_of) {
#pragma unroll
    for (int i = 0; i < F::kLoads; ++i) from[i] = g.lane_of[from[i]];
  }
  // of a step's four pieces of a row this lane's; behind the last group the last (all codes are finite)
  const int piece = (lane & 3) ^ tile_key(lane >> 2), last_step = (g.groups - 1) >> 2;
#pragma unroll
  for (int i = 0; i < F::kLoads; ++i) {
    const int id = min(wave * F::kLoads + i, F::kAll - 1);
    walks[i] = 0;
    by[i] = 0;
    if (id < F::kLaneLoads) {
      const int c = id % F::kChunks;
      if constexpr (T == 0) {
        const int low = first + min(16 * (id / F::kChunks), count - 1);
        base[i] = g.act.code + (size_t)low * g.act.code_stride;
        off[i] = (uint32_t)(from[i] - low) * (uint32_t)g.act.code_stride;
        by[i] = 64;
        walks[i] = ~0u;
      } else {
        // two pieces of eight lanes, or one of sixteen
        const int in = 8 * (c % 2) + lane / 8;
        base[i] = g.terms + (size_t)(c / 2) * (size_t)g.term_lanes * 128;
        off[i] = F::pair(c) ? (uint32_t)from[i] * 128 + 16 * ((lane & 7) ^ pair_key(in))
                            : (uint32_t)from[i] * 64 + 16 * ((lane & 3) ^ tile_key(lane >> 2));
        by[i] = (uint32_t)g.term_lanes * (F::kChunks * 64);
      }
    } else if (id < F::kLaneLoads + F::kRowLoads) {
      const int r = 16 * (id - F::kLaneLoads);  // sixteen rows, four pieces each
      const int block = block0 + r / F::kWaveRows, j = r % F::kWaveRows / 16;
      const int low = tile_row<NT, PAIR>(block, j, 0, g.rows), row = tile_row<NT, PAIR>(block, j, lane / 4, g.rows);
      base[i] = g.w.code + (row0 + (size_t)low) * g.w.code_stride;
      off[i] = (uint32_t)(row - low) * (uint32_t)g.w.code_stride;
      by[i] = 64;
      walks[i] = ~0u;
    } else if (id < F::kLaneLoads + F::kRowLoads + F::kScaleLoads) {
      const int byte = (id - F::kLaneLoads - F::kRowLoads) * 1024 + lane * 16;  // of the blocks' 64 NT bytes each
      const int low = min(block0, blocks - 1), block = min(block0 + min(byte / (64 * NT), WN - 1), blocks - 1);
      base[i] = g.row_scales + ((size_t)expert * blocks + low) * (size_t)steps * (64 * NT);
      off[i] = (uint32_t)(block - low) * (uint32_t)(steps * (64 * NT)) + byte % (64 * NT);
      by[i] = 64 * NT;
    } else {
      const int byte = (id - F::kLaneLoads - F::kRowLoads - F::kScaleLoads) * 1024 + lane * 16;
      const int low = first / 64, block = min(low + byte / 256, (g.lanes - 1) / 64);
      base[i] = reinterpret_cast<const uint8_t *>(g.lane_scales) + (size_t)low * (size_t)steps * 256;
      off[i] = (uint32_t)(block - low) * (uint32_t)(steps * 256) + byte % 256;
      by[i] = 256;
    }
  }
  auto bring = [&](int step, int turn, int i) {
    uint8_t *dst = lds_x + turn % ST * F::kStage + min(wave * F::kLoads + i, F::kAll - 1) * 1024;
    const uint8_t *const at_step = base[i] + (size_t)min((uint32_t)step, (uint32_t)last_step | ~walks[i]) * by[i];
    const int most = g.groups - 1 - 4 * min(step, last_step);  // of a step's pieces
    const uint32_t more = 16u * (uint32_t)min(piece, most) & walks[i];
    __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void *)(at_step + (off[i] + more)),
                                     (__attribute__((address_space(3))) void *)dst, 16, 0, 0);
  };

  float4_t acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};

  // A tile that an expert does not fill: waves without lanes only bring
  const bool busy = 16 * wm * MT < count;
  // Workgroups of neighbouring rows begin at other columns: rows are often a power of
  // two bytes apart, and all at the same column would ask the same cache channels
  const int k_first = blockIdx.z * g.slice, k_end = min(k_first + g.slice, steps), k_count = k_end - k_first;
  int k = k_first + 2 * tile_x % k_count, k_ahead = k;
  auto next = [&](int at) { return at + 1 < k_end ? at + 1 : k_first; };
#pragma unroll
  for (int s = 0; s < ST - 1; ++s)
    if (s < k_count) {
#pragma unroll
      for (int i = 0; i < F::kLoads; ++i) bring(k_ahead, s, i);
      k_ahead = next(k_ahead);
    }
  // A step; its stage `ST - 1` ahead is brought a load after every few products (all at once,
  // loads hold the wave up while they are taken, and the matrix cores wait)
  auto step = [&](int s, auto ahead) {
    constexpr bool kBring = decltype(ahead)::value;
    // lgkmcnt(0), and of this wave's loads all but the ST - 2 stages behind this step's
    constexpr int kBehind = (ST - 2) * F::kLoads;
    static_assert(kBehind < 64, "vmcnt");
    if (ST > 2 && (kBring || s + ST - 2 < k_count))
      __builtin_amdgcn_s_waitcnt((kBehind & 15) | (kBehind >> 4) << 14 | 0x0070);
    else
      __builtin_amdgcn_s_waitcnt(0x0070);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    const uint8_t *st = lds_x + s % ST * F::kStage;
    if (kBring && (!F::kSpread || !busy)) {
#pragma unroll
      for (int i = 0; i < F::kLoads; ++i) bring(k_ahead, s + ST - 1, i);
    }
    if (!busy) return;
    // A share of the loads ahead, behind the run-th of `runs` parts of the products
    auto spread = [&](int run, auto runs) {
      constexpr int kEach = (F::kLoads + decltype(runs)::value - 1) / decltype(runs)::value;
      if (kBring && F::kSpread) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < kEach; ++u)
          if (run * kEach + u < F::kLoads) bring(k_ahead, s + ST - 1, run * kEach + u);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    uint32_t ws[NT / 4];
#pragma unroll
    for (int q = 0; q < NT / 4; ++q)
      ws[q] = *reinterpret_cast<const uint32_t *>(st + F::kScalesAt + (wn * 64 + lane) * NT + 4 * q);
    auto read_codes = [&](int j) {
      const int r = 16 * j + at;
      return *reinterpret_cast<const uint4_t *>(st + F::kRowsAt + (wn * F::kWaveRows + r) * 64 + 16 * (part ^ tile_key(r)));
    };
    if constexpr (T == kPlain) {
      // Codes as bf16, eight of a group at a time (a part's group is its scale's, so it is multiplied in as they
      // are converted, exactly; 255 gives NaNs), against the same eight of every lane tile
      bf16x8_t x[2][MT];
      auto read_eight = [&](int c) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
          x[c % 2][i] = *reinterpret_cast<const bf16x8_t *>(st + (wm * MT + i) * F::kChunks * 1024 + c / 2 * 2048 +
                                                            at * 128 + 16 * ((4 * (c % 2) + part) ^ pair_key(at)));
      };
      read_eight(0);
      uint4_t code[NT];
      float scale[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        code[j] = read_codes(j);
        scale[j] = __builtin_bit_cast(float, (ws[j / 4] >> 8 * (j % 4) & 0xFFu) << 23);
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        __builtin_amdgcn_sched_barrier(0);
        if (c + 1 < 4) read_eight(c + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const bf16x8_t w = mx4_bf16(code[j][c], scale[j]);
#pragma unroll
          for (int i = 0; i < MT; ++i) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, x[c % 2][i], acc[i][j], 0, 0, 0);
          if (j % (NT / 2) == NT / 2 - 1) spread(2 * c + j / (NT / 2), Count<8>());
        }
      }
    } else {
      // Lanes' terms behind the last group are zeros, and codes are finite; of microscaled lanes neither side's are
      const uint32_t keep = T != 0 || 4 * k + part < g.groups ? 0xFFFFFFFFu : 0u;
      constexpr int kOps = F::kAhead ? 2 : 1;
      int8v_t op[kOps][T == 0 ? 1 : T];
      uint2_t scale[kOps];
      auto read_lanes = [&](int i) {
        const uint8_t *mine = st + (wm * MT + i) * F::kChunks * 1024;
        uint4_t piece[F::kChunks];
#pragma unroll
        for (int c = 0; c < F::kChunks; ++c)
          piece[c] = *reinterpret_cast<const uint4_t *>(
              F::pair(c) ? mine + c / 2 * 2048 + at * 128 + 16 * ((4 * (c % 2) + part) ^ pair_key(at))
                         : mine + c * 1024 + at * 64 + 16 * (part ^ tile_key(at)));
#pragma unroll
        for (int t = 0; t < (T == 0 ? 1 : T); ++t) {
          const uint4_t a = piece[t], b = T == 0 ? uint4_t{0, 0, 0, 0} : piece[T == 0 ? 0 : T + t / 2];
          op[i % kOps][t] = int8v_t{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[2 * (t % 2)], (int)b[2 * (t % 2) + 1], 0, 0};
        }
        if constexpr (T != 0) scale[i % kOps] = uint2_t{piece[F::kChunks - 1][2], piece[F::kChunks - 1][3]};
      };
      int8v_t w[NT];
      read_lanes(0);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        uint4_t c = read_codes(j);
        if (T == 0) c &= keep;
        w[j] = int8v_t{(int)c[0], (int)c[1], (int)c[2], (int)c[3], 0, 0, 0, 0};
      }
      int ls = 0;
      if constexpr (T == 0) {
        static_assert(MT == 4 || T != 0, "a byte of the packed scales a tile");
        ls = *reinterpret_cast<const int *>(st + F::kLaneScalesAt + wm * 256 + lane * 4);
      }
#define MX4_PRODUCT(I, J, A, FMT, OPSEL, SCALE)                                                                      \
  switch (J % 4) {                                                                                                   \
    case 0:                                                                                                          \
      acc[I][J] =                                                                                                    \
          __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w[J], A, acc[I][J], 4, FMT, 0, ws[J / 4], OPSEL, SCALE);  \
      break;                                                                                                         \
    case 1:                                                                                                          \
      acc[I][J] =                                                                                                    \
          __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w[J], A, acc[I][J], 4, FMT, 1, ws[J / 4], OPSEL, SCALE);  \
      break;                                                                                                         \
    case 2:                                                                                                          \
      acc[I][J] =                                                                                                    \
          __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w[J], A, acc[I][J], 4, FMT, 2, ws[J / 4], OPSEL, SCALE);  \
      break;                                                                                                         \
    default:                                                                                                         \
      acc[I][J] =                                                                                                    \
          __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w[J], A, acc[I][J], 4, FMT, 3, ws[J / 4], OPSEL, SCALE);  \
  }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        // the next lanes' operands are on their way while these are multiplied
        __builtin_amdgcn_sched_barrier(0);
        if (F::kAhead && i + 1 < MT) read_lanes(i + 1);
        if (!F::kAhead && i > 0) read_lanes(i);
        __builtin_amdgcn_sched_barrier(0);
        // a term at a time over the row tiles: products that add to the same sums lie apart
#pragma unroll
        for (int t = 0; t < (T == 0 ? 1 : T); ++t) {
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            constexpr int kFmt = T == 0 ? 4 : 2;
            const int a = T == 0 ? ls : (int)scale[i % kOps][t / 4];
            const int byte = T == 0 ? i : t % 4;
            if (byte == 0) MX4_PRODUCT(i, j, op[i % kOps][t], kFmt, 0, a)
            if (byte == 1) MX4_PRODUCT(i, j, op[i % kOps][t], kFmt, 1, a)
            if (byte == 2) MX4_PRODUCT(i, j, op[i % kOps][t], kFmt, 2, a)
            if (byte == 3) MX4_PRODUCT(i, j, op[i % kOps][t], kFmt, 3, a)
          }
          spread(i * (T == 0 ? 1 : T) + t, Count<MT *(T == 0 ? 1 : T)>());
        }
      }
#undef MX4_PRODUCT
    }
  };
  int s = 0;
  for (; s < k_count - (ST - 1); ++s) {
    step(s, Choice<true>());
    k = next(k);
    k_ahead = next(k_ahead);
  }
  for (; s < k_count; ++s) {
    step(s, Choice<false>());
    k = next(k);
  }
  // every lane took part in the products: nothing of them may move behind a branch that some leave
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) asm volatile("" : "+v"(acc[i][j]));
  __syncthreads();

  if constexpr (PAIR) {
    // h = gate(g) u, both in this lane's registers; through LDS, so that a lane has the 32 values of a group.  The
    // wave takes its own room, lanes by pitch
    constexpr int kHalf = F::kWaveRows / 2, kPitch = kHalf + 4;
    float *const turn = reinterpret_cast<float *>(lds_x) + wave * 16 * MT * kPitch;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT / 2; ++j) {
        float4_t h;
#pragma unroll
        for (int r = 0; r < 4; ++r)
          h[r] = (g.silu ? silu_near(acc[i][j][r]) : gelu_near(acc[i][j][r])) * acc[i][j + NT / 2][r];
        *reinterpret_cast<float4_t *>(turn + (16 * i + at) * kPitch + 16 * j + 4 * part) = h;
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // one wave's room, no barrier
    const int inner_groups = g.rows / 2 / kMx4Group, group0 = (block0 + wn) * (kHalf / kMx4Group);
    constexpr int kGroups = kHalf / kMx4Group;
    for (int item = lane; item < 16 * MT * kGroups; item += 64) {
      const int m = item / kGroups, group = group0 + item % kGroups;
      const int place = 16 * wm * MT + m;
      if (place >= count || group >= inner_groups) continue;
      float x[32];
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const float4_t f = *reinterpret_cast<const float4_t *>(turn + m * kPitch + item % kGroups * 32 + 4 * q);
#pragma unroll
        for (int d = 0; d < 4; ++d) x[4 * q + d] = f[d];
      }
      uint8_t *const h = static_cast<uint8_t *>(g.out);
      const size_t to = (size_t)(first + place), of = (size_t)g.out_stride;
      auto step = [&](int group) { return h + (size_t)(group >> 2) * of * TermForm<kTerms>::kStep; };
      mx4_terms<kTerms>(x, step(group), to, of, group & 3);
      if (group + 1 == inner_groups)  // the groups behind the last are zeros
        for (int z = group + 1; z < 4 * mx4_steps(inner_groups); ++z)
          for (int c = 0; c < TermForm<kTerms>::kChunks; ++c)
            *reinterpret_cast<uint4_t *>(step(z) + term_piece<kTerms>(to, of, c, z & 3)) = uint4_t{0, 0, 0, 0};
    }
    return;
  }
  // The weight is the first operand: this wave lane holds rows 4 part .. + 3 of lane
  // `at`.  They cross LDS so that a lane's rows of the wave are stored in one go: four
  // by four, sixteen lanes' lines would be written in halves, each to the same channel.
  constexpr int kPitch = F::kWaveRows + 4;
  float *const turn = reinterpret_cast<float *>(lds_x) + wave * 16 * kPitch;
  const int n0 = (block0 + wn) * F::kWaveRows;
  constexpr int kBytes = OUT == kOutBf16 ? 2 : 4;
  const bool whole = g.out_stride % (16 / kBytes) == 0 && ((uintptr_t)g.out & 15u) == 0;
  constexpr int kOf = 16 / kBytes;                 // outputs of a store
  constexpr int kRowLanes = F::kWaveRows / kOf;    // wave lanes that store a lane's rows
#pragma unroll
  for (int i = 0; i < MT; ++i) {
#pragma unroll
    for (int j = 0; j < NT; ++j)
      *reinterpret_cast<float4_t *>(turn + at * kPitch + 16 * j + 4 * part) = acc[i][j];
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // one wave's room, no barrier
#pragma unroll
    for (int r = 0; r < 16 * kRowLanes / 64; ++r) {
      const int m = r * (64 / kRowLanes) + lane / kRowLanes, c = lane % kRowLanes * kOf;
      float v[kOf];
#pragma unroll
      for (int q = 0; q < kOf / 4; ++q) {
        const float4_t f = *reinterpret_cast<const float4_t *>(turn + m * kPitch + c + 4 * q);
#pragma unroll
        for (int d = 0; d < 4; ++d) v[4 * q + d] = f[d];
      }
      const int n = n0 + c;
      const int place = 16 * (wm * MT + i) + m;
      if (place >= count) continue;
      const size_t out = (size_t)blockIdx.z * g.slice_out + (size_t)(first + place) * (size_t)g.out_stride + n;
      if (whole && n + kOf <= g.rows) {
        uint4_t b;
        if (OUT == kOutBf16) {
#pragma unroll
          for (int d = 0; d < 4; ++d)
            b[d] = float_bf16(v[(2 * d) % kOf]) | (uint32_t)float_bf16(v[(2 * d + 1) % kOf]) << 16;
        } else {
#pragma unroll
          for (int d = 0; d < 4; ++d) b[d] = __builtin_bit_cast(uint32_t, v[d]);
        }
        *reinterpret_cast<uint4_t *>(static_cast<uint8_t *>(g.out) + out * kBytes) = b;
      } else {
#pragma unroll
        for (int d = 0; d < kOf; ++d)
          if (n + d < g.rows) {
            if (OUT == kOutBf16)
              static_cast<uint16_t *>(g.out)[out + d] = float_bf16(v[d]);
            else
              static_cast<float *>(g.out)[out + d] = v[d];
          }
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

// ---- the experts' feed-forward ------------------------------------------------------

// The codes and scale of group g of a row as loaded: behind its last group the last one's,
// which `mx4_clear` makes zeros.
struct Mx4Codes {
  uint4_t code;
  int scale;
};

__device__ __forceinline__ Mx4Codes mx4_load(const uint8_t *code, const uint8_t *scale, int g, int groups) {
  const int at = min(g, groups - 1);
  return Mx4Codes{*reinterpret_cast<const uint4_t *>(code + 16 * (size_t)at), scale[at]};
}

__device__ __forceinline__ int8v_t mx4_clear(const Mx4Codes &c, int g, int groups) {
  const uint4_t k = g < groups ? c.code : uint4_t{0, 0, 0, 0};
  return int8v_t{(int)k[0], (int)k[1], (int)k[2], (int)k[3], 0, 0, 0, 0};
}

// The product of few lanes, sixteen a workgroup, with a sheet that the caches hold (6144 x 1536:
// 8 lanes of floats 10 us with the terms' launch, microscaled ones 5): a workgroup takes 16 RT
// rows and its four waves every fourth step, operands straight to registers, four steps'
// codes in flight a wave; sums meet in LDS.  Lane l of a wave holds group l / 16 of row and
// of lane l % 16.  T terms (five), 0: microscaled lanes.
constexpr int kFewAhead = 4;

template <int T, int RT, int OUT>
__global__ __launch_bounds__(256) void mx4_few_kernel(Mx4Args g) {
  __shared__ float4_t sums[3][RT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int part = lane >> 4, at = lane & 15;
  const int n0 = blockIdx.x * 16 * RT, steps = mx4_steps(g.groups);
  const int first = 16 * blockIdx.y, count = min(16, g.lanes - first);
  const uint8_t *code[RT], *scale[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const size_t row = (size_t)min(n0 + 16 * r + at, g.rows - 1);
    code[r] = g.w.code + row * g.w.code_stride;
    scale[r] = g.w.scale + row * g.w.scale_stride;
  }
  const size_t from = (size_t)(first + min(at, count - 1));
  float4_t acc[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) acc[r] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
  for (int s0 = wave; s0 < steps; s0 += 4 * kFewAhead) {
    Mx4Codes w[kFewAhead][RT];
#pragma unroll
    for (int u = 0; u < kFewAhead; ++u)
#pragma unroll
      for (int r = 0; r < RT; ++r) w[u][r] = mx4_load(code[r], scale[r], 4 * (s0 + 4 * u) + part, g.groups);
#pragma unroll
    for (int u = 0; u < kFewAhead; ++u) {
      const int s = s0 + 4 * u;
      if (s >= steps) break;
      const int group = 4 * s + part;
      if constexpr (T == 0) {
        const Mx4Codes c = mx4_load(g.act.code + from * g.act.code_stride, g.act.scale + from * g.act.scale_stride, group,
                                    g.groups);
        const int8v_t a = mx4_clear(c, group, g.groups);
#pragma unroll
        for (int r = 0; r < RT; ++r)
          acc[r] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx4_clear(w[u][r], group, g.groups), a, acc[r], 4, 4, 0,
                                                                    group < g.groups ? w[u][r].scale : 0, 0,
                                                                    group < g.groups ? c.scale : 0);
      } else {
        // lanes' terms behind the last group are zeros, and codes are finite; their scales may not be
        const size_t of = (size_t)g.term_lanes;
        const uint8_t *step = g.terms + (size_t)s * of * TermForm<kTerms>::kStep;
        const uint2_t scales = term_scales<kTerms>(step, from, of, part);
#pragma unroll
        for (int q = 0; q < T; ++q) {
          const int8v_t a = term_operand<kTerms>(step, from, of, q, part);
          const int as = q < 4 ? (int)(scales[0] >> (8 * q)) : (int)scales[1];
#pragma unroll
          for (int r = 0; r < RT; ++r)
            acc[r] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx4_clear(w[u][r], group, g.groups), a, acc[r], 4, 2,
                                                                      0, group < g.groups ? w[u][r].scale : 0, 0, as);
        }
      }
    }
  }
  // every lane took part in the products: nothing of them may move behind a branch that some leave
#pragma unroll
  for (int r = 0; r < RT; ++r) asm volatile("" : "+v"(acc[r]));
  if (wave > 0)
#pragma unroll
    for (int r = 0; r < RT; ++r) sums[wave - 1][r][lane] = acc[r];
  __syncthreads();
  if (wave > 0 || at >= count) return;
  const size_t out = (size_t)(first + at) * (size_t)g.out_stride;
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    float4_t v = acc[r];
#pragma unroll
    for (int w = 0; w < 3; ++w) v += sums[w][r][lane];
    const int n = n0 + 16 * r + 4 * part;
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      if (n + d >= g.rows) continue;
      if (OUT == kOutBf16)
        static_cast<uint16_t *>(g.out)[out + n + d] = float_bf16(v[d]);
      else
        static_cast<float *>(g.out)[out + n + d] = v[d];
    }
  }
}

// ---- a few lanes of floats, cut where they are used -----------------------------------

// A wave cuts the groups that its own steps need (first, first + stride, ..: `count` steps of
// one row of `groups` groups) into LDS, [step][part] records of terms and scales.
constexpr int kRecord = 24 * kTerms + 8;  // bytes

template <bool BF16>
__device__ __forceinline__ void own_terms(const void *row, int groups, int first, int stride, int count, int lane,
                                          uint8_t *room) {
  for (int i = lane; i < 4 * count; i += 64) {
    const int g = 4 * (first + i / 4 * stride) + i % 4;
    float x[32];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float part[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
      if (g < groups) mx4_load8<BF16>(row, 32 * (size_t)g + 8 * e, part);
#pragma unroll
      for (int q = 0; q < 8; ++q) x[8 * e + q] = part[q];
    }
    mx4_terms_record(x, room + i * kRecord);
  }
}

// Column c of an operand of single lanes: term c % 5 of lane c / 5 (columns behind the last
// hold anything), from the lanes' records.
__device__ __forceinline__ int8v_t own_operand(const uint8_t *record, int t, int &scale) {
  const uint2_t a = *reinterpret_cast<const uint2_t *>(record + 24 * t);
  const uint2_t b = *reinterpret_cast<const uint2_t *>(record + 24 * t + 8);
  const uint2_t c = *reinterpret_cast<const uint2_t *>(record + 24 * t + 16);
  const uint2_t s = *reinterpret_cast<const uint2_t *>(record + 24 * kTerms);
  scale = t < 4 ? (int)(s[0] >> (8 * t)) : (int)s[1];
  return int8v_t{(int)a[0], (int)a[1], (int)b[0], (int)b[1], (int)c[0], (int)c[1], 0, 0};
}

// One to three lanes, a token's step: a lane's terms are columns of
// the one operand, so five terms cost one product, and a wave cuts the lanes itself while
// its first codes are on their way: no launch before.  Sums of terms and waves in LDS.
// One fp32 lane of 6144 x 1536: 5.7 us, 4.8 at best, of which a launch by itself is 2 and
// the codes a microsecond; with terms from a launch before it 12.8.
// kOutGate: blockIdx.y a slot of the experts: its expert's gate and up rows, the gated
// products as floats.
template <int RT, int OUT, bool BF16>
__global__ __launch_bounds__(256) void mx4_step_kernel(Mx4Args g) {
  constexpr bool PAIR = OUT == kOutGate;
  static_assert(!PAIR || RT == 2, "a tile of gate rows, and the rows they gate");
  extern __shared__ __attribute__((aligned(16))) uint8_t lds_x[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int part = lane >> 4, at = lane & 15;
  const int steps = mx4_steps(g.groups), mine = (steps - wave + 3) / 4;
  const int half = g.rows / 2, n0 = blockIdx.x * 16 * (PAIR ? 1 : RT);
  int lanes = g.lanes;
  size_t row0 = 0, from = 0;
  if (PAIR) {
    const int e = g.lane_of[blockIdx.y];  // the picks
    if ((uint32_t)e >= (uint32_t)g.experts) return;
    row0 = (size_t)e * (size_t)g.rows;
    from = blockIdx.y / (uint32_t)g.top;
    lanes = 1;
  }
  const uint8_t *code[RT], *scale[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const size_t row = row0 + (size_t)(PAIR ? r * half + min(n0 + at, half - 1) : min(n0 + 16 * r + at, g.rows - 1));
    code[r] = g.w.code + row * g.w.code_stride;
    scale[r] = g.w.scale + row * g.w.scale_stride;
  }
  Mx4Codes w[kFewAhead][RT];
  auto load = [&](int i0) {
#pragma unroll
    for (int u = 0; u < kFewAhead; ++u)
#pragma unroll
      for (int r = 0; r < RT; ++r) w[u][r] = mx4_load(code[r], scale[r], 4 * (wave + 4 * (i0 + u)) + part, g.groups);
  };
  load(0);
  const int room_lane = 4 * ((steps + 3) / 4) * kRecord;  // of a lane, this wave's
  uint8_t *const room = lds_x + wave * lanes * room_lane;
  for (int m = 0; m < lanes; ++m)
    own_terms<BF16>(static_cast<const uint8_t *>(g.act_rows) + (from + m) * (size_t)g.act_stride * (BF16 ? 2 : 4),
                       g.groups, wave, 4, mine, lane, room + m * room_lane);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the wave's own, no barrier
  const int column_lane = min(at / kTerms, lanes - 1), column_term = at / kTerms < lanes ? at % kTerms : 0;
  float4_t acc[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) acc[r] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
  for (int i0 = 0; i0 < mine; i0 += kFewAhead) {
    if (i0) load(i0);
#pragma unroll
    for (int u = 0; u < kFewAhead; ++u) {
      if (i0 + u >= mine) break;
      const int group = 4 * (wave + 4 * (i0 + u)) + part;
      int as;
      const int8v_t a =
          own_operand(room + column_lane * room_lane + (4 * (i0 + u) + part) * kRecord, column_term, as);
#pragma unroll
      for (int r = 0; r < RT; ++r)
        acc[r] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx4_clear(w[u][r], group, g.groups), a, acc[r], 4, 2, 0,
                                                                  group < g.groups ? w[u][r].scale : 0, 0, as);
    }
  }
#pragma unroll
  for (int r = 0; r < RT; ++r) asm volatile("" : "+v"(acc[r]));  // as in mx4_few_kernel
  __syncthreads();
  // [wave][row][column]
  float *const sums = reinterpret_cast<float *>(lds_x);
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int d = 0; d < 4; ++d) sums[((wave * RT + r) * 16 + 4 * part + d) * 17 + at] = acc[r][d];
  __syncthreads();
  auto total = [&](int r, int row, int m) {  // terms from the smallest on, waves in order
    float v = 0.0f;
#pragma unroll
    for (int t = kTerms - 1; t >= 0; --t)
#pragma unroll
      for (int q = 0; q < 4; ++q) v += sums[((q * RT + r) * 16 + row) * 17 + m * kTerms + t];
    return v;
  };
  if (PAIR) {
    if (threadIdx.x >= 16 || n0 + (int)threadIdx.x >= half) return;
    const float gate = total(0, threadIdx.x, 0), up = total(RT - 1, threadIdx.x, 0);
    static_cast<float *>(g.out)[(size_t)blockIdx.y * half + n0 + threadIdx.x] =
        (g.silu ? silu_near(gate) : gelu_near(gate)) * up;
    return;
  }
  for (int i = threadIdx.x; i < 16 * RT * lanes; i += 256) {
    const int m = i / (16 * RT), n = i % (16 * RT);
    if (n0 + n >= g.rows) continue;
    const float v = total(n / 16, n % 16, m);
    const size_t out = (size_t)m * (size_t)g.out_stride + n0 + n;
    if (OUT == kOutBf16)
      static_cast<uint16_t *>(g.out)[out] = float_bf16(v);
    else
      static_cast<float *>(g.out)[out] = v;
  }
}

// Up to sixteen lanes of floats of a sheet of many rows (a vocabulary), bound by its bytes:
// workgroups that stay, a wave sixteen rows at a time, the next rows' codes and scales on
// their way to registers while these are multiplied.  Lanes' terms are columns of
// operands (five lanes of fp32 two), cut by the workgroup and kept in LDS as they are
// read; sums cross LDS to be added and stored.  Five fp32 lanes of 262144 x 1536: 47 us
// out of the caches (4.6 TB/s; a copy has 4.96), 39 in them; as tiles 55 and 42, of which
// packing the scales is ten, and a workgroup every 64 rows 74.  Loads past the caches
// 50 either way.  Three operands and more take longer than tiles (8 lanes 57 for 44, in
// the caches).
constexpr int kHeadWaves = 8;
constexpr int kHeadSteps = 4;  // of a piece: sixteen scales of a row
constexpr int kHeadAhead = 6;  // pieces of a wave on their way

struct HeadForm {
  static constexpr int kImage = 64 * 28;  // bytes of an operand: sixteen a wave lane, eight, a scale
  static int operands(int lanes) { return (lanes * kTerms + 15) / 16; }
  static size_t sums(int lanes) { return (size_t)kHeadWaves * 16 * (16 * operands(lanes) + 1) * sizeof(float); }
  static size_t lds(int groups, int lanes) { return (size_t)operands(lanes) * mx4_steps(groups) * kImage + sums(lanes); }
};

// A piece of sixteen rows: codes, a group a wave lane and step, and the scales of its row.
struct HeadPiece {
  uint4_t code[kHeadSteps], scale;
};

template <int OPERANDS, int OUT, bool BF16>
__global__ __launch_bounds__(64 * kHeadWaves, 2) void mx4_head_kernel(Mx4Args g) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds_x[];
  constexpr int kImage = HeadForm::kImage, kPitch = 16 * OPERANDS + 1;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int part = lane >> 4, at = lane & 15;
  const int steps = mx4_steps(g.groups), pieces = (steps + kHeadSteps - 1) / kHeadSteps;
  const int blocks = (g.rows + 15) / 16, stride = gridDim.x * kHeadWaves;
  float *const sums = reinterpret_cast<float *>(lds_x + (size_t)OPERANDS * steps * kImage) + wave * 16 * kPitch;
  HeadPiece ring[kHeadAhead];
  auto load = [&](HeadPiece &r, int block, int piece) {  // no branch: what lies behind is a row's last, and cleared
    const size_t row = (size_t)min(16 * block + at, g.rows - 1);
    const uint8_t *code = g.w.code + row * g.w.code_stride, *scale = g.w.scale + row * g.w.scale_stride;
#pragma unroll
    for (int s = 0; s < kHeadSteps; ++s)
      r.code[s] =
          *reinterpret_cast<const uint4_t *>(code + 16 * (size_t)min(4 * (piece * kHeadSteps + s) + part, g.groups - 1));
    struct __attribute__((packed)) Words {
      uint32_t w[4];
    };
    const Words b = *reinterpret_cast<const Words *>(scale + min(16 * piece, g.groups - 16));
    r.scale = uint4_t{b.w[0], b.w[1], b.w[2], b.w[3]};
  };
  int block = blockIdx.x * kHeadWaves + wave;
  int ahead = block, ahead_piece = 0, piece = 0;
  auto load_next = [&](HeadPiece &r) {
    load(r, min(ahead, blocks - 1), ahead_piece);
    if (++ahead_piece == pieces) ahead_piece = 0, ahead += stride;
  };
#pragma unroll
  for (int i = 0; i < kHeadAhead; ++i) load_next(ring[i]);
  // the lanes' operands; columns that no term has hold anything
  for (int i = threadIdx.x; i < g.lanes * 4 * steps; i += 64 * kHeadWaves) {
    const int m = i / (4 * steps), group = i - m * 4 * steps;
    const void *row = static_cast<const uint8_t *>(g.act_rows) + (size_t)m * (size_t)g.act_stride * (BF16 ? 2 : 4);
    float x[32];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
      if (group < g.groups) mx4_load8<BF16>(row, 32 * (size_t)group + 8 * e, v);
#pragma unroll
      for (int q = 0; q < 8; ++q) x[8 * e + q] = v[q];
    }
    auto image = [&](int t) { return lds_x + (size_t)((m * kTerms + t) / 16 * steps + group / 4) * kImage; };
    auto slot = [&](int t) { return group % 4 * 16 + (m * kTerms + t) % 16; };
    mx4_cut<kTerms>(
        x,
        [&](int t, const uint6_t &w) {
          *reinterpret_cast<uint4_t *>(image(t) + 16 * slot(t)) = uint4_t{w[0], w[1], w[2], w[3]};
          *reinterpret_cast<uint2_t *>(image(t) + 1024 + 8 * slot(t)) = uint2_t{w[4], w[5]};
        },
        [&](const uint2_t &s) {
#pragma unroll
          for (int t = 0; t < kTerms; ++t)
            *reinterpret_cast<uint32_t *>(image(t) + 1536 + 4 * slot(t)) = t < 4 ? s[0] >> (8 * t) : s[1];
        });
  }
  __syncthreads();
  float4_t acc[OPERANDS];
  auto multiply = [&](HeadPiece &r, int piece) {
    // a row's last sixteen scales, where its last piece has fewer, moved down to where they belong
    int late = 16 * piece - min(16 * piece, g.groups - 16);
    if (late) {
      for (; late >= 4; late -= 4) r.scale = uint4_t{r.scale[1], r.scale[2], r.scale[3], 0u};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        r.scale[i] = (uint32_t)(((uint64_t)(i < 3 ? r.scale[i + 1] : 0u) << 32 | r.scale[i]) >> (8 * late));
    }
#pragma unroll
    for (int s = 0; s < kHeadSteps; ++s) {
      const int step = piece * kHeadSteps + s;
      if (step >= steps) break;
      const bool in = 4 * step + part < g.groups;
      const uint4_t c = in ? r.code[s] : uint4_t{0, 0, 0, 0};
      const int8v_t w = {(int)c[0], (int)c[1], (int)c[2], (int)c[3], 0, 0, 0, 0};
      const int ws = (int)(r.scale[s] >> (8 * part));  // zeros behind the last
#pragma unroll
      for (int q = 0; q < OPERANDS; ++q) {
        const uint8_t *image = lds_x + (size_t)(q * steps + step) * kImage;
        const uint4_t a = *reinterpret_cast<const uint4_t *>(image + 16 * lane);
        const uint2_t b = *reinterpret_cast<const uint2_t *>(image + 1024 + 8 * lane);
        const int as = *reinterpret_cast<const int *>(image + 1536 + 4 * lane);
        const int8v_t op = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], 0, 0};
        acc[q] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, op, acc[q], 4, 2, 0, ws, 0, as);
      }
    }
  };
  auto store = [&](int of) {
#pragma unroll
    for (int q = 0; q < OPERANDS; ++q) {
      asm volatile("" : "+v"(acc[q]));  // every lane took part in the products, as in mx4_few_kernel
#pragma unroll
      for (int d = 0; d < 4; ++d) sums[(4 * part + d) * kPitch + 16 * q + at] = acc[q][d];
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the wave's own, no barrier
    for (int i = lane; i < 16 * g.lanes; i += 64) {
      const int m = i / 16, n = 16 * of + i % 16;
      float v = 0.0f;
#pragma unroll
      for (int t = kTerms - 1; t >= 0; --t) v += sums[i % 16 * kPitch + m * kTerms + t];
      if (n >= g.rows) continue;
      const size_t out = (size_t)m * (size_t)g.out_stride + n;
      if (OUT == kOutBf16)
        static_cast<uint16_t *>(g.out)[out] = float_bf16(v);
      else
        static_cast<float *>(g.out)[out] = v;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  };
  while (block < blocks) {
#pragma unroll
    for (int i = 0; i < kHeadAhead; ++i) {
      if (block >= blocks) break;
      if (piece == 0)
#pragma unroll
        for (int q = 0; q < OPERANDS; ++q) acc[q] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
      multiply(ring[i], piece);
      load_next(ring[i]);
      if (++piece == pieces) {
        store(block);
        piece = 0;
        block += stride;
      }
    }
  }
}

// The down products of a token's experts and their sum: blockIdx.y a lane, eight waves, each
// every eighth of its choices (its hidden values cut by the wave), sixteen rows.  Eight of
// 128 experts, 1536 and 768: 6.2 us behind 7.6 of gate and up (13.6 a call); by experts, in four
// launches, 34.
template <bool BF16>
__global__ __launch_bounds__(512) void expert_step_kernel(Mx4Args g, const float *hidden, const float *weight, void *out) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds_x[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int part = lane >> 4, at = lane & 15;
  const int steps = mx4_steps(g.groups), n0 = blockIdx.x * 16;
  uint8_t *const room = lds_x + wave * (4 * steps * kRecord);
  float4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int j = wave; j < g.top; j += 8) {
    const size_t slot = (size_t)blockIdx.y * (size_t)g.top + j;
    const int e = g.lane_of[slot];
    if ((uint32_t)e >= (uint32_t)g.experts) continue;
    const size_t row = (size_t)e * (size_t)g.rows + (size_t)min(n0 + at, g.rows - 1);
    const uint8_t *code = g.w.code + row * g.w.code_stride, *scale = g.w.scale + row * g.w.scale_stride;
    constexpr int kAhead = 6;
    Mx4Codes w[kAhead];
    auto load = [&](int s0) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) w[u] = mx4_load(code, scale, 4 * (s0 + u) + part, g.groups);
    };
    load(0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    own_terms<false>(hidden + slot * (size_t)(32 * g.groups), g.groups, 0, 1, steps, lane, room);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the wave's own, no barrier
    float4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s0 = 0; s0 < steps; s0 += kAhead) {
      if (s0) load(s0);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (s0 + u >= steps) break;
        const int group = 4 * (s0 + u) + part;
        int as;
        const int8v_t a = own_operand(room + (4 * (s0 + u) + part) * kRecord, at < kTerms ? at : 0, as);
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx4_clear(w[u], group, g.groups), a, acc, 4, 2, 0,
                                                               group < g.groups ? w[u].scale : 0, 0, as);
      }
    }
    asm volatile("" : "+v"(acc));
    const float share = weight[slot];
#pragma unroll
    for (int d = 0; d < 4; ++d) sum[d] = __builtin_fmaf(share, acc[d], sum[d]);
  }
  __syncthreads();
  float *const sums = reinterpret_cast<float *>(lds_x);
#pragma unroll
  for (int d = 0; d < 4; ++d) sums[(wave * 16 + 4 * part + d) * 17 + at] = sum[d];
  __syncthreads();
  if (threadIdx.x >= 16 || n0 + (int)threadIdx.x >= g.rows) return;
  float v = 0.0f;
#pragma unroll
  for (int t = kTerms - 1; t >= 0; --t)
#pragma unroll
    for (int q = 0; q < 8; ++q) v += sums[(q * 16 + threadIdx.x) * 17 + t];
  const size_t to = (size_t)blockIdx.y * (size_t)g.out_stride + n0 + threadIdx.x;
  if (BF16)
    static_cast<uint16_t *>(out)[to] = float_bf16(v);
  else
    static_cast<float *>(out)[to] = v;
}

// out[lane] = sum over its choices, in their order, of weight * row of the slot's place.
// 2047 lanes of eight rows of 1536: 17 us, 6.3 TB/s of rows that the launch before wrote.
template <bool BF16>
__global__ __launch_bounds__(256) void expert_join_kernel(const float *rows, const int *place_of, const float *weight,
                                                          int top, int hidden, int lanes, void *out, long long out_stride) {
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  const int quads = hidden / 4;
  const long long lane = id / quads;
  if (lane >= lanes) return;
  const int n = 4 * (int)(id - lane * quads);
  float4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int j0 = 0; j0 < top; j0 += 8) {
    float4_t v[8];
    float w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {  // eight rows on their way at once
      const int place = j0 + j < top ? place_of[lane * top + j0 + j] : -1;
      w[j] = place >= 0 ? weight[lane * top + j0 + j] : 0.0f;
      v[j] = place >= 0 ? __builtin_nontemporal_load(reinterpret_cast<const float4_t *>(rows + (size_t)place * hidden + n))
                        : float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int d = 0; d < 4; ++d) sum[d] = __builtin_fmaf(w[j], v[j][d], sum[d]);
  }
  const size_t to = (size_t)lane * (size_t)out_stride + n;
  struct __attribute__((packed)) Half4 {
    uint16_t v[4];
  };
  if (BF16) {
    Half4 h;
#pragma unroll
    for (int d = 0; d < 4; ++d) h.v[d] = float_bf16(sum[d]);
    *reinterpret_cast<Half4 *>(static_cast<uint16_t *>(out) + to) = h;
  } else {
    Mx4Quad f;
#pragma unroll
    for (int d = 0; d < 4; ++d) f.v[d] = sum[d];
    *reinterpret_cast<Mx4Quad *>(static_cast<float *>(out) + to) = f;
  }
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

template <int T>
static size_t terms_bytes(int lanes, int cols) {
  return mx4_up((size_t)lanes * mx4_steps(cols / kMx4Group) * TermForm<T>::kStep);
}

static hipError_t launch_terms(const void *act, int bf16, long long act_stride, int lanes, int cols, uint8_t *terms,
                               hipStream_t stream) {
  const int groups = cols / kMx4Group;
  const unsigned blocks = (unsigned)(((long long)lanes * 4 * mx4_steps(groups) + 255) / 256);
  if (bf16)
    hipLaunchKernelGGL((mx4_terms_kernel<true>), dim3(blocks), dim3(256), 0, stream, act, act_stride, groups, lanes,
                       terms);
  else
    hipLaunchKernelGGL((mx4_terms_kernel<false>), dim3(blocks), dim3(256), 0, stream, act, act_stride, groups, lanes,
                       terms);
  return hipGetLastError();
}

// Bytes of packed scales of `experts` sheets of `rows`.
template <int NT, bool PAIR>
static size_t pack_bytes(int rows, int groups, int experts) {
  return mx4_up((size_t)experts * tile_blocks<NT, PAIR>(rows) * mx4_steps(groups) * 64 * NT);
}

template <int NT, bool PAIR>
static unsigned pack_blocks(int rows, int groups, int experts) {
  const long long threads = (long long)experts * tile_blocks<NT, PAIR>(rows) * ((mx4_steps(groups) + 3) / 4) * 16 * (NT / 4);
  return (unsigned)((threads + kPrepareThreads - 1) / kPrepareThreads);
}

// The launch before products of many lanes, what of it there is to do: `a` filled but for
// the workgroups' numbers.
template <int T, int NT, bool BF16>
static hipError_t launch_prepare(PrepareArgs a, hipStream_t stream) {
  long long block = a.place.experts;
  a.lane_block = (int)block;
  if (T == 0)
    block += pack_blocks<4, false>(a.lane_scales.rows, a.lane_scales.groups, 1);
  else
    block += ((long long)a.lanes * 4 * mx4_steps(a.groups) + kPrepareThreads - 1) / kPrepareThreads;
  a.pairs.first_block = (int)block;
  if (a.pairs.dst) block += pack_blocks<NT, true>(a.pairs.rows, a.pairs.groups, a.pairs.experts);
  a.rows.first_block = (int)block;
  block += pack_blocks<NT, false>(a.rows.rows, a.rows.groups, a.rows.experts);
  hipLaunchKernelGGL((mx4_prepare_kernel<T, NT, BF16>), dim3((unsigned)block), dim3(kPrepareThreads), 0, stream, a);
  return hipGetLastError();
}

template <int T, int MT, int NT, int WM, int WN, int ST, int OUT>
static hipError_t launch_tile(Mx4Args a, int tiles, int slices, hipStream_t stream) {
  using F = TileForm<T, MT, NT, WM, WN, ST>;
  static bool granted = false;  // the dynamic LDS a kernel asks for is granted once
  if (!granted) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(&mx4_tile_kernel<T, MT, NT, WM, WN, ST, OUT>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, F::lds(OUT == kOutGate));
    if (e != hipSuccess) return e;
    granted = true;
  }
  const unsigned gx = (unsigned)((tile_blocks<NT, OUT == kOutGate>(a.rows) + WN - 1) / WN);
  // grouped: one run of tiles for each of eight XCDs
  const dim3 grid = a.tiles ? dim3((gx * (unsigned)tiles + 7) / 8 * 8) : dim3(gx, (unsigned)tiles, (unsigned)slices);
  const int steps = mx4_steps(a.groups);
  a.slice = (steps + slices - 1) / slices;
  hipLaunchKernelGGL((mx4_tile_kernel<T, MT, NT, WM, WN, ST, OUT>), grid, dim3(64 * F::kWaves),
                     (size_t)F::lds(OUT == kOutGate), stream, a);
  return hipGetLastError();
}

// Slices' sums added in their order.
template <bool BF16>
__global__ __launch_bounds__(256) void mx4_fold_kernel(const float *sums, int slices, size_t slice_out, int rows, void *out,
                                                       long long out_stride) {
  const int n = blockIdx.x * 256 + threadIdx.x;
  if (n >= rows) return;
  const float *from = sums + (size_t)blockIdx.y * rows + n;
  float v = 0.0f;
#pragma unroll 8
  for (int z = 0; z < slices; ++z) v += from[(size_t)z * slice_out];
  const size_t to = (size_t)blockIdx.y * (size_t)out_stride + n;
  if (BF16)
    static_cast<uint16_t *>(out)[to] = float_bf16(v);
  else
    static_cast<float *>(out)[to] = v;
}

// A product of few lanes, sixteen a tile, its terms (if any) prepared: workgroups of 64 rows
// where they still give every CU four, of 16 below.
template <int T, int OUT>
static hipError_t launch_few(const Mx4Args &a, hipStream_t stream) {
  const int tiles = (a.lanes + 15) / 16;
  if ((long long)a.rows * tiles >= 64 * 1024)
    hipLaunchKernelGGL((mx4_few_kernel<T, 4, OUT>), dim3((a.rows + 63) / 64, tiles), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((mx4_few_kernel<T, 1, OUT>), dim3((a.rows + 15) / 16, tiles), dim3(256), 0, stream, a);
  return hipGetLastError();
}

// LDS of a step's workgroup: every wave's records of its steps, or the sums.
static size_t step_lds(int groups, int lanes, int row_tiles, int waves, int stride) {
  const size_t records = (size_t)waves * lanes * 4 * ((mx4_steps(groups) + stride - 1) / stride) * kRecord;
  const size_t sums = (size_t)waves * row_tiles * 16 * 17 * sizeof(float);
  return records > sums ? records : sums;
}

template <typename K>
static hipError_t grant_lds(K kernel, size_t bytes, size_t &granted) {
  if (bytes <= granted) return hipSuccess;
  const hipError_t e =
      hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == hipSuccess) granted = bytes;
  return e;
}

constexpr size_t kStepLds = 100 * 1024;  // a token's longest rows: one workgroup a CU still takes them
constexpr size_t kExpertLds = 150 * 1024;  // and its experts': by experts takes three times as long

template <int RT, int OUT, bool BF16>
static hipError_t launch_step(const Mx4Args &a, dim3 grid, int lanes, hipStream_t stream) {
  static size_t granted = 0;
  const size_t lds = step_lds(a.groups, lanes, RT, 4, 4);
  const hipError_t e = grant_lds(&mx4_step_kernel<RT, OUT, BF16>, kStepLds, granted);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((mx4_step_kernel<RT, OUT, BF16>), grid, dim3(256), lds, stream, a);
  return hipGetLastError();
}

constexpr size_t kHeadLds = 156 * 1024;

template <int OPERANDS, bool BF16>
static hipError_t launch_head(const Mx4Args &a, int out_bf16, hipStream_t stream) {
  static size_t granted = 0, granted16 = 0;
  const dim3 grid(min(256, ((a.rows + 15) / 16 + kHeadWaves - 1) / kHeadWaves)), block(64 * kHeadWaves);
  const size_t lds = HeadForm::lds(a.groups, a.lanes);
  hipError_t e;
  if (out_bf16) {
    if ((e = grant_lds(&mx4_head_kernel<OPERANDS, kOutBf16, BF16>, kHeadLds, granted16)) != hipSuccess) return e;
    hipLaunchKernelGGL((mx4_head_kernel<OPERANDS, kOutBf16, BF16>), grid, block, lds, stream, a);
  } else {
    if ((e = grant_lds(&mx4_head_kernel<OPERANDS, kOutF32, BF16>, kHeadLds, granted)) != hipSuccess) return e;
    hipLaunchKernelGGL((mx4_head_kernel<OPERANDS, kOutF32, BF16>), grid, block, lds, stream, a);
  }
  return hipGetLastError();
}

// What a product's lanes are, as plans and workspaces are told.
enum { kMx4Lanes = 0, kBf16Lanes = 3, kF32Lanes = 5 };

// Tiles of a product, and slices of its columns: as many as cost the least, a power of two, as
// long as fewer give less than 160 CUs a workgroup and a slice has two steps.  A step takes
// 0.7 us, the launch that adds the sums 3, sums are written and read at 4 TB/s.  37 lanes of
// floats of 2048 x 8192: 17 us in sixteen slices, 49 in one; 17 of 8192 x 2048 11.3 in eight, 17.5 in
// one; 256 microscaled lanes of 6144 x 1536, whose sums are 12 MB: 21.5 in two, 16.4 in one.
static long long mx4_tiles(int rows, int lanes, int tile_lanes, int tile_rows) {
  return (long long)((lanes + tile_lanes - 1) / tile_lanes) * ((rows + tile_rows - 1) / tile_rows);
}

static int mx4_slices(int rows, int groups, int lanes, int tile_lanes, int tile_rows) {
  const long long tiles = mx4_tiles(rows, lanes, tile_lanes, tile_rows);
  const int steps = mx4_steps(groups);
  auto cost = [&](long long s) { return 700 * steps / s + (s > 1 ? 3000 + 2 * s * lanes * rows / 1000 : 0); };
  int slices = 1;
  for (int s = 2; tiles * s < 320 && steps >= 2 * s; s *= 2)
    if (cost(s) < cost(slices)) slices = s;
  const int each = (steps + slices - 1) / slices;
  return (steps + each - 1) / each;  // none empty
}

// A product of many lanes: the launch that prepares it and the product.
template <int T, int MT, int NT, int WM, int WN, int ST, bool BF16>
static hipError_t launch_many(Mx4Args a, const void *act, int act_stride, int out_bf16, uint8_t *work, bool slice,
                              hipStream_t stream) {
  using F = TileForm<T, MT, NT, WM, WN, ST>;
  const size_t lanes_bytes =
      T == 0 ? pack_bytes<4, false>(a.lanes, a.groups, 1) : terms_bytes<T>(a.lanes, a.groups * kMx4Group);
  PrepareArgs p = {};
  p.act = act;
  p.act_stride = act_stride;
  p.groups = a.groups;
  p.lanes = a.lanes;
  p.terms = work;
  p.lane_scales = PackArgs{a.act, a.lanes, a.groups, 1, 0, work};
  p.rows = PackArgs{a.w, a.rows, a.groups, 1, 0, work + lanes_bytes};
  const size_t sums = lanes_bytes + pack_bytes<NT, false>(a.rows, a.groups, 1);
  const int tiles = (a.lanes + F::kLanes - 1) / F::kLanes;
  const int slices = slice ? mx4_slices(a.rows, a.groups, a.lanes, F::kLanes, F::kRows) : 1;
  if (sums + (slices > 1 ? (size_t)slices * a.lanes * a.rows * sizeof(float) : 0) >
      igl_mx4_work_bytes(a.rows, a.groups * kMx4Group, a.lanes, T == 0 ? kMx4Lanes : BF16 ? kBf16Lanes : kF32Lanes))
    return hipErrorInvalidValue;
  const hipError_t e = launch_prepare<T, NT, BF16>(p, stream);
  if (e != hipSuccess) return e;
  a.terms = work;
  a.term_lanes = a.lanes;
  a.lane_scales = reinterpret_cast<const uint32_t *>(work);
  a.row_scales = work + lanes_bytes;
  if (slices == 1)
    return out_bf16 ? launch_tile<T, MT, NT, WM, WN, ST, kOutBf16>(a, tiles, 1, stream)
                    : launch_tile<T, MT, NT, WM, WN, ST, kOutF32>(a, tiles, 1, stream);
  Mx4Args b = a;
  b.out = work + sums;
  b.out_stride = a.rows;
  b.slice_out = (size_t)a.lanes * a.rows;
  const hipError_t f = launch_tile<T, MT, NT, WM, WN, ST, kOutF32>(b, tiles, slices, stream);
  if (f != hipSuccess) return f;
  const dim3 grid((a.rows + 255) / 256, a.lanes);
  if (out_bf16)
    hipLaunchKernelGGL((mx4_fold_kernel<true>), grid, dim3(256), 0, stream, (const float *)b.out, slices, b.slice_out,
                       a.rows, a.out, a.out_stride);
  else
    hipLaunchKernelGGL((mx4_fold_kernel<false>), grid, dim3(256), 0, stream, (const float *)b.out, slices, b.slice_out,
                       a.rows, a.out, a.out_stride);
  return hipGetLastError();
}

// Which kernels a product of `lanes` takes.  Both sides, us:
//   * a sheet past the caches' reach, up to sixteen lanes of floats: operands of columns up to two
//     of them, else tiles of 16 lanes.  32768 x 2048: 3 lanes 16.9, a few lanes a workgroup 31
//   * few lanes: every sixteen of them and of rows read their own from the caches, and a wave
//     fetches terms for itself, so as long as these are few, and a row's chain is short: 4 lanes of
//     floats of 1536 x 6144 14.3 for 11.1 in tiles, 8 of 8192 x 2048 11.8 for 10.3, 8 of 6144 x 1536
//     9.9 for 10.7, 33 of it 17.7 for 13.7; 64 microscaled ones of it 9.4 for 12, 100 14.9 for 14.3,
//     and 8 of 32768 x 2048 13.7 for 16.2
//   * tiles as large as still give most CUs one: 2047 bf16 lanes of 8192 x 2048 75 in 64 x 256, 66 in
//     128 x 512; 512 of them 25 in 64 x 256, 30 in 32 x 256 and 51 in 128 x 512; 300 of 6144 x 1536
//     16 in 32 x 256, 18 in 64 x 256
enum { kFormFew = 0, kFormHead, kFormSmall, kFormLarge, kFormWhole, kFormTall };

constexpr long long kFewBytes = 28 << 20;

static long long mx4_bytes(int rows, int groups) { return (long long)rows * groups * 17; }

static int mx4_form(int rows, int groups, int lanes, int kind) {
  const int steps = mx4_steps(groups);
  const long long bytes = mx4_bytes(rows, groups);
  if (kind != kMx4Lanes && lanes <= 16 && rows >= 32768 && bytes >= kFewBytes)
    return HeadForm::operands(lanes) <= 2 && groups >= 16 && HeadForm::lds(groups, lanes) <= kHeadLds ? kFormHead : kFormTall;
  const long long few = mx4_tiles(rows, lanes, 16, 16) * steps;
  if (kind != kMx4Lanes ? few < 6000 && steps <= 24 : few < (lanes <= 16 ? 38000 : 24000)) return kFormFew;
  if (kind == kBf16Lanes && lanes > 64 && mx4_tiles(rows, lanes, 128, 512) >= 192) return kFormWhole;
  const bool large = kind == kF32Lanes    ? lanes > 32 && mx4_tiles(rows, lanes, 64, 512) >= 192
                     : kind == kBf16Lanes ? lanes > 32 && mx4_tiles(rows, lanes, 64, 256) >= 192
                                          : lanes > 64 && mx4_tiles(rows, lanes, 128, 256) >= 192;
  return large ? kFormLarge : kFormSmall;
}

// A token's step: its kernel cuts the lanes itself.
static bool mx4_single(int rows, int groups, int lanes, int form, int kind) {
  return kind != kMx4Lanes && form != kFormHead && lanes <= 3 && (lanes == 1 || mx4_bytes(rows, groups) < kFewBytes) &&
         step_lds(groups, lanes, 1, 4, 4) <= kStepLds;
}

// What a product's form uses: its lanes as terms, or their scales, the sheet's scales packed (eight
// tiles a block at most), and slices' sums; a token's step and a head nothing.
extern "C" size_t igl_mx4_work_bytes(int rows, int cols, int lanes, int kind) {
  const int groups = cols / kMx4Group, form = mx4_form(rows, groups, lanes, kind);
  const bool plain = kind == kBf16Lanes && form != kFormFew;
  const size_t of_lanes = kind == kMx4Lanes ? pack_bytes<4, false>(lanes, groups, 1)
                          : plain           ? terms_bytes<kPlain>(lanes, cols)
                                            : terms_bytes<kTerms>(lanes, cols);
  if (form == kFormHead || mx4_single(rows, groups, lanes, form, kind)) return 0;
  if (form == kFormFew) return kind == kMx4Lanes ? 0 : of_lanes;
  const int slices = form == kFormSmall ? mx4_slices(rows, groups, lanes, kind == kMx4Lanes ? 64 : 32, 256) : 1;
  return of_lanes + pack_bytes<8, false>(rows, groups, 1) +
         (slices > 1 ? mx4_up((size_t)slices * lanes * rows * sizeof(float)) : 0);
}

// A product of lanes of floats, by its form.
template <bool BF16>
static hipError_t launch_floats(Mx4Args a, const void *act, int act_stride, int out_bf16, uint8_t *room, hipStream_t stream) {
  constexpr int kKind = BF16 ? kBf16Lanes : kF32Lanes;
  const int form = mx4_form(a.rows, a.groups, a.lanes, kKind);
  a.act_rows = act;
  a.act_stride = act_stride;
  if (mx4_single(a.rows, a.groups, a.lanes, form, kKind)) {
    const dim3 grid((a.rows + 15) / 16);
    return out_bf16 ? launch_step<1, kOutBf16, BF16>(a, grid, a.lanes, stream)
                    : launch_step<1, kOutF32, BF16>(a, grid, a.lanes, stream);
  }
  if (form == kFormHead)
    return HeadForm::operands(a.lanes) == 1 ? launch_head<1, BF16>(a, out_bf16, stream)
                                            : launch_head<2, BF16>(a, out_bf16, stream);
  constexpr int kForm = BF16 ? kPlain : kTerms;  // of a lane in tiles
  if (form == kFormTall) return launch_many<kForm, 1, 4, 1, 4, 3, BF16>(a, act, act_stride, out_bf16, room, false, stream);
  if (form == kFormSmall) return launch_many<kForm, 1, 4, 2, 4, 3, BF16>(a, act, act_stride, out_bf16, room, true, stream);
  if constexpr (BF16) {
    if (form == kFormLarge) return launch_many<kPlain, 2, 4, 2, 4, 2, true>(a, act, act_stride, out_bf16, room, false, stream);
    if (form == kFormWhole) return launch_many<kPlain, 4, 8, 2, 4, 2, true>(a, act, act_stride, out_bf16, room, false, stream);
  } else {
    if (form == kFormLarge) return launch_many<kTerms, 2, 8, 2, 4, 2, false>(a, act, act_stride, out_bf16, room, false, stream);
  }
  const hipError_t e = launch_terms(act, BF16, act_stride, a.lanes, a.groups * kMx4Group, room, stream);
  if (e != hipSuccess) return e;
  a.terms = room;
  a.term_lanes = a.lanes;
  return out_bf16 ? launch_few<kTerms, kOutBf16>(a, stream) : launch_few<kTerms, kOutF32>(a, stream);
}

extern "C" hipError_t igl_launch_mx4_mat_mat(const igl_mx4 *sheet, const void *act, int act_bf16, int act_stride,
                                             int lanes, void *out, int out_bf16, int out_stride, void *work,
                                             hipStream_t stream) {
  Mx4Args a = {};
  a.w = mx4_view(sheet, 0);
  a.rows = sheet->row_count;
  a.groups = sheet->col_count / kMx4Group;
  a.lanes = lanes;
  a.out = out;
  a.out_stride = out_stride;
  uint8_t *const room = static_cast<uint8_t *>(work);
  return act_bf16 ? launch_floats<true>(a, act, act_stride, out_bf16, room, stream)
                  : launch_floats<false>(a, act, act_stride, out_bf16, room, stream);
}

extern "C" hipError_t igl_launch_mx4_mat_mx4(const igl_mx4 *sheet, const igl_mx4 *act, int lane_first, int lanes,
                                             void *out, int out_bf16, int out_stride, void *work, hipStream_t stream) {
  Mx4Args a = {};
  a.w = mx4_view(sheet, 0);
  a.rows = sheet->row_count;
  a.groups = sheet->col_count / kMx4Group;
  a.act = mx4_view(act, lane_first);
  a.lanes = lanes;
  a.out = out;
  a.out_stride = out_stride;
  const int form = mx4_form(a.rows, a.groups, lanes, kMx4Lanes);
  if (form == kFormSmall)
    return launch_many<0, 4, 4, 1, 4, 3, false>(a, nullptr, 0, out_bf16, static_cast<uint8_t *>(work), true, stream);
  if (form == kFormLarge)
    return launch_many<0, 4, 4, 2, 4, 2, false>(a, nullptr, 0, out_bf16, static_cast<uint8_t *>(work), false, stream);
  return out_bf16 ? launch_few<0, kOutBf16>(a, stream) : launch_few<0, kOutF32>(a, stream);
}

namespace igl {

// The places of a call's experts, its lanes' and hidden values' terms, packed scales, and
// the rows that are joined.
struct ExpertRoom {
  size_t lane_of, place_of, tiles, x, gate_up, down, h, rows, end;
};

constexpr int kExpertTile = 16;  // lanes of the smallest tile

static int expert_tiles(int slots, int experts, int tile) { return slots / tile + experts; }

static ExpertRoom expert_room(const igl_experts *x, int lanes, int top, int /* lanes of either type: terms are the most */) {
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
  r.tiles = take((size_t)expert_tiles((int)slots, x->expert_count, kExpertTile) * sizeof(Mx4Tile));
  r.x = take(terms_bytes<kTerms>(lanes, x->hidden));
  r.gate_up = take(pack_bytes<8, true>(2 * x->inner, x->hidden / kMx4Group, x->expert_count));
  r.down = take(pack_bytes<8, false>(x->hidden, x->inner / kMx4Group, x->expert_count));
  r.h = take(terms_bytes<kTerms>((int)slots, x->inner));
  r.rows = take(slots * x->hidden * sizeof(float));
  r.end = at;
  return r;
}

// Whether a call's slots are taken one by one.  That reads an expert's weights for each, by
// experts takes two launches more: up to a count, and while what is read twice (slots^2 /
// (experts + slots) of them where picks are even) is less than those launches.  48 slots of 64
// experts 34 us for 39, 64 of 128 42 for 46, 32 of eight 26 for 24; 32 of sixteen of 13 MB
// each 165 for 59
static bool expert_steps(const igl_experts *x, int slots) {
  const long long expert_bytes = 3LL * x->hidden * x->inner * 17 / 32;
  return slots <= 64 && slots <= 20 + x->expert_count / 2 &&
         slots * expert_bytes / (x->expert_count + slots) < (50 << 20) / slots &&
         step_lds(x->hidden / kMx4Group, 1, 2, 4, 4) <= kStepLds && step_lds(x->inner / kMx4Group, 1, 1, 8, 1) <= kExpertLds;
}

// Tiles of as many places as an expert has, while smaller ones are more than two workgroups a
// CU: 12 of 64 experts 45 us in 32s and 51 in 16s, 16 of 128 77 and 84, but 16 of 32 49 and 45;
// 64 of eight small ones 24 in 16s and 26 in 32s.  In 64s, of which an expert's last is nearly
// empty, bf16 lanes win from 60 on (62 of 16 72 and 75 in 32s, 128 of 128 247 and 261; 56 of 64
// 89 and 79), fp32 ones, whose tiles of 64 leave a CU one workgroup, from 250 (125 of 32 140 and 116,
// 256 of 128 472 and 483).
static int expert_tile(const igl_experts *x, int slots, int bf16) {
  const int each = slots / x->expert_count, blocks = (2 * x->inner + 255) / 256;
  auto groups = [&](int tile) { return (long long)expert_tiles(slots, x->expert_count, tile) * blocks; };
  return each >= (bf16 ? 60 : 250) && groups(32) >= 520 ? 64 : each >= 12 && groups(16) >= 520 ? 32 : 16;
}

// What an experts' call is: its arguments and its room.
struct ExpertCall {
  const igl_experts *x;
  const void *act;
  int act_stride, lanes;
  const int32_t *pick;
  const float *weight;
  int top;
  void *out;
  int out_bf16, out_stride;
  uint8_t *base;
  ExpertRoom room;
};

template <int T, int MT, int NT, int WM, int WN, int ST, bool BF16>
static hipError_t experts_grouped(const ExpertCall &c, hipStream_t stream) {
  using F = TileForm<T, MT, NT, WM, WN, ST>;
  const igl_experts *x = c.x;
  const ExpertRoom &r = c.room;
  const int slots = c.lanes * c.top, tiles = expert_tiles(slots, x->expert_count, F::kLanes);
  hipError_t e;
  PrepareArgs p = {};
  p.act = c.act;
  p.act_stride = c.act_stride;
  p.groups = x->hidden / kMx4Group;
  p.lanes = c.lanes;
  p.terms = c.base + r.x;
  p.place = PlaceArgs{c.pick, slots, x->expert_count, F::kLanes, place_inverse(c.top), (int *)(c.base + r.lane_of),
                      (int *)(c.base + r.place_of), (Mx4Tile *)(c.base + r.tiles)};
  p.pairs = PackArgs{mx4_view(&x->gate_up, 0), 2 * x->inner, p.groups, x->expert_count, 0, c.base + r.gate_up};
  p.rows = PackArgs{mx4_view(&x->down, 0), x->hidden, x->inner / kMx4Group, x->expert_count, 0, c.base + r.down};
  if ((e = launch_prepare<T, NT, BF16>(p, stream)) != hipSuccess) return e;
  Mx4Args a = {};
  a.w = p.pairs.w;
  a.rows = p.pairs.rows;
  a.groups = p.groups;
  a.terms = p.terms;
  a.term_lanes = c.lanes;
  a.tiles = p.place.tiles;
  a.tile_count = tiles;
  a.lane_of = p.place.lane_of;
  a.row_scales = p.pairs.dst;
  a.out = c.base + r.h;
  a.out_stride = slots;
  a.silu = x->gate == IGL_GATE_SILU;
  if ((e = launch_tile<T, MT, NT, WM, WN, ST, kOutGate>(a, tiles, 1, stream)) != hipSuccess) return e;
  a.w = p.rows.w;
  a.rows = p.rows.rows;
  a.groups = p.rows.groups;
  a.terms = c.base + r.h;
  a.term_lanes = slots;
  a.lane_of = nullptr;
  a.row_scales = p.rows.dst;
  a.out = c.base + r.rows;
  a.out_stride = x->hidden;
  if ((e = launch_tile<kTerms, MT, NT, WM, WN, ST, kOutF32>(a, tiles, 1, stream)) != hipSuccess) return e;
  const unsigned blocks = (unsigned)(((long long)c.lanes * (x->hidden / 4) + 255) / 256);
  if (c.out_bf16)
    hipLaunchKernelGGL((expert_join_kernel<true>), dim3(blocks), dim3(256), 0, stream, (const float *)(c.base + r.rows),
                       p.place.place_of, c.weight, c.top, x->hidden, c.lanes, c.out, c.out_stride);
  else
    hipLaunchKernelGGL((expert_join_kernel<false>), dim3(blocks), dim3(256), 0, stream, (const float *)(c.base + r.rows),
                       p.place.place_of, c.weight, c.top, x->hidden, c.lanes, c.out, c.out_stride);
  return hipGetLastError();
}

// A few lanes' experts, a slot at a time: gate and up, then down and the sum, two launches.
template <bool BF16>
static hipError_t experts_step(const ExpertCall &c, hipStream_t stream) {
  static size_t granted = 0;
  const igl_experts *x = c.x;
  Mx4Args a = {};
  a.w = mx4_view(&x->gate_up, 0);
  a.rows = 2 * x->inner;
  a.groups = x->hidden / kMx4Group;
  a.lanes = c.lanes;
  a.lane_of = c.pick;
  a.act_rows = c.act;
  a.act_stride = c.act_stride;
  a.experts = x->expert_count;
  a.top = c.top;
  a.silu = x->gate == IGL_GATE_SILU;
  a.out = c.base;  // hidden values as floats, all it keeps
  hipError_t e = launch_step<2, kOutGate, BF16>(a, dim3((x->inner + 15) / 16, c.lanes * c.top), 1, stream);
  if (e != hipSuccess) return e;
  a.w = mx4_view(&x->down, 0);
  a.rows = x->hidden;
  a.groups = x->inner / kMx4Group;
  a.out_stride = c.out_stride;
  const size_t lds = step_lds(a.groups, 1, 1, 8, 1);
  const dim3 grid((x->hidden + 15) / 16, c.lanes);
  if (c.out_bf16) {
    static size_t granted16 = 0;
    if ((e = grant_lds(&expert_step_kernel<true>, kExpertLds, granted16)) != hipSuccess) return e;
    hipLaunchKernelGGL((expert_step_kernel<true>), grid, dim3(512), lds, stream, a, (const float *)c.base,
                       c.weight, c.out);
  } else {
    if ((e = grant_lds(&expert_step_kernel<false>, kExpertLds, granted)) != hipSuccess) return e;
    hipLaunchKernelGGL((expert_step_kernel<false>), grid, dim3(512), lds, stream, a, (const float *)c.base,
                       c.weight, c.out);
  }
  return hipGetLastError();
}

}  // namespace igl

extern "C" size_t igl_experts_work_bytes(const igl_experts *x, int lanes, int top, int act_bf16) {
  return expert_steps(x, lanes * top) ? mx4_up((size_t)lanes * top * x->inner * sizeof(float))
                                      : expert_room(x, lanes, top, act_bf16).end;
}

extern "C" hipError_t igl_launch_experts(const igl_experts *x, const void *act, int act_bf16, int act_stride, int lanes,
                                         const int32_t *pick, const float *weight, int top, void *out, int out_bf16,
                                         int out_stride, void *work, hipStream_t stream) {
  const ExpertCall c = {x,   act,      act_stride, lanes, pick, weight, top,
                        out, out_bf16, out_stride, static_cast<uint8_t *>(work), expert_room(x, lanes, top, act_bf16)};
  const int slots = lanes * top;
  if (expert_steps(x, slots)) return act_bf16 ? experts_step<true>(c, stream) : experts_step<false>(c, stream);
  const int tile = expert_tile(x, slots, act_bf16);
  if (act_bf16)
    return tile == 64   ? experts_grouped<kPlain, 2, 4, 2, 4, 2, true>(c, stream)
           : tile == 32 ? experts_grouped<kPlain, 1, 4, 2, 4, 2, true>(c, stream)
                        : experts_grouped<kPlain, 1, 4, 1, 4, 3, true>(c, stream);
  if (tile == 64) return experts_grouped<kTerms, 2, 8, 2, 4, 2, false>(c, stream);
  if (tile == 32) return experts_grouped<kTerms, 1, 4, 2, 4, 2, false>(c, stream);
  return experts_grouped<kTerms, 1, 4, 1, 4, 3, false>(c, stream);
}
