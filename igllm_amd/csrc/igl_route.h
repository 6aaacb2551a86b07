// igl_route.h - the choice of experts, gfx950: scores of a lane's logits, a bias for
// balance, groups of experts, the best of the kept groups, their weights.
//
//     s_e = softmax(x)_e or 1 / (1 + e^-x_e),   c_e = s_e + bias_e
//     a group's score is the sum of its largest one or two c; the best groups stay
//     the chosen are the largest c among them, the lowest index first where equal
//     w = s of the chosen (over their sum), times the rule's gain and the expert's
// A choice next to another's must fall as the reals' does, so scores are formed and
// compared in double.  Without a bias and groups s rises with x, and x decides, also where
// scores are one double (sigmoid's 1 of logits above 37).
#pragma once

#include <type_traits>

#include "igl_device.h"
#include "igl_launch.h"

namespace igl {

constexpr int kRouteWaves = 4;  // lanes of a batch a workgroup, a wave each

struct RouteArgs {
  igl_route rule;
  const float *logits;
  long long logit_stride;
  int lanes;
  const float *bias, *gain;
  int32_t *pick;
  float *weight;
  uint32_t each_inverse;  // of a group's experts: e / each = e * each_inverse >> 20 for e < 1024
};

// e^x in double: x = k ln 2 + r, |r| <= 0.35, the series of e^r to the thirteenth power
// (what is left out is below 2^-57 of it), times 2^k.  x not above 1024; 0 far below, and of
// a NaN.  No branch: a wave has its experts' exponentials on their way side by side.
__device__ __forceinline__ double exp_f64(double x) {
  x = fmax(x, -1100.0);
  const double k = __builtin_rint(x * 1.4426950408889634);
  double r = __builtin_fma(k, -0.69314718036912382, x);  // ln 2 in two pieces, the first of 32 bits: k times it is exact
  r = __builtin_fma(k, -1.9082149292705877e-10, r);
  double p = 1.0 / 6227020800.0;
  p = __builtin_fma(p, r, 1.0 / 479001600.0);
  p = __builtin_fma(p, r, 1.0 / 39916800.0);
  p = __builtin_fma(p, r, 1.0 / 3628800.0);
  p = __builtin_fma(p, r, 1.0 / 362880.0);
  p = __builtin_fma(p, r, 1.0 / 40320.0);
  p = __builtin_fma(p, r, 1.0 / 5040.0);
  p = __builtin_fma(p, r, 1.0 / 720.0);
  p = __builtin_fma(p, r, 1.0 / 120.0);
  p = __builtin_fma(p, r, 1.0 / 24.0);
  p = __builtin_fma(p, r, 1.0 / 6.0);
  p = __builtin_fma(p, r, 0.5);
  p = __builtin_fma(p, r, 1.0);
  p = __builtin_fma(p, r, 1.0);
  return __builtin_ldexp(p, (int)k);
}

// 1 / d, d in [1, infinity]: the hardware's estimate and two Newton steps.
__device__ __forceinline__ double recip_f64(double d) {
  double r = __builtin_amdgcn_rcp(d);
  r = __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
  r = __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
  return d < __builtin_inf() ? r : 0.0;
}

// A number's bits so that they order as it does, above 0 for all but a NaN.
__device__ __forceinline__ uint64_t route_key(double c) {
  const uint64_t u = __builtin_bit_cast(uint64_t, c);
  return u >> 63 ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ uint32_t route_key(float c) {
  const uint32_t u = __builtin_bit_cast(uint32_t, c);
  return u >> 31 ? ~u : u | 1u << 31;
}

// The largest of a wave's numbers, in every lane: a word at a time along the rows of a wave.
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
  auto step = [&](int moved) { v = max(v, (uint32_t)moved); };
  step(__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true));   // quad_perm [1,0,3,2]
  step(__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true));   // quad_perm [2,3,0,1]
  step(__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, true));  // row_half_mirror
  step(__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, true));  // row_mirror
  step(__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, true));  // row_bcast:15
  step(__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, true));  // row_bcast:31
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// The lanes that hold the wave's largest key.
__device__ __forceinline__ uint64_t route_best(uint32_t key, bool &any) {
  const uint32_t top = wave_max_u32(key);
  any = top > 0;
  return __ballot(key == top);
}
__device__ __forceinline__ uint64_t route_best(uint64_t key, bool &any) {
  const uint32_t high = (uint32_t)(key >> 32), top = wave_max_u32(high);
  any = top > 0;
  uint64_t at = __ballot(high == top);
  if (at & (at - 1)) {  // upper words are seldom equal
    const uint32_t low = high == top ? (uint32_t)key : 0u, rest = wave_max_u32(low);
    at = __ballot(high == top && low == rest);
  }
  return at;
}

// A wave a lane of the batch; wave lane l holds experts PER l .. PER l + PER - 1, so that
// of equal ones the lowest lane's is the lowest.  WIDE: choices are doubles (a bias, or
// groups); else the logits.  What may not be chosen has key 0.
template <int PER, bool WIDE>
__global__ __launch_bounds__(64 * kRouteWaves) void route_kernel(RouteArgs a) {
  using Key = typename std::conditional<WIDE, uint64_t, uint32_t>::type;
  __shared__ double room[WIDE ? kRouteWaves : 1][WIDE ? 64 * PER : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long m = (long long)blockIdx.x * kRouteWaves + wave;
  if (m >= a.lanes) return;  // a wave's own from here on, no barrier
  const int E = a.rule.expert_count, first = PER * lane;
  const float *x = a.logits + m * a.logit_stride;
  const double none = -__builtin_inf();
  float v[PER];
  float top = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < PER; ++i) v[i] = x[min(first + i, E - 1)];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (first + i >= E || !(v[i] >= -3.402823466e38f)) v[i] = -__builtin_inff();  // a NaN is never chosen
    v[i] = fminf(v[i], 3.402823466e38f) + 0.0f;  // a zero without its sign: keys are bits
    top = fmaxf(top, v[i]);
  }
  const bool soft = a.rule.score == IGL_ROUTE_SOFTMAX;
  double sum = 1.0;  // of the exponentials, where it is asked for
  if (soft) {
    const uint32_t key = wave_max_u32(route_key(top));  // at least minus infinity's
    top = __builtin_bit_cast(float, key >> 31 ? key & 0x7FFFFFFFu : ~key);
  }
  // s before softmax's division, 0 of minus infinity; where the logits decide, only of the chosen
  auto share_of = [&](float t) { return exp_f64((double)t - (double)top); };
  auto sigmoid = [&](float t) { return recip_f64(1.0 + exp_f64(fmin(-(double)t, 800.0))); };
  double s[WIDE ? PER : 1];
  Key key[PER];
  if (soft && (WIDE || !a.rule.renorm)) {
    sum = 0.0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const double t = share_of(v[i]);
      if constexpr (WIDE) s[i] = t;
      sum += t;
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
    sum = sum > 0.0 ? sum : 1.0;
  } else if constexpr (WIDE) {
#pragma unroll
    for (int i = 0; i < PER; ++i) s[i] = sigmoid(v[i]);
  }
  if constexpr (WIDE) {
    const double inverse = soft ? 1.0 / sum : 1.0;
    double c[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      s[i] *= inverse;
      c[i] = v[i] == -__builtin_inff() ? none : s[i] + (a.bias ? (double)a.bias[min(first + i, E - 1)] : 0.0);
      if (!(c[i] > none)) c[i] = none;  // and a bias that is a NaN
    }
    uint64_t kept = ~0ull;
    if (a.rule.group_count > 1) {
      const int each = E / a.rule.group_count;
      double group_score = none;
#pragma unroll
      for (int i = 0; i < PER; ++i) room[wave][first + i] = c[i];
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      const int lanes_each = each / PER;
      if (each % PER == 0 && (lanes_each & (lanes_each - 1)) == 0) {
        // a group is a run of lanes, a power of two: the two largest of each, merged
        double most = none, second = none;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          second = fmax(second, fmin(most, c[i]));
          most = fmax(most, c[i]);
        }
        for (int d = 1; d < lanes_each; d *= 2) {
          const double other = __shfl_xor(most, d), other_second = __shfl_xor(second, d);
          second = fmax(fmin(most, other), fmax(second, other_second));
          most = fmax(most, other);
        }
        const double of_group = a.rule.group_best == 2 && second > none ? most + second : most;
        group_score = __shfl(of_group, min(lane * lanes_each, 63));
      } else if (lane < a.rule.group_count) {
        double most = none, second = none;
        for (int i = 0; i < each; ++i) {
          const double t = room[wave][lane * each + i];
          second = fmax(second, fmin(most, t));
          most = fmax(most, t);
        }
        group_score = a.rule.group_best == 2 && second > none ? most + second : most;
      }
      if (lane >= a.rule.group_count) group_score = none;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      room[wave][lane] = group_score;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      // a group stays if fewer than group_top come before it
      int ahead = 0;
#pragma unroll 8
      for (int q = 0; q < a.rule.group_count; ++q) {
        const double other = room[wave][q];
        ahead += other > group_score || (other == group_score && q < lane);
      }
      kept = __ballot(ahead < a.rule.group_top && group_score > none);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const bool in = a.rule.group_count == 1 || (kept >> ((uint32_t)(first + i) * a.each_inverse >> 20 & 63) & 1);
      key[i] = in && c[i] > none ? route_key(c[i]) : 0;
    }
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) key[i] = v[i] == -__builtin_inff() ? 0 : route_key(v[i]);
  }
  // the best, one at a time; wave lane j keeps the j-th's
  int mine = -1;
  double share = 0.0, total = 0.0;
  for (int j = 0; j < a.rule.top; ++j) {
    Key best = key[0];
    int at = 0;
#pragma unroll
    for (int i = 1; i < PER; ++i)
      if (key[i] > best) best = key[i], at = i;
    bool any;
    const int from = __builtin_ctzll(route_best(best, any));
    if (!any) break;
    const int slot = __builtin_amdgcn_readlane(at, from);
    double taken = 0.0;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (i == slot) {
        if constexpr (WIDE) taken = s[i];
        if (lane == from) key[i] = 0;
      }
    if constexpr (WIDE) {
      const uint64_t bits = __builtin_bit_cast(uint64_t, taken);
      const uint32_t low = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)bits, from);
      const uint32_t high = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(bits >> 32), from);
      taken = __builtin_bit_cast(double, (uint64_t)high << 32 | low);
      total += taken;
    }
    if (lane == j) mine = PER * from + slot, share = taken;
  }
  if constexpr (!WIDE) {
    if (mine >= 0) {
      const float t = fminf(x[mine], 3.402823466e38f);
      share = soft ? share_of(t) / sum : sigmoid(t);
    }
    total = share;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) total += __shfl_xor(total, d);
  }
  if (lane >= a.rule.top) return;
  if (a.rule.renorm) share = total > 0.0 ? share / total : 0.0;
  share *= (double)a.rule.gain_scale;
  if (a.gain && mine >= 0) share *= (double)a.gain[mine];
  a.pick[m * a.rule.top + lane] = mine;
  a.weight[m * a.rule.top + lane] = mine >= 0 ? (float)share : 0.0f;
}

// The largest, or least, of each row of sixteen wave lanes, in all of them.
__device__ __forceinline__ uint32_t row_max_u32(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, true));
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, true));
}
__device__ __forceinline__ uint32_t row_min_u32(uint32_t v) { return ~row_max_u32(~v); }

// Many lanes of a batch: four a wave, sixteen wave lanes each, so that a round of the choice
// serves four: 16383 lanes of 256 experts, eight groups of which four stay, 21 us where
// a wave a lane takes 27 (2048 lanes 11.5 and 12).  Vector issue is half of a SIMD's
// cycles: 2100 instructions a wave, 750 of them the eight rounds, 650 the exponentials in
// double; the logits are 3.4 us of a copy.  Wave lane l of a row holds experts 64 q + 4 l + 0 .. 3, a quad each
// of PER / 4.  E a multiple of four, sixteen choices and groups at most.
template <int PER, bool WIDE>
__global__ __launch_bounds__(64 * kRouteWaves) void route_rows_kernel(RouteArgs a) {
  __shared__ double room[WIDE ? kRouteWaves : 1][WIDE ? 64 * PER : 1];  // choices, then scores, of four rows
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, row = lane >> 4;
  const long long m0 = ((long long)blockIdx.x * kRouteWaves + wave) * 4;
  if (m0 >= a.lanes) return;  // a wave's own from here on, no barrier
  const long long m = min(m0 + row, (long long)a.lanes - 1);
  const int E = a.rule.expert_count;
  const float *x = a.logits + m * a.logit_stride;
  const double none = -__builtin_inf();
  struct __attribute__((packed)) Quad {
    float v[4];
  };
  auto load = [&](const float *from, float (&to)[PER]) {
#pragma unroll
    for (int q = 0; q < PER / 4; ++q) {
      const Quad f = *reinterpret_cast<const Quad *>(from + min(64 * q + 4 * l, E - 4));
#pragma unroll
      for (int d = 0; d < 4; ++d) to[4 * q + d] = f.v[d];
    }
  };
  auto expert = [&](int i) { return 64 * (i / 4) + 4 * l + i % 4; };
  float v[PER], bias[WIDE ? PER : 4] = {};
  load(x, v);
  if constexpr (WIDE)
    if (a.bias) load(a.bias, bias);
  float top = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (expert(i) >= E || !(v[i] >= -3.402823466e38f)) v[i] = -__builtin_inff();  // a NaN is never chosen
    v[i] = fminf(v[i], 3.402823466e38f) + 0.0f;  // a zero without its sign: keys are bits
    top = fmaxf(top, v[i]);
  }
  const bool soft = a.rule.score == IGL_ROUTE_SOFTMAX;
  if (soft) {
    const uint32_t key = row_max_u32(route_key(top));
    top = __builtin_bit_cast(float, key >> 31 ? key & 0x7FFFFFFFu : ~key);
  }
  auto share_of = [&](float t) { return exp_f64((double)t - (double)top); };
  auto sigmoid = [&](float t) { return recip_f64(1.0 + exp_f64(fmin(-(double)t, 800.0))); };
  double s[WIDE ? PER : 1], sum = 1.0;
  uint32_t key[PER], low[WIDE ? PER : 1];  // keys' upper words, 0 of what may not be chosen, and lower ones
  if (soft && (WIDE || !a.rule.renorm)) {
    double of_all = 0.0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const double t = share_of(v[i]);
      if constexpr (WIDE) s[i] = t;
      of_all += t;
    }
#pragma unroll
    for (int d = 1; d < 16; d *= 2) of_all += __shfl_xor(of_all, d);
    sum = of_all > 0.0 ? of_all : 1.0;
  } else if constexpr (WIDE) {
#pragma unroll
    for (int i = 0; i < PER; ++i) s[i] = sigmoid(v[i]);
  }
  if constexpr (WIDE) {
    double *const mine = room[wave] + row * 16 * PER;
    const double inverse = 1.0 / sum;
    double c[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      s[i] *= inverse;
      c[i] = v[i] == -__builtin_inff() ? none : s[i] + (double)bias[i];
      if (!(c[i] > none)) c[i] = none;  // and a bias that is a NaN
    }
    uint32_t kept = ~0u;
    if (a.rule.group_count > 1) {
      const int G = a.rule.group_count, each = E / G;
#pragma unroll
      for (int i = 0; i < PER; ++i) mine[expert(i)] = c[i];
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      // a group's two largest, by `split` wave lanes, which begin at different experts
      const int split = G <= 2 ? 8 : G <= 4 ? 4 : G <= 8 ? 2 : 1;
      const int group = l / split, part = l % split, n = (each - part + split - 1) / split;
      double most = none, second = none;
      if (group < G && n > 0) {
        const int from = lane % n;
#pragma unroll 8
        for (int i = 0; i < n; ++i) {
          const int at = from + i < n ? from + i : from + i - n;
          const double t = mine[group * each + part + split * at];
          second = fmax(second, fmin(most, t));
          most = fmax(most, t);
        }
      }
      for (int d = 1; d < split; d *= 2) {
        const double other = __shfl_xor(most, d), other_second = __shfl_xor(second, d);
        second = fmax(fmin(most, other), fmax(second, other_second));
        most = fmax(most, other);
      }
      double score_of = a.rule.group_best == 2 && second > none ? most + second : most;
      score_of = __shfl(score_of, 16 * row + min(l * split, 15));
      if (l >= G) score_of = none;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      mine[l] = score_of;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      // a group stays if fewer than group_top come before it
      int ahead = 0;
#pragma unroll 8
      for (int q = 0; q < G; ++q) {
        const double other = mine[q];
        ahead += other > score_of || (other == score_of && q < l);
      }
      kept = (uint32_t)(__ballot(ahead < a.rule.group_top && score_of > none) >> (16 * row)) & 0xFFFFu;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) mine[expert(i)] = s[i];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const bool in = a.rule.group_count == 1 || (kept >> ((uint32_t)expert(i) * a.each_inverse >> 20 & 31) & 1);
      const uint64_t k = route_key(c[i]);
      key[i] = in && c[i] > none ? (uint32_t)(k >> 32) : 0;
      low[i] = (uint32_t)k;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) key[i] = v[i] == -__builtin_inff() ? 0 : route_key(v[i]);
  }
  // the best, one at a time, by upper words; wave lane j of a row keeps the j-th's
  int chosen = -1;
  for (int j = 0; j < a.rule.top; ++j) {
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) word = max(word, key[i]);
    const uint32_t most = row_max_u32(word);
    uint32_t at = ~0u;
    int holders = 0;
#pragma unroll
    for (int i = PER - 1; i >= 0; --i) {
      const bool holds = key[i] == most;
      at = holds ? 64 * (i / 4) + i % 4 : at;
      if (WIDE) holders += __builtin_popcountll(__ballot(holds));
    }
    if (WIDE && holders > 4) {  // upper words are seldom equal
      uint32_t rest = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) rest = max(rest, key[i] == most ? low[WIDE ? i : 0] : 0u);
      rest = row_max_u32(rest);
      at = ~0u;
#pragma unroll
      for (int i = PER - 1; i >= 0; --i) at = key[i] == most && low[WIDE ? i : 0] == rest ? 64 * (i / 4) + i % 4 : at;
    }
    const int e = (int)row_min_u32(at != ~0u ? at + 4 * l : ~0u);  // of equal ones the lowest
    if (__ballot(most > 0) == 0) break;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (e - 4 * l == 64 * (i / 4) + i % 4) key[i] = 0;
    if (l == j && most > 0) chosen = e;
  }
  double share = 0.0, total;
  if (chosen >= 0) {
    const float t = fminf(x[chosen], 3.402823466e38f);
    share = WIDE ? room[wave][WIDE ? row * 16 * PER + chosen : 0] : soft ? share_of(t) / sum : sigmoid(t);
  }
  total = share;
#pragma unroll
  for (int d = 1; d < 16; d *= 2) total += __shfl_xor(total, d);
  if (l >= a.rule.top || m0 + row >= a.lanes) return;
  if (a.rule.renorm) share = total > 0.0 ? share / total : 0.0;
  share *= (double)a.rule.gain_scale;
  if (a.gain && chosen >= 0) share *= (double)a.gain[chosen];
  a.pick[m * a.rule.top + l] = chosen;
  a.weight[m * a.rule.top + l] = chosen >= 0 ? (float)share : 0.0f;
}

template <int PER>
static hipError_t launch_route_rows(const RouteArgs &a, hipStream_t stream) {
  const dim3 grid((unsigned)((a.lanes + 4 * kRouteWaves - 1) / (4 * kRouteWaves))), block(64 * kRouteWaves);
  if (a.bias || a.rule.group_count > 1)
    hipLaunchKernelGGL((route_rows_kernel<PER, true>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((route_rows_kernel<PER, false>), grid, block, 0, stream, a);
  return hipGetLastError();
}

template <int PER>
static hipError_t launch_route(const RouteArgs &a, hipStream_t stream) {
  const dim3 grid((unsigned)((a.lanes + kRouteWaves - 1) / kRouteWaves)), block(64 * kRouteWaves);
  if (a.bias || a.rule.group_count > 1)
    hipLaunchKernelGGL((route_kernel<PER, true>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((route_kernel<PER, false>), grid, block, 0, stream, a);
  return hipGetLastError();
}

}  // namespace igl

extern "C" hipError_t igl_launch_route(const igl_route *rule, const float *logits, int logit_stride, int lanes,
                                       const float *bias, const float *gain, int32_t *pick, float *weight,
                                       hipStream_t stream) {
  const int each = rule->expert_count / rule->group_count;
  const igl::RouteArgs a = {*rule, logits, logit_stride, lanes, bias, gain, pick, weight,
                            (uint32_t)(((1 << 20) + each - 1) / each)};
  if (lanes >= 2048 && rule->expert_count % 4 == 0 && rule->expert_count <= 256 && rule->top <= 16 && rule->group_count <= 16)
    return rule->expert_count <= 64    ? igl::launch_route_rows<4>(a, stream)
           : rule->expert_count <= 128 ? igl::launch_route_rows<8>(a, stream)
                                       : igl::launch_route_rows<16>(a, stream);
  const int per = (rule->expert_count + 63) / 64;
  return per <= 1   ? igl::launch_route<1>(a, stream)
         : per <= 2 ? igl::launch_route<2>(a, stream)
         : per <= 4 ? igl::launch_route<4>(a, stream)
         : per <= 8 ? igl::launch_route<8>(a, stream)
                    : igl::launch_route<16>(a, stream);
}
