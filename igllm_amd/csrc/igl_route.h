// igl_route.h - the choice of experts, gfx950: scores of a lane's logits, a bias for
// balance, groups of experts, the best of the kept groups, their weights.
//
//     s_e = softmax(x)_e or 1 / (1 + e^-x_e),   c_e = s_e + bias_e
//     a group's score is the sum of its largest one or two c; the best groups stay
//     the chosen are the largest c among them, the lowest index first where equal
//     w = s of the chosen (over their sum), times the rule's gain and the expert's
// A choice next to another's must fall as the reals' does, so scores are formed and
// compared in double; without a bias and groups s rises with x, and x decides.
#pragma once

#include "igl_device.h"
#include "igl_launch.h"

namespace igl {

constexpr int kRouteWaves = 4;  // lanes a workgroup, a wave each

struct RouteArgs {
  igl_route rule;
  const float *logits;
  long long logit_stride;
  int lanes;
  const float *bias, *gain;
  int32_t *pick;
  float *weight;
};

__device__ __forceinline__ double shfl_f64(double v, int from) { return __shfl(v, from); }

// The larger choice, the lower index where equal.
__device__ __forceinline__ bool route_before(double a, int ia, double b, int ib) {
  return a > b || (a == b && ia < ib);
}

// A wave a lane of the batch; wave lane l holds experts l, l + 64, .. (PER of them).
// What may not be chosen has choice -infinity.
template <int PER>
__global__ __launch_bounds__(64 * kRouteWaves) void route_kernel(RouteArgs a) {
  __shared__ double choices[kRouteWaves][64 * PER];
  __shared__ double scores[kRouteWaves][64];  // of groups
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long m = (long long)blockIdx.x * kRouteWaves + wave;
  const bool here = m < a.lanes;
  const int E = a.rule.expert_count;
  const float *x = a.logits + (here ? m : 0) * a.logit_stride;
  const double none = -__builtin_inf();
  float v[PER];
  float top = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane + 64 * i;
    v[i] = e < E ? x[e] : -__builtin_inff();
    if (!(v[i] >= -3.402823466e38f)) v[i] = -__builtin_inff();  // a NaN is never chosen
    if (v[i] > 3.402823466e38f) v[i] = 3.402823466e38f;
    top = fmaxf(top, v[i]);
  }
  double s[PER], c[PER];
  if (a.rule.score == IGL_ROUTE_SOFTMAX) {
    for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      s[i] = v[i] == -__builtin_inff() ? 0.0 : exp((double)v[i] - (double)top);
      sum += s[i];
    }
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
#pragma unroll
    for (int i = 0; i < PER; ++i) s[i] = sum > 0.0 ? s[i] / sum : 0.0;
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) s[i] = v[i] == -__builtin_inff() ? 0.0 : 1.0 / (1.0 + exp(-(double)v[i]));
  }
  const bool plain = !a.bias && a.rule.group_count == 1;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane + 64 * i;
    c[i] = v[i] == -__builtin_inff() ? none : plain ? (double)v[i] : s[i] + (a.bias && e < E ? (double)a.bias[e] : 0.0);
    if (!(c[i] > none)) c[i] = none;  // a bias that is a NaN
    choices[wave][e] = c[i];
  }
  __syncthreads();
  if (a.rule.group_count > 1) {
    const int each = E / a.rule.group_count;
    double score = none;
    if (lane < a.rule.group_count) {
      double first = none, second = none;
      for (int i = 0; i < each; ++i) {
        const double t = choices[wave][lane * each + i];
        if (t > first) {
          second = first;
          first = t;
        } else if (t > second) {
          second = t;
        }
      }
      score = a.rule.group_best == 2 && second > none ? first + second : first;
    }
    scores[wave][lane] = score;
    __syncthreads();
    // a group stays if fewer than group_top come before it
    int ahead = 0;
    for (int g = 0; g < a.rule.group_count; ++g) ahead += route_before(scores[wave][g], g, score, lane);
    scores[wave][lane] = ahead < a.rule.group_top && score > none ? 1.0 : 0.0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = lane + 64 * i;
      if (e < E && scores[wave][e / each] == 0.0) c[i] = none;
    }
  }
  // the best, one at a time; wave lane j keeps the j-th's
  int mine = -1;
  double share = 0.0, total = 0.0;
  for (int j = 0; j < a.rule.top; ++j) {
    double best = none, score = 0.0;
    int at = 0x7FFFFFFF;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (c[i] > best) best = c[i], at = lane + 64 * i, score = s[i];
    for (int d = 32; d; d >>= 1) {
      const double other = __shfl_xor(best, d), other_score = __shfl_xor(score, d);
      const int other_at = __shfl_xor(at, d);
      if (route_before(other, other_at, best, at)) best = other, at = other_at, score = other_score;
    }
    if (!(best > none)) break;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (lane + 64 * i == at) c[i] = none;
    total += score;
    if (lane == j) mine = at, share = score;
  }
  if (!here || lane >= a.rule.top) return;
  if (a.rule.renorm) share = total > 0.0 ? share / total : 0.0;
  share *= (double)a.rule.gain_scale;
  if (a.gain && mine >= 0) share *= (double)a.gain[mine];
  a.pick[m * a.rule.top + lane] = mine;
  a.weight[m * a.rule.top + lane] = mine >= 0 ? (float)share : 0.0f;
}

}  // namespace igl

extern "C" hipError_t igl_launch_route(const igl_route *rule, const float *logits, int logit_stride, int lanes,
                                       const float *bias, const float *gain, int32_t *pick, float *weight,
                                       hipStream_t stream) {
  const igl::RouteArgs a = {*rule, logits, logit_stride, lanes, bias, gain, pick, weight};
  const dim3 grid((unsigned)((lanes + igl::kRouteWaves - 1) / igl::kRouteWaves)), block(64 * igl::kRouteWaves);
  const int per = (rule->expert_count + 63) / 64;
  if (per <= 1)
    hipLaunchKernelGGL((igl::route_kernel<1>), grid, block, 0, stream, a);
  else if (per <= 2)
    hipLaunchKernelGGL((igl::route_kernel<2>), grid, block, 0, stream, a);
  else if (per <= 4)
    hipLaunchKernelGGL((igl::route_kernel<4>), grid, block, 0, stream, a);
  else if (per <= 8)
    hipLaunchKernelGGL((igl::route_kernel<8>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((igl::route_kernel<16>), grid, block, 0, stream, a);
  return hipGetLastError();
}
