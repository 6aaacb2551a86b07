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
  int lanes;
  int window;
  float key_factor;      // key scale, score scale and log2 e
  float value_scale;
};

// The blocks of kCache4Block slots that hold what lanes at positions first ..
// last see: blocks 0 .. low - 1, then mid .. mid + count - low - 1.  The visible
// slots are the sinks' and the ring's from the oldest position to the newest,
// cut in two where the ring wraps; the piece from slot sinks on joins the sinks.
struct Blocks4 {
  int low, mid, count;
  __host__ __device__ int at(int i) const { return i < low ? i : mid + i - low; }
};

__host__ __device__ __forceinline__ Blocks4 attend4_blocks(int span, int sinks, int window, int first, int last) {
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
  b.low = (low_slots + kCache4Block - 1) / kCache4Block;
  b.mid = mid_first / kCache4Block;
  if (b.mid < b.low) b.mid = b.low;
  const int end = mid_last < 0 ? 0 : mid_last / kCache4Block + 1;
  b.count = b.low + (end > b.mid ? end - b.mid : 0);
  return b;
}

// The position whose row a slot holds once `newest` is laid; INT_MAX: none.
__device__ __forceinline__ int attend4_place(int slot, int sinks, int span, int newest) {
  if (slot >= span) return 0x7FFFFFFF;
  if (slot < sinks) return slot;
  if (newest < sinks) return 0x7FFFFFFF;
  const int ring = span - sinks;
  int back = (newest - sinks) % ring - (slot - sinks);
  if (back < 0) back += ring;
  return newest - back >= sinks ? newest - back : 0x7FFFFFFF;
}

// A workgroup a lane and query head: thread t scores slot t of the block, then
// blends dims t, t + 64, ...
template <int HEAD, int FMT>
__global__ __launch_bounds__(64) void attend4_row_kernel(Attend4Args a) {
  __shared__ float qs[HEAD];
  __shared__ float ps[64];
  const int t = threadIdx.x;
  const int lane = blockIdx.x / a.share, h = blockIdx.x % a.share, kv = blockIdx.y;
  const int pos = a.place + lane, newest = a.place + a.lanes - 1;
  const size_t row_at = (size_t)lane * a.lane_stride + ((size_t)kv * a.share + h) * HEAD;
  for (int d = t; d < HEAD; d += 64) qs[d] = a.query[row_at + d];
  __syncthreads();
  const Blocks4 b = attend4_blocks(a.span, a.sinks, a.window, pos, pos);
  float base = -INFINITY, total = 0.0f, out[HEAD / 64];
#pragma unroll
  for (int j = 0; j < HEAD / 64; ++j) out[j] = 0.0f;
  for (int i = 0; i < b.count; ++i) {
    const int slot0 = b.at(i) * kCache4Block;
    const int slot = slot0 + t;
    const int place = attend4_place(slot, a.sinks, a.span, newest);
    const bool seen = place <= pos && (a.window == 0 || place > pos - a.window || place < a.sinks);
    const size_t row = (size_t)min(slot, a.span - 1);
    const uint8_t *codes = a.key_code + (row * a.kv_width + (size_t)kv * HEAD) / 2;
    float s = 0.0f;
    for (int g = 0; g < HEAD / kCache4Group; ++g) {
      float part = 0.0f;
      for (int d = 0; d < kCache4Group; d += 2) {
        const uint32_t c = codes[(g * kCache4Group + d) / 2];
        part += cache4_level<FMT>(c & 15u) * qs[g * kCache4Group + d];
        part += cache4_level<FMT>(c >> 4) * qs[g * kCache4Group + d + 1];
      }
      s += part * cache4_gain(a.key_gain[(size_t)(kv * (HEAD / kCache4Group) + g) * a.room + row]);
    }
    s = seen ? s * a.key_factor : -INFINITY;
    float peak = s;
    for (int off = 32; off > 0; off >>= 1) peak = fmaxf(peak, __shfl_xor(peak, off));
    const float next = fmaxf(base, peak);
    const float keep = base != -INFINITY ? __builtin_amdgcn_exp2f(base - next) : 0.0f;
    const float p = seen ? __builtin_amdgcn_exp2f(s - next) : 0.0f;
    float sum = p;
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
    total = total * keep + sum;
    base = next;
    ps[t] = p;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < HEAD / 64; ++j) {
      const int d = t + 64 * j;
      float o = 0.0f;
      for (int e = 0; e < kCache4Block; ++e) {
        const size_t r = (size_t)min(slot0 + e, a.span - 1);
        const uint32_t c = (a.value_code[(r * a.kv_width + (size_t)kv * HEAD + d) / 2] >> (4 * (d & 1))) & 15u;
        const float gain = cache4_gain(a.value_gain[(size_t)(kv * (HEAD / kCache4Group) + d / kCache4Group) * a.room + r]);
        o += ps[e] * (cache4_level<FMT>(c) * gain);
      }
      out[j] = out[j] * keep + o;
    }
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < HEAD / 64; ++j) a.out[row_at + t + 64 * j] = out[j] * a.value_scale * (1.0f / total);
}

}  // namespace igl

using namespace igl;

template <int HEAD>
static hipError_t attend4_launch(const Attend4Args &a, int format, int kv_count, hipStream_t stream) {
  const long long rows = (long long)a.lanes * a.share;
  if (rows > 0x7FFFFFFF) return hipErrorInvalidValue;
  const dim3 grid((unsigned)rows, kv_count);
  if (format == IGL_CACHE4_INT4)
    hipLaunchKernelGGL((attend4_row_kernel<HEAD, IGL_CACHE4_INT4>), grid, dim3(64), 0, stream, a);
  else
    hipLaunchKernelGGL((attend4_row_kernel<HEAD, IGL_CACHE4_E2M1>), grid, dim3(64), 0, stream, a);
  return hipGetLastError();
}

extern "C" hipError_t igl_launch_attend4(const igl_cache4 *store, int group_share, const float *query, int lane_stride,
                                         int place_first, int window, int lanes, float score_scale, float *blend_out,
                                         float *work, hipStream_t stream) {
  Attend4Args a = {};
  (void)work;
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
  a.lanes = lanes;
  a.window = window;
  a.key_factor = (float)((double)store->key_scale * score_scale * 1.4426950408889634);  // log2 e
  a.value_scale = store->value_scale;
  switch (store->head_size) {
    case 64: return attend4_launch<64>(a, store->format, store->kv_count, stream);
    case 128: return attend4_launch<128>(a, store->format, store->kv_count, stream);
    case 256: return attend4_launch<256>(a, store->format, store->kv_count, stream);
    case 512: return attend4_launch<512>(a, store->format, store->kv_count, stream);
    default: return hipErrorInvalidValue;
  }
}
