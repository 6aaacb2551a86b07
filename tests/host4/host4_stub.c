/* host4_stub.c - the stand-in HIP runtime with the 4-bit ring's launchers
 * wrapped: each buffer a launch touches, at the extent its arguments imply, has
 * to lie inside one recorded allocation.  TEST INFRASTRUCTURE ONLY. */
#include "audit_stub.c"

static void check_ring(const char *w, const igl_cache4 *s) {
  const size_t codes = (size_t)s->cache_span * s->kv_count * s->head_size / 2;
  const size_t gains = ((size_t)s->cache_span + 63) / 64 * 64 * s->kv_count * s->head_size / 32;
  check_range(w, "key_code", s->key_code, codes);
  check_range(w, "value_code", s->value_code, codes);
  check_range(w, "key_gain", s->key_gain, gains);
  check_range(w, "value_gain", s->value_gain, gains);
}

hipError_t R(igl_launch_cache4_lay)(const igl_cache4 *, const float *, const float *, int, int, int, hipStream_t);
hipError_t W(igl_launch_cache4_lay)(const igl_cache4 *s, const float *key, const float *value, int row_stride,
                                    int place_first, int lanes, hipStream_t stream) {
  const char *w = "igl_launch_cache4_lay";
  const size_t rows = rows_bytes(lanes, row_stride, (size_t)s->kv_count * s->head_size, sizeof(float));
  check_ring(w, s);
  check_range(w, "key", key, rows);
  check_range(w, "value", value, rows);
  return R(igl_launch_cache4_lay)(s, key, value, row_stride, place_first, lanes, stream);
}

hipError_t R(igl_launch_cache4_read)(const igl_cache4 *, int, int, float *, float *, int, hipStream_t);
hipError_t W(igl_launch_cache4_read)(const igl_cache4 *s, int place_first, int lanes, float *key, float *value,
                                     int row_stride, hipStream_t stream) {
  const char *w = "igl_launch_cache4_read";
  const size_t rows = rows_bytes(lanes, row_stride, (size_t)s->kv_count * s->head_size, sizeof(float));
  check_ring(w, s);
  if (key) check_range(w, "key", key, rows);
  if (value) check_range(w, "value", value, rows);
  return R(igl_launch_cache4_read)(s, place_first, lanes, key, value, row_stride, stream);
}

hipError_t R(igl_launch_attend4)(const igl_cache4 *, int, const float *, int, int, int, int, float, float *, float *,
                                 hipStream_t);
hipError_t W(igl_launch_attend4)(const igl_cache4 *s, int share, const float *query, int lane_stride, int place_first,
                                 int window, int lanes, float score_scale, float *blend, float *work,
                                 hipStream_t stream) {
  const char *w = "igl_launch_attend4";
  const size_t rows = rows_bytes(lanes, lane_stride, (size_t)s->kv_count * s->head_size * share, sizeof(float));
  check_ring(w, s);
  check_range(w, "query", query, rows);
  check_range(w, "blend", blend, rows);
  check_range(w, "work", work, IGL_ATTEND4_FLOATS * sizeof(float));
  return R(igl_launch_attend4)(s, share, query, lane_stride, place_first, window, lanes, score_scale, blend, work,
                               stream);
}
