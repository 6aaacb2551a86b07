/* hostmx_stub.c - the stand-in HIP runtime with the launchers of microscaled rows
 * and of experts wrapped: each buffer a launch touches, at the extent its
 * arguments imply, has to lie inside one recorded allocation.  TEST
 * INFRASTRUCTURE ONLY. */
#include "audit_stub.c"

static void check_mx4(const char *w, const char *what, const igl_mx4 *s, int first, int count) {
  check_range(w, what, s->code + (size_t)first * s->code_stride,
              (size_t)(count - 1) * s->code_stride + (size_t)s->col_count / 2);
  check_range(w, what, s->scale + (size_t)first * s->scale_stride,
              (size_t)(count - 1) * s->scale_stride + (size_t)s->col_count / 32);
}

static void check_lanes(const char *w, const char *what, const void *rows, int bf16, int stride, int lanes, int width) {
  check_range(w, what, rows, rows_bytes(lanes, stride, width, bf16 ? 2 : 4));
}

hipError_t R(igl_launch_mx4_lay)(const igl_mx4 *, int, int, const void *, int, int, hipStream_t);
hipError_t W(igl_launch_mx4_lay)(const igl_mx4 *store, int row_first, int rows, const void *src, int bf16,
                                 int src_stride, hipStream_t stream) {
  const char *w = "igl_launch_mx4_lay";
  check_mx4(w, "store", store, row_first, rows);
  check_lanes(w, "src", src, bf16, src_stride, rows, store->col_count);
  return R(igl_launch_mx4_lay)(store, row_first, rows, src, bf16, src_stride, stream);
}

hipError_t R(igl_launch_mx4_read)(const igl_mx4 *, int, int, void *, int, int, hipStream_t);
hipError_t W(igl_launch_mx4_read)(const igl_mx4 *store, int row_first, int rows, void *dst, int bf16, int dst_stride,
                                  hipStream_t stream) {
  const char *w = "igl_launch_mx4_read";
  check_mx4(w, "store", store, row_first, rows);
  check_lanes(w, "dst", dst, bf16, dst_stride, rows, store->col_count);
  return R(igl_launch_mx4_read)(store, row_first, rows, dst, bf16, dst_stride, stream);
}

hipError_t R(igl_launch_mx4_mat_mat)(const igl_mx4 *, const void *, int, int, int, void *, int, int, void *, hipStream_t);
hipError_t W(igl_launch_mx4_mat_mat)(const igl_mx4 *sheet, const void *act, int act_bf16, int act_stride, int lanes,
                                     void *out, int out_bf16, int out_stride, void *work, hipStream_t stream) {
  const char *w = "igl_launch_mx4_mat_mat";
  const size_t bytes = igl_mx4_work_bytes(sheet->row_count, sheet->col_count, lanes, act_bf16 ? 3 : 5);
  check_mx4(w, "sheet", sheet, 0, sheet->row_count);
  check_lanes(w, "act", act, act_bf16, act_stride, lanes, sheet->col_count);
  check_lanes(w, "out", out, out_bf16, out_stride, lanes, sheet->row_count);
  if (bytes) check_range(w, "work", work, bytes);
  return R(igl_launch_mx4_mat_mat)(sheet, act, act_bf16, act_stride, lanes, out, out_bf16, out_stride, work, stream);
}

hipError_t R(igl_launch_mx4_mat_mx4)(const igl_mx4 *, const igl_mx4 *, int, int, void *, int, int, void *, hipStream_t);
hipError_t W(igl_launch_mx4_mat_mx4)(const igl_mx4 *sheet, const igl_mx4 *act, int lane_first, int lanes, void *out,
                                     int out_bf16, int out_stride, void *work, hipStream_t stream) {
  const char *w = "igl_launch_mx4_mat_mx4";
  const size_t bytes = igl_mx4_work_bytes(sheet->row_count, sheet->col_count, lanes, 0);
  check_mx4(w, "sheet", sheet, 0, sheet->row_count);
  check_mx4(w, "act", act, lane_first, lanes);
  check_lanes(w, "out", out, out_bf16, out_stride, lanes, sheet->row_count);
  if (bytes) check_range(w, "work", work, bytes);
  return R(igl_launch_mx4_mat_mx4)(sheet, act, lane_first, lanes, out, out_bf16, out_stride, work, stream);
}

hipError_t R(igl_launch_route)(const igl_route *, const float *, int, int, const float *, const float *, int32_t *,
                               float *, hipStream_t);
hipError_t W(igl_launch_route)(const igl_route *rule, const float *logits, int logit_stride, int lanes,
                               const float *bias, const float *gain, int32_t *pick, float *weight,
                               hipStream_t stream) {
  const char *w = "igl_launch_route";
  const size_t chosen = (size_t)lanes * rule->top * 4;
  check_lanes(w, "logits", logits, 0, logit_stride, lanes, rule->expert_count);
  if (bias) check_range(w, "bias", bias, (size_t)rule->expert_count * 4);
  if (gain) check_range(w, "gain", gain, (size_t)rule->expert_count * 4);
  check_range(w, "pick", pick, chosen);
  check_range(w, "weight", weight, chosen);
  return R(igl_launch_route)(rule, logits, logit_stride, lanes, bias, gain, pick, weight, stream);
}

hipError_t R(igl_launch_experts)(const igl_experts *, const void *, int, int, int, const int32_t *, const float *, int,
                                 void *, int, int, void *, hipStream_t);
hipError_t W(igl_launch_experts)(const igl_experts *x, const void *act, int act_bf16, int act_stride, int lanes,
                                 const int32_t *pick, const float *weight, int top, void *out, int out_bf16,
                                 int out_stride, void *work, hipStream_t stream) {
  const char *w = "igl_launch_experts";
  const size_t chosen = (size_t)lanes * top * 4;
  check_mx4(w, "gate_up", &x->gate_up, 0, x->gate_up.row_count);
  check_mx4(w, "down", &x->down, 0, x->down.row_count);
  check_lanes(w, "act", act, act_bf16, act_stride, lanes, x->hidden);
  check_lanes(w, "out", out, out_bf16, out_stride, lanes, x->hidden);
  check_range(w, "pick", pick, chosen);
  check_range(w, "weight", weight, chosen);
  check_range(w, "work", work, igl_experts_work_bytes(x, lanes, top, act_bf16));
  return R(igl_launch_experts)(x, act, act_bf16, act_stride, lanes, pick, weight, top, out, out_bf16, out_stride, work,
                               stream);
}
