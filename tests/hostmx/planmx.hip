// planmx.hip - the backend's igl_gemm_level.hip with the plans of the microscaled
// products laid open.  TEST INFRASTRUCTURE ONLY.
#include "igl_gemm_level.hip"

#include <vector>

// The form of a product (0 few, 1 head, 2 small, 3 large, 4 whole) and its slices.
extern "C" int planmx_form(int rows, int cols, int lanes, int terms) {
  return mx4_form(rows, cols / kMx4Group, lanes, terms);
}

extern "C" int planmx_slices(int rows, int cols, int lanes, int tile_lanes, int tile_rows) {
  return mx4_slices(rows, cols / kMx4Group, lanes, tile_lanes, tile_rows);
}

extern "C" int planmx_steps(int cols) { return mx4_steps(cols / kMx4Group); }

// Zero, or the first thing wrong: pieces of the experts' room that do not follow one
// another, or are smaller than what the forms put there.
extern "C" int planmx_room(int experts, int hidden, int inner, int lanes, int top, int bf16) {
  igl_experts x = {};
  x.expert_count = experts;
  x.hidden = hidden;
  x.inner = inner;
  const ExpertRoom r = expert_room(&x, lanes, top, bf16);
  const size_t slots = (size_t)lanes * top, step = bf16 ? 320 : 512;
  const size_t gate_blocks = (size_t)experts * ((inner + 31) / 32), down_blocks = (size_t)experts * ((hidden + 63) / 64);
  const size_t h_steps = mx4_steps(inner / 32), x_steps = mx4_steps(hidden / 32);
  if (r.lane_of != 0 || r.place_of - r.lane_of < slots * 4 || r.tiles - r.place_of < slots * 4) return 1;
  for (int tile = 16; tile <= 128; tile *= 2)
    if (r.x - r.tiles < (slots / tile + experts) * sizeof(Mx4Tile)) return 2;
  if (r.gate_up - r.x < lanes * x_steps * step) return 3;
  if (r.down - r.gate_up < gate_blocks * x_steps * 256) return 4;  // four tiles a block, half of them gate rows
  if (r.h - r.down < down_blocks * h_steps * 256) return 5;
  if (r.rows - r.h < slots * h_steps * step || r.rows - r.h < slots * inner * sizeof(float)) return 6;
  if (r.end - r.rows < slots * hidden * sizeof(float)) return 7;
  if ((r.lane_of | r.place_of | r.tiles | r.x | r.gate_up | r.down | r.h | r.rows) % 256) return 8;
  return 0;
}

// The places of a call's tiles of experts, or zero where slots are taken one by one.
extern "C" int planmx_experts(int experts, int hidden, int inner, int lanes, int top, int bf16) {
  igl_experts x = {};
  x.expert_count = experts;
  x.hidden = hidden;
  x.inner = inner;
  return expert_steps(&x, lanes * top) ? 0 : expert_tile(&x, lanes * top, bf16);
}

// Whether a product is a token's step.
extern "C" int planmx_single(int rows, int cols, int lanes, int kind) {
  return mx4_single(rows, cols / kMx4Group, lanes, mx4_form(rows, cols / kMx4Group, lanes, kind), kind);
}

// Zero, or a slot whose lane is not slot / top.
extern "C" int planmx_lanes(int top) {
  for (int slot = 0; slot < 1 << 20; ++slot)
    if (place_lane(slot, place_inverse(top)) != slot / top) return slot;
  return 0;
}

// Zero, or the first thing wrong with a step's pieces of `lanes` lanes of terms: bytes of
// two groups at one place, or a step's not all taken.
template <int T>
static int pieces_wrong(int lanes) {
  std::vector<int> taken((size_t)lanes * TermForm<T>::kStep / 16, 0);
  for (int lane = 0; lane < lanes; ++lane)
    for (int c = 0; c < TermForm<T>::kChunks; ++c)
      for (int part = 0; part < 4; ++part) {
        const size_t at = term_piece<T>(lane, lanes, c, part);
        if (at % 16 || at / 16 >= taken.size() || taken[at / 16]++) return 1 + c;
      }
  return 0;
}

extern "C" int planmx_pieces(int terms, int lanes) { return terms == 3 ? pieces_wrong<3>(lanes) : pieces_wrong<5>(lanes); }

// Zero, or which of the eight lanes' runs that LDS serves together meet a bank twice:
// sixteen rows of 64 bytes (a step's codes) or of 128 (two pieces of terms).
extern "C" int planmx_banks(int width, int keyed) {
  static const int together[2][16] = {{0, 1, 2, 3, 12, 13, 14, 15, 20, 21, 22, 23, 24, 25, 26, 27},
                                      {4, 5, 6, 7, 8, 9, 10, 11, 16, 17, 18, 19, 28, 29, 30, 31}};
  for (int half = 0; half < width / 64; ++half)
    for (int run = 0; run < 4; ++run) {
      unsigned slots = 0;
      for (int i = 0; i < 16; ++i) {
        const int lane = together[run & 1][i] + 32 * (run >> 1), row = lane & 15, part = lane >> 4;
        const int key = !keyed ? 0 : width == 64 ? tile_key(row) : pair_key(row);
        slots |= 1u << ((row * width / 16 + ((4 * half + part) ^ key)) & 15);
      }
      if (slots != 0xFFFFu) return 1 + run;
    }
  return 0;
}

// Zero, or the step at which tiles of an expert's places fail: counts that do not add up, or
// two experts' tiles at one number (what expert_place writes, counted on the host).
extern "C" int planmx_tiles(const int *count, int experts, int tile) {
  int slots = 0;
  for (int e = 0; e < experts; ++e) slots += count[e];
  const int total = expert_tiles(slots, experts, tile);
  int before = 0, next = 0;
  for (int e = 0; e < experts; ++e) {
    const int first = before / tile + e;
    const int end = e + 1 < experts ? (before + count[e]) / tile + e + 1 : total;
    if (first != next || first + (count[e] + tile - 1) / tile > end || end > total) return e + 1;
    before += count[e];
    next = end;
  }
  return next == total ? 0 : -1;
}
