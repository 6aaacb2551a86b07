// plan4.hip - the backend's igl_gemv.hip with its attention's plans laid open: every
// tile's blocks, segments and masks against counting.  TEST INFRASTRUCTURE ONLY.
#include "igl_gemv.hip"

#include <vector>

// Zero, or the number of the first thing found wrong, for one call of the
// attention over the ring.
extern "C" int plan4_check(int head, int kv, int span, int sinks, int share, int place, int window, int lanes) {
  igl_cache4 store = {};
  store.cache_span = span;
  store.sink_count = sinks;
  store.kv_count = kv;
  store.head_size = head;
  store.key_scale = store.value_scale = 1.0f;
  Attend4Args a = attend4_args(&store, share, nullptr, 0, place, window, lanes, 1.0f, nullptr);
  const Attend4Plan p = attend4_plan(a, head, kv);

  // ---- the cut
  if (a.rows != lanes * share || (long long)p.tiles * p.each < a.rows || (long long)(p.tiles - 1) * p.each >= a.rows) return 1;
  if (a.segments < 1 || a.segments > kAttend4Segments || a.per < 1) return 2;
  if (a.part_row0 < 0 || a.part_row0 >= a.rows || a.part_row0 % p.each != 0 || (p.step && a.part_row0 != 0)) return 3;
  if (a.segments > 1 && (long long)a.segments * kv * (a.rows - a.part_row0) * (head + 2) > (long long)IGL_ATTEND4_FLOATS)
    return 4;
  if (p.tiles > 65535 * 1024 || kv > 65535) return 5;
  for (int row = 0; row < a.rows; row += 1 + row / 7)
    if (attend4_lane(row, a) != row / share) return 6;

  // ---- what a slot holds once the last lane is laid
  std::vector<int> held(span, 0x7FFFFFFF);
  for (int q = 0; q < sinks; ++q) held[q] = q;  // no other; later than every lane where not yet laid
  for (long long q = a.newest; q >= sinks && q > (long long)a.newest - (span - sinks); --q) held[cache4_slot((int)q, sinks, span)] = (int)q;
  for (int slot = 0; slot < span + 200; ++slot)
    if (attend4_place(slot, a) != (slot < span ? held[slot] : 0x7FFFFFFF)) return 7;
  auto sees = [&](int at, int lane) {
    return at <= lane && (window == 0 || at > lane - window || at < sinks);
  };

  // ---- every tile: each visible slot in one of its blocks, once, and each block in one segment
  std::vector<int> taken;
  for (int tile = 0; tile < p.tiles; ++tile) {
    const int row0 = tile * p.each, row_last = (row0 + p.each < a.rows ? row0 + p.each : a.rows) - 1;
    const int low = place + row0 / share, high = place + row_last / share;
    const Blocks4 b = attend4_blocks(p.block, low, high, a);
    if (b.count < 1 || b.count > p.blocks) return 8;
    taken.assign((span + p.block - 1) / p.block, 0);
    const bool split = a.segments > 1 && (p.step || row0 >= a.part_row0);
    for (int seg = 0; seg < (split ? a.segments : 1); ++seg) {
      const int first = b.count < seg * a.per ? b.count : seg * a.per;
      const int next = b.count < first + a.per ? b.count : first + a.per;
      const int end = !split || seg == a.segments - 1 ? b.count : next;
      for (int i = first; i < end; ++i) {
        const int at = b.at(i);
        if (at < 0 || at >= (int)taken.size() || taken[at]++) return 9;
        const int slot0 = at * p.block, ahead = i < b.low ? b.low_ahead : b.mid_ahead;
        for (int half = 0; half < p.block; half += 32) {  // as whole blocks, and in parts of 32
          const int count = half ? 32 : p.block, from = half ? slot0 + half : slot0;
          const bool all = attend4_all(from, count, ahead, low, high, a);
          for (int slot = from; all && slot < from + count; ++slot)
            if (slot >= span || !sees(held[slot], low) || !sees(held[slot], high)) return 10;
        }
      }
    }
    for (int slot = 0; slot < span; ++slot)
      for (int lane = low; lane <= high; lane += high > low ? high - low : 1) {
        const bool seen = sees(held[slot], lane);
        if (seen != attend4_seen(slot, lane, a)) return 11;
        if (seen && !taken[slot / p.block]) return 12;
      }
  }
  return 0;
}

// The form a call takes: 0 tiles of 64 rows, 1 of sixteen, 2 of eight, 3 the same
// in deep blocks; plus 4 times its segments.
extern "C" int plan4_form(int head, int kv, int span, int sinks, int share, int place, int window, int lanes) {
  igl_cache4 store = {};
  store.cache_span = span;
  store.sink_count = sinks;
  store.kv_count = kv;
  store.head_size = head;
  store.key_scale = store.value_scale = 1.0f;
  Attend4Args a = attend4_args(&store, share, nullptr, 0, place, window, lanes, 1.0f, nullptr);
  const Attend4Plan p = attend4_plan(a, head, kv);
  return (p.deep ? 3 : p.pair ? 2 : p.step ? 1 : 0) + 4 * a.segments;
}
