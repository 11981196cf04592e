// TEST INFRASTRUCTURE ONLY - never linked into or loaded by the product.
//
// fx_kv_split.h over a whole call: which rows and steps every part takes, and how many parts are shared.
#include <map>
#include <set>
#include <tuple>

#include "../../functs_amd/csrc/fxhip/fx_kv_split.h"

// 0: every (head, tile, step that some row sees) is taken exactly once, spans are those of the definition and the shared parts fit the
// workspace; else the number of the check that failed.  out[0..2]: units, shared parts, shared items.
extern "C" int fx_kv_split_check(int requests, const int* starts, const int* lens, int tokens, int room, int group, int window, int heads, int tile_rows,
                                 int least, long long* out) {
  int64_t work = 0, units = 0, parts = 0, items = 0;
  for (int b = 0; b < requests; ++b) {
    const FxKvRequest r = fx_kv_request(starts[b], starts[b + 1], lens[b], tokens, room, group, window, tile_rows);
    if (r.start < 0 || r.rows < 0 || r.start + r.rows > tokens || r.len < 0 || r.len > room || r.steps < 0) return 1;
    work += (int64_t)r.tiles * r.steps;
  }
  const int chunk = fx_kv_chunk(work * heads, least);
  for (int b = 0; b < requests; ++b) {
    const FxKvRequest r = fx_kv_request(starts[b], starts[b + 1], lens[b], tokens, room, group, window, tile_rows);
    const int splits = fx_kv_parts(r.steps, chunk);
    const int64_t here = (int64_t)r.tiles * heads;
    units += here * splits;
    if (splits > 1) {
      parts += here * splits;
      items += here;
    }
    for (int tile = 0; tile < r.tiles; ++tile) {
      int low = 1 << 30, high = 0, all_low = 0, all_high = 1 << 30;
      for (int row = tile * tile_rows; row < (tile + 1) * tile_rows && row < r.rows * group; ++row) {
        const int pos = r.len - r.rows + row / group, hi = pos + 1 > 0 ? pos + 1 : 0, lo = window > 0 && hi - window > 0 ? hi - window : 0;
        if (hi > high) high = hi;
        if (lo < low) low = lo;
        if (hi < all_high) all_high = hi;
        if (lo > all_low) all_low = lo;
      }
      int at = -1, end = -1;
      for (int p = 0; p < splits; ++p) {
        const FxKvSpan s = fx_kv_span(r, group, window, tile * tile_rows, tile_rows, p, splits);
        if (s.high != high || s.low != low || s.all_low != all_low || s.all_high != all_high) return 2;
        if (s.high > r.len || s.to < s.from || (s.to > s.from && (int64_t)(s.to - 1) * FX_KV_STEP >= s.high)) return 3;   // (no step behind the last token)
        if (p > 0 && s.from != end) return 4;
        if (p == 0) at = s.from;
        end = s.to;
      }
      if (high > low && (at * FX_KV_STEP > low || end * FX_KV_STEP < high)) return 5;
      if (high <= low && end != at && high > 0 && low < high) return 6;
    }
  }
  out[0] = units;
  out[1] = parts;
  out[2] = items;
  if (parts > 2 * FX_KV_TARGET || items > FX_KV_TARGET) return 7;
  return 0;
}
extern "C" int fx_kv_page_of(int entry, int pages) { return fx_kv_page(entry, pages); }
