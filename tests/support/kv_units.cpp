// TEST INFRASTRUCTURE ONLY - never linked into or loaded by the product.
//
// How a unit of an attention call is found from sums of 32 bits, as the kernels do it for many requests, where offsets may fall.
#include <algorithm>
#include <vector>

#include "../../functs_amd/csrc/fxhip/fx_kv_split.h"

// 0: every unit that is looked at (the first ones, the last ones and `step` apart between them) is one of its request's, and its parts lie in the
// workspace; else the number of the check that failed.  Sums wrap as the kernels' do.
extern "C" int fx_kv_units_check(int requests, const int* starts, const int* lens, int tokens, int room, int group, int heads, int tile_rows, int least,
                                 int step, int* shared_items) {
  std::vector<FxKvRequest> all;
  int64_t work = 0;
  for (int b = 0; b < requests; ++b) {
    all.push_back(fx_kv_request(starts[b], starts[b + 1], lens[b], tokens, room, group, 0, tile_rows));
    work = std::min(work + fx_kv_work(starts[b], starts[b + 1], all[b]), FX_KV_ENDLESS);
  }
  const int chunk = fx_kv_chunk(work >= FX_KV_ENDLESS ? work : work * heads, least);
  std::vector<int> units{0}, cuts{0};
  for (const FxKvRequest& r : all) {
    const int splits = fx_kv_parts(r.steps, chunk);
    const uint32_t items = (uint32_t)r.tiles * heads, mine = items * splits;
    units.push_back((int)((uint32_t)units.back() + mine));
    cuts.push_back((int)((uint32_t)cuts.back() + (splits > 1 ? (items << 16) + mine : 0)));
  }
  *shared_items = (int)((uint32_t)cuts.back() >> 16);
  if (*shared_items > FX_KV_TARGET) return 1;
  for (int64_t v = 0; v < units.back(); v += v < 4096 || v > units.back() - 4096 ? 1 : step) {
    const int u = (int)v;
    int lo = 0;
    for (int b = 0; b < requests; ++b)
      if (units[b] <= u) lo = b;
    const int splits = fx_kv_parts(all[lo].steps, chunk);
    int item, tile, head;
    if (!fx_kv_item(all[lo], heads, splits, u - units[lo], &item, &tile, &head)) continue;
    const int split = u - units[lo] - item * splits;
    if (tile < 0 || tile >= all[lo].tiles || head < 0 || head >= heads || split < 0 || split >= splits) return 2;
    if (splits > 1 && ((cuts[lo] & 0xffff) + (item + 1) * splits > 2 * FX_KV_TARGET || (int)((uint32_t)cuts[lo] >> 16) + item >= *shared_items)) return 3;
  }
  return 0;
}
