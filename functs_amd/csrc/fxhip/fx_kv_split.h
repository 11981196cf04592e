// Which workgroup of an attention call takes which rows and cached tokens (plain C++: the tests check it on the CPU).
//
// An item is a tile of rows of one request and key head; its cached tokens are taken in steps of FX_KV_STEP.  The lengths
// are on the device, so every workgroup adds up all steps of the call and cuts them into chunks of about 1 / FX_KV_TARGET of them: a
// request of more steps than a chunk has its items shared by several workgroups.  An item of t steps, more than a
// chunk of c, gets ceil(t / c) <= 2 t / c parts, so there are fewer than FX_KV_TARGET shared items and at most
// 2 FX_KV_TARGET parts whatever the lengths: the sizes of the workspace.
// Measured with 128, 256 and 512: one request of 130 000 tokens 64, 55 and 57 us; 64 of up to 4 000 64, 63 and 72; prompts 390, 391 and
// 421; 24 requests of a few rows 19, 20 and 23.
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#define FX_KV_HD __host__ __device__ __forceinline__
#else
#define FX_KV_HD inline
#endif

#define FX_KV_STEP 64    // cached tokens of a step of a wave
#define FX_KV_TARGET 256 // parts that a call's work is cut into, about

struct FxKvRequest {
  int start, rows, len, tiles, steps;   // steps: of all its rows together
};
// a request's numbers as they are in memory (any values) to what may be used: rows inside `tokens`, tokens inside `room`
FX_KV_HD FxKvRequest fx_kv_request(int start, int end, int len, int tokens, int room, int group, int window, int tile_rows) {
  FxKvRequest r;
  const int s = start < 0 ? 0 : start > tokens ? tokens : start, e = end < 0 ? 0 : end > tokens ? tokens : end;
  r.start = s;
  r.rows = e > s ? e - s : 0;
  r.len = len < 0 ? 0 : len > room ? room : len;
  r.tiles = (int)(((int64_t)r.rows * group + tile_rows - 1) / tile_rows);
  const int64_t first = (int64_t)r.len - r.rows + 1 - window;
  const int low = window > 0 && first > 0 ? (int)(first < r.len ? first : r.len) : 0;
  r.steps = (r.len + FX_KV_STEP - 1) / FX_KV_STEP - low / FX_KV_STEP;
  return r;
}
// Steps of a request's tiles, of one head, for the sum of a call.  Offsets that fall (there are none in a call that is meant) let requests
// overlap, whose units may be more than 31 bits count: the work is endless then, so that nothing is cut and no part lies outside the workspace
#define FX_KV_ENDLESS (int64_t{1} << 60)
FX_KV_HD int64_t fx_kv_work(int start, int end, const FxKvRequest& r) { return start > end ? FX_KV_ENDLESS : (int64_t)r.tiles * r.steps; }
// steps of a chunk, of `work` steps in all: a multiple of `least`
FX_KV_HD int fx_kv_chunk(int64_t work, int least) {
  const int64_t steps = (work + FX_KV_TARGET - 1) / FX_KV_TARGET, chunk = (steps + least - 1) / least * least;
  return (int)(chunk < least ? least : chunk > (1 << 30) ? (1 << 30) : chunk);
}
FX_KV_HD int fx_kv_parts(int steps, int chunk) { return steps > chunk ? (steps + chunk - 1) / chunk : 1; }

// Unit `rest` of a request, of `splits` for each item: false where it has none of that number
FX_KV_HD bool fx_kv_item(const FxKvRequest& r, int heads, int splits, int rest, int* item, int* tile, int* head) {
  *item = rest / splits;
  *tile = *item / heads;
  *head = *item - *tile * heads;
  return rest >= 0 && *tile < r.tiles;
}

struct FxKvSpan {
  int low, high;            // tokens that some row of the tile sees: [low, high)
  int all_low, all_high;    // tokens that every row of it sees
  int from, to;             // steps of a part
};
// tile rows [r0, r0 + tile_rows) (row = token of the request * group + query head of the key head) and part `part` of `parts`
FX_KV_HD FxKvSpan fx_kv_span(const FxKvRequest& r, int group, int window, int r0, int tile_rows, int part, int parts) {
  FxKvSpan s;
  const int64_t n = (int64_t)r.rows * group, behind = (int64_t)r0 + tile_rows;
  const int last = (int)((behind < n ? behind : n) - 1);
  const int first_pos = r.len - r.rows + r0 / group, last_pos = r.len - r.rows + last / group;
  s.high = last_pos + 1 > 0 ? last_pos + 1 : 0;
  s.all_high = first_pos + 1 > 0 ? first_pos + 1 : 0;
  s.low = window > 0 && first_pos + 1 - window > 0 ? first_pos + 1 - window : 0;
  s.all_low = window > 0 && last_pos + 1 - window > 0 ? last_pos + 1 - window : 0;
  const int step0 = s.low / FX_KV_STEP, all = (s.high + FX_KV_STEP - 1) / FX_KV_STEP - step0, steps = all > 0 ? all : 0;
  s.from = step0 + (int)((int64_t)steps * part / parts);
  s.to = step0 + (int)((int64_t)steps * (part + 1) / parts);
  return s;
}
// the entry of a table that may be used: a page of the cache, or -1
FX_KV_HD int fx_kv_page(int entry, int pages) { return (unsigned)entry < (unsigned)pages ? entry : -1; }
