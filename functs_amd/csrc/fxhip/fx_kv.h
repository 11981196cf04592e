// The paged 8-bit key / value cache: arguments of its kernels (fx_kv.hip, fx_kv_attn.h).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../../include/fxhip.h"
#include "fx_kv_split.h"
#include "fx_rotary.h"

// A cache as the kernels see it.  Keys [pages][heads][page][depth]; values [pages][heads][page / 16][depth][16]: the
// second product of attention contracts over tokens, and a lane's operand is 8 or 16 of them side by side.
struct FxKvCache {
  uint8_t *k, *v;
  float *k_scale, *v_scale;               // [pages][heads], rows scale_stride apart
  uint32_t k_stride, v_stride;            // bytes from page to page
  uint32_t ks_stride, vs_stride;          // floats from page to page
  int32_t pages, heads, depth, log_page;  // (page: 16 to 256 tokens, a power of two)
};

struct FxKvPlanArgs {
  const int32_t *past, *added, *free_pages, *free_start;
  int32_t* table;
  int64_t* slots;
  int32_t *positions, *starts, *lens, *taken;
  int64_t table_stride;
  int32_t requests, columns, n_free, log_page, tokens;
};

// rows of keys and values outside the cache: [tokens][heads][depth], a depth contiguous
struct FxKvRows {
  void *k, *v;
  int64_t k_token, k_head, v_token, v_head;  // elements
  const int64_t* slots;
  int32_t tokens, dtype;
};

#define FX_KV_STORE_MOST 63   // tokens that a workgroup of fx_kv_store takes at most: a lane each, and one for the token before them
hipError_t fx_launch_kv_plan(const FxKvPlanArgs& a, hipStream_t stream);
hipError_t fx_launch_kv_store(const FxKvCache& c, const FxKvRows& r, int held, hipStream_t stream);
hipError_t fx_launch_kv_append(const FxKvCache& c, const FxKvRows& r, const FxRotary& q, int held, hipStream_t stream);
hipError_t fx_launch_kv_read(const FxKvCache& c, const FxKvRows& r, int held, hipStream_t stream);

#define FX_KV_ROWS 16   // rows (tokens of a request times query heads of a key head) of a tile of fx_kv_rows
// rows of a tile of fx_kv_tiles: 32 for each of 8 waves; of 4 where a wave needs more than half of a SIMD's registers
FX_KV_HD int fx_kv_tile_rows(int depth) { return depth <= 128 ? 256 : 128; }
// fx_kv_tiles takes the requests of more than FX_KV_FEW rows of calls of 16-bit queries with at least FX_KV_MANY rows of all heads (192 for
// each CU: with fewer its large tiles leave CUs idle); all others are fx_kv_rows'.  Measured, fx_kv_rows against fx_kv_tiles (us, e4m3, bf16):
//   calls     1 request, 32 heads of 128: 32 000 rows 84 / 104, 64 000 rows 188 / 105; 4 requests, 192 000 rows 880 / 414; 12 heads of 64,
//             96 000 rows 95 / 85, 192 000 rows 204 / 156; depth 256: 16 000 rows 76 / 86, 64 000 rows 447 / 368; depth 80: 32 000 rows 67 / 111
//   requests  of 100 rows, 51 200 in all 46 / 71; of 128 rows, 65 536 in all 97 / 86, of 400 rows, 102 400 in all 116 / 84
//   fp32      (three numbers for each query and weight) 64 000 rows 238 / 267, 192 000 rows 1 000 / 1 335, depth 256 517 / 1 002: fx_kv_rows always
// Not measured on both sides: fp16, int8, pages of 16 and 32, depths below 64; they go by the same rule.
#define FX_KV_FEW 128
#define FX_KV_MANY 49152
struct FxKvItem {   // rows whose cached tokens several workgroups shared
  int32_t request, head, tile, first, parts;
};
struct FxKvParts {
  float* acc;        // [parts][tile_rows][depth]
  float* ml;         // [parts][tile_rows][2]: maximum, sum
  FxKvItem* items;
  int32_t* n_items;
  int32_t tile_rows;
};
struct FxKvAttnArgs {
  FxKvCache c;
  const void* q;
  void* out;
  float* lse;
  const int32_t *table, *lens, *starts;
  int64_t q_token, q_head, out_token, table_stride;   // elements (out and lse: contiguous rows of all heads)
  int32_t tokens, requests, columns, q_heads, group, window;
  float scale;                                        // times log2(e)
  FxKvParts parts;
  int32_t* offsets;                                   // of more than 64 requests: see fx_kv_offsets
  int32_t fill;                                       // rows of no request are cleared
  int32_t q_vec;                                      // rows of queries are 16-byte aligned
  int64_t rows_above, rows_upto;                      // requests that this kernel takes: by rows of all query heads of a key head
};
struct FxKvLaunch {
  int held, type;                   // FX_KV_E4M3, FX_KV_INT8; 0 bf16, 1 fp16, 2 fp32
  bool shared;                      // items may be shared by workgroups
  int64_t rows_grid, tiles_grid;    // workgroups of fx_kv_rows and fx_kv_tiles (0: not needed)
  FxKvParts rows_parts, tiles_parts;
};
hipError_t fx_launch_kv_attention(const FxKvAttnArgs& a, const FxKvLaunch& l, hipStream_t stream, int* launched);   // launched: how many kernels
