// Pages of the paged cache behind a beam search's selection: arguments of their kernels (fx_kv_fork.hip).
#pragma once
#include "fx_kv.h"

// What fx_kv_fork_plan says of a row, as an old one and as a new one
struct FxKvForkRow {
  int32_t from;    // the old row of its group that the new one continues (-1: none)
  int32_t last;    // the page in which the new row's tokens end, where they do not fill it
  int32_t tokens;  // of the new row
  int32_t held;    // tokens of the old one
  int32_t alive;   // the old row is continued
  int32_t reused;  // the old row's last page, which nobody continues, is another's now
  int32_t unused[2];
};
struct FxKvForkArgs {
  const int32_t *parents, *lens, *free_pages, *free_start;
  int32_t *table, *out_lens, *copies, *taken, *freed, *n_freed;
  int64_t table_stride;
  FxKvForkRow* rows;   // [groups * beams]
  int32_t* counts;     // [groups * blocks]: pages that each block of columns frees
  int32_t* lists;      // [groups * blocks][beams * FX_KV_FORK_COLUMNS]
  int32_t groups, beams, columns, n_free, log_page, blocks;
};
#define FX_KV_FORK_COLUMNS 256   // of a workgroup of fx_kv_fork_tables
hipError_t fx_launch_kv_fork(const FxKvForkArgs& a, hipStream_t stream, int* launched);

#define FX_KV_COPY_LAYERS 32     // of a launch
struct FxKvCopyArgs {
  struct { uint8_t *k, *v; float *ks, *vs; } layer[FX_KV_COPY_LAYERS];
  FxKvCache c;                   // sizes and strides, which all layers share
  const int32_t* copies;         // [rows][3]: page, to page, tokens
  int32_t rows, layers, heads_a_unit, units_a_page;
};
hipError_t fx_launch_kv_copy(const FxKvCopyArgs& a, hipStream_t stream);
