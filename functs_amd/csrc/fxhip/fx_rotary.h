// Rotary positions: arguments of their kernels (fx_rotary.hip, fx_kv_append.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../../include/fxhip.h"

// By how much the pairs of a token turn
struct FxTurns {
  const void* positions;     // int32, or int64 (wide)
  const void* frequencies;   // [pairs] radians a token: double, or float (narrow)
  int32_t pairs, wide, narrow, interleaved, back;
  float magnitude;
};
// Rows outside the cache: [batch][tokens][heads][depth], a depth contiguous
struct FxRotary {
  FxTurns turns;
  const void* x;
  void* y;
  int64_t x_batch, x_token, x_head, y_batch, y_token, y_head, position_batch;  // elements
  int32_t batch, tokens, heads, depth, dtype;
  // how the work is dealt out (fx_rotary_shape): `per` tokens a block of which `slices` workgroups share the units, `units` of them a head and
  // `turning` of those turn; magic: 2^32 / (units of all heads), 2^32 / units, 2^32 / pairs, rounded up (0: plain division)
  int32_t per, slices, blocks, units, turning;
  uint32_t magic_token, magic_head, magic_pair;
};
#define FX_ROTARY_ANGLES 2048   // that a workgroup keeps: at most so many pairs, and tokens times pairs
void fx_rotary_shape(FxRotary& a);
hipError_t fx_launch_rotary(const FxRotary& a, hipStream_t stream);
