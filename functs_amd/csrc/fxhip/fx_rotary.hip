// Rotary positions, forward and backward (fx_rotary_device.h has the mathematics).
//
// Bound: HBM (each number is read and written once) from a few thousand rows on, latency below.  A workgroup takes some tokens with all their heads, so that an
// angle is formed once, in LDS, while the first of its four units a thread, two at a time, are under way; what is left of the address arithmetic is multiplications.
// 3 x 1 999 tokens of 40 heads of 128 columns, bf16, either way: 26 us, 4.7 TB/s (a large copy: 5.4); 30 001 of 24 heads of 64, fp16, half of their columns turning in
// neighbouring pairs: 35 us, 5.3 TB/s; 61 single tokens: 3.5 us.
#include <algorithm>

#include "fx_rotary_device.h"

namespace {
template <class T, int PV, bool INTER>
__global__ __launch_bounds__(256) void fx_rotary_kernel(const FxRotary a) {
  __shared__ Turn s_turn[FX_ROTARY_ANGLES];
  rotary_rows<T, PV, INTER>(a, (int)(blockIdx.x / (unsigned)a.slices), (int)(blockIdx.x % (unsigned)a.slices), s_turn);
}

// n / d as the upper word of n * magic, for n up to `most` (0: not exact there)
uint32_t magic_of(uint32_t d, uint64_t most) { return d > 1 && most * d < uint64_t{1} << 32 ? (uint32_t)((uint64_t{1} << 32) / d) + 1 : 0; }
}  // namespace

// Units of 16 bytes twice where a head has as many pairs, single pairs (and single columns that do not turn) otherwise: 30 000 tokens of 24 heads of 128 columns, fp16: 75 us with 8
// pairs, 155 to 160 with 4; of 32 columns 17 and 39 (a copy's rate: 68 and 17)
static int rotary_pairs_a_unit(const FxRotary& a) {
  const int pv = a.dtype == FX_DT_F32 ? 4 : 8;
  return a.turns.pairs >= pv ? pv : 1;
}
void fx_rotary_shape(FxRotary& a) {
  const int pv = rotary_pairs_a_unit(a), rest = a.depth - 2 * a.turns.pairs;
  a.turning = (a.turns.pairs + pv - 1) / pv;
  a.units = a.turning + (rest >= 2 * pv ? (rest + 2 * pv - 1) / (2 * pv) : rest > 0 ? 1 : 0);
  const int64_t row = (int64_t)a.units * a.heads, total = (int64_t)a.batch * a.tokens;
  // two times two units a thread (two at once: 86 registers and 23 us become 68 and 21 for 3 x 1 999 tokens of 40 heads of 128, bf16, the same ones in each call, which
  // the caches keep, and 26 for others in each; once, or four times: 22 of the same), and not fewer than two workgroups a CU where there are as many tokens
  int64_t per = std::min<int64_t>(std::max<int64_t>(1024 / row, 1), FX_ROTARY_ANGLES / a.turns.pairs);
  per = std::max<int64_t>(std::min(per, total / 512), 1);
  a.per = (int32_t)per;
  a.blocks = (int32_t)((total + per - 1) / per);
  const int64_t rounds = (per * row + 255) / 256;
  a.slices = (int32_t)std::max<int64_t>(std::min<int64_t>(rounds, 512 / a.blocks), (rounds + 31) / 32);
  a.magic_token = magic_of((uint32_t)row, (uint64_t)(per * row));
  a.magic_head = magic_of((uint32_t)a.units, (uint64_t)row);
  a.magic_pair = magic_of((uint32_t)a.turns.pairs, (uint64_t)per * a.turns.pairs);
}

hipError_t fx_launch_rotary(const FxRotary& a, hipStream_t stream) {
#define FX_ROW(T, PV) {(const void*)fx_rotary_kernel<T, 1, false>, (const void*)fx_rotary_kernel<T, 1, true>, (const void*)fx_rotary_kernel<T, PV, false>, (const void*)fx_rotary_kernel<T, PV, true>}
  static const void* const kernels[3][4] = {FX_ROW(float, 4), FX_ROW(_Float16, 8), FX_ROW(__bf16, 8)};
#undef FX_ROW
  FxRotary args = a;
  void* kargs[1] = {(void*)&args};
  const int type = a.dtype == FX_DT_F32 ? 0 : a.dtype == FX_DT_F16 ? 1 : 2;
  return hipLaunchKernel(kernels[type][(rotary_pairs_a_unit(a) > 1 ? 2 : 0) + (a.turns.interleaved ? 1 : 0)], dim3((unsigned)a.blocks * (unsigned)a.slices), dim3(256), kargs, 0, stream);
}
