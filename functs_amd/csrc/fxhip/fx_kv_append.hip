// fx_kv_append: fx_kv_store with keys that turn by their positions on the way into the cache, and the queries of the same tokens turned beside
// it, in one launch.
//
// A key is turned in fp32 and rounded once, to its code.  The first workgroups of the launch store (fx_kv_store.h), the others turn queries
// (fx_rotary_device.h): the long runs begin first.  (Queries first: 65 us instead of 59; in turn: 57, but a step of single tokens 8.2 instead of 7.5.)
// Bound: HBM; single tokens: latency.  Four waves a SIMD without registers in memory, which the numbers' whole words and frequencies in LDS allow: three took 69 us.
// 10 565 tokens of 5 prompts, 32 query heads on 8 of 128 columns, fp16 to int8: 58 us, 4.1 TB/s; 64 single tokens, bf16 to e4m3: 7.4.
#include "fx_kv_store.h"

namespace {
template <int HELD, class T, bool INTER>
__global__ __launch_bounds__(kThreads, 4) void fx_kv_append_kernel(const FxKvCache c, const FxKvRows r, int per, int vec, unsigned stores, const FxRotary q) {
  __shared__ unsigned s_tops[2][kStoreWaves];
  __shared__ Turn s_turn[FX_ROTARY_ANGLES];
  constexpr int PV = sizeof(T) == 4 ? 4 : 8;
  if (blockIdx.x < stores) {
    static_assert(sizeof s_turn >= kTurnPairs * sizeof(double), "either part's numbers");
    store_chunk<HELD, T, true, INTER>(c, r, per, vec, blockIdx.x, &q.turns, (double*)s_turn, s_tops);
    return;
  }
  const unsigned share = blockIdx.x - stores;
  const int block = (int)(share / (unsigned)q.slices), slice = (int)(share % (unsigned)q.slices);
  if (q.turns.pairs >= PV) rotary_rows<T, PV, INTER>(q, block, slice, s_turn);
  else rotary_rows<T, 1, INTER>(q, block, slice, s_turn);
}
}  // namespace

hipError_t fx_launch_kv_append(const FxKvCache& c, const FxKvRows& r, const FxRotary& q, int held, hipStream_t stream) {
#define FX_ROW(H, T) {(const void*)fx_kv_append_kernel<H, T, false>, (const void*)fx_kv_append_kernel<H, T, true>}
  static const void* const kernels[2][3][2] = {{FX_ROW(0, float), FX_ROW(0, _Float16), FX_ROW(0, __bf16)}, {FX_ROW(1, float), FX_ROW(1, _Float16), FX_ROW(1, __bf16)}};
#undef FX_ROW
  StoreShape shape = store_shape(c, r);
  FxKvCache cache = c;
  FxKvRows rows = r;
  FxRotary queries = q;
  unsigned stores = (unsigned)shape.blocks;
  void* kargs[6] = {(void*)&cache, (void*)&rows, (void*)&shape.per, (void*)&shape.vec, (void*)&stores, (void*)&queries};
  const int type = r.dtype == FX_DT_F32 ? 0 : r.dtype == FX_DT_F16 ? 1 : 2;
  return hipLaunchKernel(kernels[held][type][q.turns.interleaved ? 1 : 0], dim3(stores + (unsigned)q.blocks * (unsigned)q.slices), dim3(kThreads), kargs, 0, stream);
}
