// Attention over e4m3 caches, and what both kinds share.
#include "fx_kv_attn.h"

const void* fx_kv_rows_kernel_e4m3(int type, int depth) { return fxkv::rows_kernel<0>(type, depth); }

hipError_t fx_launch_kv_attention(const FxKvAttnArgs& a, int held, int type, int64_t grid, int64_t join_grid, hipStream_t stream) {
  FxKvAttnArgs args = a;
  void* kargs[1] = {(void*)&args};
  const void* kernel = held == 0 ? fx_kv_rows_kernel_e4m3(type, a.c.depth) : fx_kv_rows_kernel_int8(type, a.c.depth);
  hipError_t e = hipLaunchKernel(kernel, dim3((unsigned)grid), dim3(256), kargs, 0, stream);
  if (e != hipSuccess || join_grid == 0) return e;
  int rows = FX_KV_ROWS;
  void* join_args[2] = {(void*)&args, (void*)&rows};
  const void* join = type == fxkv::kBf16 ? (const void*)fxkv::fx_kv_join<__bf16>
                     : type == fxkv::kF16 ? (const void*)fxkv::fx_kv_join<_Float16>
                                          : (const void*)fxkv::fx_kv_join<float>;
  return hipLaunchKernel(join, dim3((unsigned)join_grid), dim3(256), join_args, 0, stream);
}
