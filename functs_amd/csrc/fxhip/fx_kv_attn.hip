// Attention over the paged 8-bit cache: launches.
#include "fx_kv_attn.h"

namespace fxkv {
// The sums of unit_at for more requests than a wave adds up: one workgroup
__global__ __launch_bounds__(1024) void fx_kv_offsets(const FxKvAttnArgs a, int tile_rows, int least) {
  constexpr int W = 16;
  __shared__ int64_t s_work[W];
  __shared__ int s_units[W], s_cuts[W];
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  int64_t work = 0;
  for (int b = (int)threadIdx.x; b < a.requests; b += 1024) {
    const FxKvRequest r = request_of(a, a.starts[b], a.starts[b + 1], a.lens[b], tile_rows);
    work = min(work + fx_kv_work(a.starts[b], a.starts[b + 1], r), FX_KV_ENDLESS);
  }
  work = wave_total(work);
  if (lane == 0) s_work[wave] = work;
  __syncthreads();
  work = 0;
  bool endless = false;
  for (int w = 0; w < W; ++w) {
    endless |= s_work[w] >= FX_KV_ENDLESS;
    work += s_work[w];
  }
  const int chunk = fx_kv_chunk(all_steps(a, endless ? FX_KV_ENDLESS : work), least);
  int32_t* units_to = a.offsets + 2;
  int units = 0, cuts = 0;   // of the rounds before
  for (int b0 = 0; b0 < a.requests; b0 += 1024) {
    const int b = b0 + (int)threadIdx.x;
    int mine = 0, cut = 0;
    if (b < a.requests) {
      const FxKvRequest r = request_of(a, a.starts[b], a.starts[b + 1], a.lens[b], tile_rows);
      const int splits = fx_kv_parts(r.steps, chunk), items = r.tiles * a.c.heads;
      mine = items * splits;
      cut = splits > 1 ? (items << 16) + mine : 0;
    }
    const int u = sum_upto(mine), c = sum_upto(cut);
    __syncthreads();
    if (lane == 63) {
      s_units[wave] = u;
      s_cuts[wave] = c;
    }
    __syncthreads();
    int before_u = units + u - mine, before_c = cuts + c - cut;
    for (int w = 0; w < W; ++w) {
      if (w < wave) {
        before_u += s_units[w];
        before_c += s_cuts[w];
      }
      units += s_units[w];
      cuts += s_cuts[w];
    }
    if (b < a.requests) {
      units_to[b] = before_u;
      units_to[a.requests + 1 + b] = before_c;
    }
  }
  if (threadIdx.x == 0) {
    units_to[a.requests] = units;
    a.offsets[0] = chunk;
    a.offsets[1] = (int)((unsigned)cuts >> 16);
  }
}
}  // namespace fxkv

namespace {
template <class... A>
hipError_t launch(int* launched, const void* kernel, int64_t grid, int threads, hipStream_t stream, A... args) {
  void* kargs[sizeof...(A)] = {(void*)&args...};
  const hipError_t e = hipLaunchKernel(kernel, dim3((unsigned)grid), dim3((unsigned)threads), kargs, 0, stream);
  *launched += e == hipSuccess;
  return e;
}
hipError_t offsets(int* launched, const FxKvAttnArgs& a, int tile_rows, int least, hipStream_t stream) {
  if (a.requests <= fxkv::kScanned) return hipSuccess;
  return launch(launched, (const void*)fxkv::fx_kv_offsets, 1, 1024, stream, a, tile_rows, least);
}
hipError_t join(int* launched, const FxKvAttnArgs& a, const FxKvLaunch& l, hipStream_t stream) {
  const int type = l.type;
  const void* kernel = type == fxkv::kBf16 ? (const void*)fxkv::fx_kv_join<__bf16>
                       : type == fxkv::kF16 ? (const void*)fxkv::fx_kv_join<_Float16>
                                            : (const void*)fxkv::fx_kv_join<float>;
  return launch(launched, kernel, 2048, 256, stream, a, l.tiles_parts, l.rows_parts);
}
}  // namespace

hipError_t fx_launch_kv_attention(const FxKvAttnArgs& a, const FxKvLaunch& l, hipStream_t stream, int* launched) {
  const bool wide = (1 << a.c.log_page) >= FX_KV_STEP;
  const fxkv::Kernels k = l.held == 0 ? fx_kv_kernels_e4m3(l.type, a.c.depth, wide) : fx_kv_kernels_int8(l.type, a.c.depth, wide);
  hipError_t e = hipSuccess;
  FxKvAttnArgs args = a;
  if (l.tiles_grid > 0) {
    args.rows_above = l.rows_grid > 0 ? FX_KV_FEW : 0;
    args.rows_upto = int64_t{1} << 31;
    args.parts = l.tiles_parts;
    if ((e = offsets(launched, args, l.tiles_parts.tile_rows, fxkv::kTileLeast, stream)) != hipSuccess) return e;
    if ((e = launch(launched, k.tiles, l.tiles_grid, 2 * l.tiles_parts.tile_rows, stream, args)) != hipSuccess) return e;
    args.fill = 0;
  }
  if (l.rows_grid > 0) {
    args.rows_above = 0;
    args.rows_upto = l.tiles_grid > 0 ? FX_KV_FEW : int64_t{1} << 31;
    args.parts = l.rows_parts;
    if ((e = offsets(launched, args, FX_KV_ROWS, fxkv::kRowLeast, stream)) != hipSuccess) return e;
    if ((e = launch(launched, k.rows, l.rows_grid, 256, stream, args)) != hipSuccess) return e;
  }
  return l.shared ? join(launched, args, l, stream) : e;
}
