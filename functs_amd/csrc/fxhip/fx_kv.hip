// The paged 8-bit key / value cache: where tokens go (fx_kv_plan), how they get there (fx_kv_store) and what is
// there (fx_kv_read).  Attention over it is fx_kv_attn.h.  (The kernel of fx_kv_store: fx_kv_store.h.)
//
// A value is code * scale, the scale a power of two for each page and head: the least 2^e with
// amax <= top * 2^e (top: 448 for e4m3, 127 for int8), -100 <= e <= 119 (e4m3) or 121 (int8), which keeps
// top * 2^e finite.  Powers of two cost e4m3 no precision, make dividing and multiplying exact (so codes are
// exactly defined), and a page whose scale grows keeps its e4m3 codes but for underflow.
#include <algorithm>

#include "fx_kv_store.h"

namespace {
// ---- fx_kv_plan ----
// Bound: latency (a few bytes a request and twelve a token).  One launch, nothing crosses workgroups: each
// takes kPlanTokens tokens and adds up the lengths of all requests by itself (kPlanRequests a round).  The
// request of a token: the workgroup's requests leave their number at their first token, and a maximum over
// the tokens before spreads it.
// Measured: 17 requests of one token 5.4 us, 700 requests of 89 000 tokens 7.4, either below the host's work for a call.
constexpr int kPlanTokens = 1024, kPlanRequests = 1024, kPer = 4;
static_assert(kPlanTokens == kThreads * kPer && kPlanRequests == kThreads * kPer, "four of each a thread");

__device__ __forceinline__ int64_t shfl_up64(int64_t v, int d) { return (int64_t)__shfl_up((unsigned long long)v, (unsigned)d, 64); }

// Exclusive sum over the workgroup; *total: the whole sum.  scratch: kThreads / 64 words that nothing else uses meanwhile
__device__ __forceinline__ int64_t block_sum_before(int64_t v, int64_t* scratch, int64_t* total) {
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  int64_t s = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t o = shfl_up64(s, d);
    if (lane >= d) s += o;
  }
  if (lane == 63) scratch[wave] = s;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    if (w < wave) before += scratch[w];
    all += scratch[w];
  }
  __syncthreads();
  *total = all;
  return before + s - v;
}

__global__ __launch_bounds__(kThreads) void fx_kv_plan_kernel(const FxKvPlanArgs a) {
  __shared__ int64_t s_scan[kThreads / 64];
  __shared__ int s_max[kThreads / 64];
  __shared__ int s_req[kPlanTokens], s_start[kPlanTokens], s_end[kPlanTokens], s_past[kPlanTokens], s_off[kPlanTokens];
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int c0 = (int)blockIdx.x * kPlanTokens, c1 = min(a.tokens, c0 + kPlanTokens);   // (tokens < 2^30: no overflow)
  const int page = 1 << a.log_page;
  for (int i = tid; i < kPlanTokens; i += kThreads) s_req[i] = 0;
  const int64_t from = a.free_start ? min(max((int64_t)*a.free_start, (int64_t)0), (int64_t)a.n_free) : 0;
  const int64_t n_free = a.n_free - from, room = (int64_t)a.columns << a.log_page;
  int64_t rows = 0, pages = 0, taken = 0;
  __syncthreads();
  for (int b0 = 0; b0 < a.requests; b0 += kPlanRequests) {
    if (blockIdx.x != 0 && rows >= c1) break;   // (the sums are the workgroup's: all threads leave)
    int past[kPer], added[kPer];
    int64_t sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int b = b0 + tid * kPer + i;
      past[i] = b < a.requests ? a.past[b] : 0;
      added[i] = b < a.requests ? a.added[b] : 0;
      sum += max(added[i], 0);
    }
    int64_t all;
    int64_t start = rows + block_sum_before(sum, s_scan, &all);
    rows += all;
    int64_t at[kPer], want[kPer], need = 0;
    bool fits[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      at[i] = start;
      start += max(added[i], 0);
      const int64_t now = (int64_t)past[i] + added[i];
      fits[i] = past[i] >= 0 && added[i] >= 0 && now <= room && start <= a.tokens;
      want[i] = fits[i] ? ((now + page - 1) >> a.log_page) - (((int64_t)past[i] + page - 1) >> a.log_page) : 0;
      need += want[i];
    }
    int64_t off = pages + block_sum_before(need, s_scan, &all);
    pages += all;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int b = b0 + tid * kPer + i;
      if (b >= a.requests) break;
      const bool granted = fits[i] && (want[i] == 0 || off + want[i] <= n_free);
      if (granted) taken += want[i];
      if (blockIdx.x == 0) {
        a.starts[b] = (int)min(at[i], (int64_t)a.tokens);
        a.lens[b] = granted ? past[i] + added[i] : 0;
      }
      const int64_t end = min(at[i] + max(added[i], 0), (int64_t)a.tokens);
      if (at[i] < c1 && end > c0 && end > at[i]) {
        const int p = (int)(max(at[i], (int64_t)c0) - c0);
        s_req[p] = granted ? b + 1 : -1 - b;
        s_start[p] = (int)at[i];
        s_end[p] = (int)end;
        s_past[p] = past[i];
        s_off[p] = (int)(from + off);   // (granted: below n_free)
      }
      off += want[i];
    }
  }
  if (blockIdx.x == 0) {
    int64_t all;
    block_sum_before(taken, s_scan, &all);
    if (tid == 0) {
      a.starts[a.requests] = (int)min(rows, (int64_t)a.tokens);
      *a.taken = (int)all;
    }
  }
  __syncthreads();
  // the last mark at or before each token
  int mark[kPer], last = -1;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (s_req[tid * kPer + i] != 0) last = tid * kPer + i;
    mark[i] = last;
  }
  int upto = last;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(upto, (unsigned)d, 64);
    if (lane >= d) upto = max(upto, o);
  }
  if (lane == 63) s_max[wave] = upto;
  int before = __shfl_up(upto, 1u, 64);
  if (lane == 0) before = -1;
  __syncthreads();
  for (int w = 0; w < wave; ++w) before = max(before, s_max[w]);
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int t = c0 + tid * kPer + i, m = max(mark[i], before);
    if (t >= c1) break;
    int64_t slot = -1;
    int pos = -1;
    if (m >= 0 && s_req[m] > 0 && t < s_end[m]) {
      const int b = s_req[m] - 1, past = s_past[m];
      pos = past + (t - s_start[m]);
      const int col = pos >> a.log_page, had = (int)(((int64_t)past + page - 1) >> a.log_page);
      int p;
      if (col < had) {
        p = a.table[(int64_t)b * a.table_stride + col];
      } else {
        p = a.free_pages[s_off[m] + (col - had)];
        if ((pos & (page - 1)) == 0) a.table[(int64_t)b * a.table_stride + col] = p;   // (a new page has a first token)
      }
      if (p >= 0) slot = ((int64_t)p << a.log_page) + (pos & (page - 1));
    }
    a.slots[t] = slot;
    a.positions[t] = pos;
  }
}

// ---- fx_kv_read ----
// Bound: HBM (1 byte read and 2 or 4 written for each number).  A wave takes the keys or the values of one head for 4 to 16
// entries of `slots`.  Keys: 8 numbers of a token a lane, four loads under way.  Values: 4 columns of 8 of the 16 tokens of a
// group, so that a lane writes 4 numbers side by side; the group is the wave's in whose entries its first token is.
// Measured: 25 500 tokens, 8 heads of 128, e4m3 to bf16, caches and results that are in no cache of the chip: 45 us, 3.5 TB/s (a large
// copy: 5.4), keys alone 18 and values 25.  32 entries a wave 45 to 47 us, 8 entries 54; groups cut where the entries end 46.
template <int HELD, class T>
__global__ __launch_bounds__(kThreads) void fx_kv_read_kernel(const FxKvCache c, const FxKvRows r, int per_wave, int n_chunks, int vec) {
  const int lane = (int)threadIdx.x & 63;
  const int64_t w = (int64_t)blockIdx.x * kStoreWaves + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const unsigned chunk_head = (unsigned)(w >> 1);
  const int half = (int)(w & 1), chunk = (int)(chunk_head / (unsigned)c.heads), head = (int)(chunk_head - (unsigned)chunk * (unsigned)c.heads);
  if (chunk >= n_chunks) return;
  const int D = c.depth, page = 1 << c.log_page;
  const int64_t n_slots = (int64_t)c.pages << c.log_page, in_page = (int64_t)head * page * D;
  const int t0 = chunk * per_wave, n = min(r.tokens - t0, per_wave);
  int64_t mine = r.slots[t0 + min(lane, n - 1)];   // lane i: of token t0 + i
  if (mine < 0 || mine >= n_slots) mine = -1;
  if (half == 0) {
    const int width = D >> 3, abreast = 64 / width, sub = lane / width, at = lane - sub * width;
    T* dst = (T*)r.k + (int64_t)t0 * r.k_token + (int64_t)head * r.k_head + at * 8;
    constexpr int kBatch = 4;
    for (int j0 = 0; j0 < n; j0 += abreast * kBatch) {
      uint2 u[kBatch];
      float scale[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int64_t s = __shfl(mine, min(j0 + i * abreast + sub, n - 1), 64);
        const int64_t p = s < 0 ? 0 : s >> c.log_page;
        scale[i] = c.k_scale[p * c.ks_stride + head];
        u[i] = *(const uint2*)(c.k + p * c.k_stride + in_page + (s < 0 ? 0 : s & (page - 1)) * D + at * 8);
        if (s < 0) u[i] = make_uint2(0, 0), scale[i] = 0.0f;
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int j = j0 + i * abreast + sub;
        if (sub >= abreast || j >= n) continue;
        float x[8];
        decode4<HELD>(x, u[i].x);
        decode4<HELD>(x + 4, u[i].y);
        union { T e[8]; uint4 u[sizeof(T) / 2]; } y;
#pragma unroll
        for (int e = 0; e < 8; ++e) y.e[e] = (T)(x[e] * scale[i]);
        T* to = dst + (int64_t)j * r.k_token;
        if (vec) {
#pragma unroll
          for (int q = 0; q < (int)sizeof(T) / 2; ++q) ((uint4*)to)[q] = y.u[q];
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) to[e] = y.e[e];
        }
      }
    }
    return;
  }
  // The wave's are the neighbours of one group of 16, their slots rising by one, that begin in its chunk; lane i has token t0 - 1 + i
  T* dst = (T*)r.v + (int64_t)t0 * r.v_token + (int64_t)head * r.v_head;
  const int token = t0 - 1 + lane;
  mine = r.slots[min(max(token, 0), r.tokens - 1)];
  if (token < 0 || token >= r.tokens || mine < 0 || mine >= n_slots) mine = -1;
  const int64_t prior = (int64_t)__shfl_up((unsigned long long)mine, 1u, 64);
  const unsigned long long follows = __ballot(lane > 0 && mine >= 0 && prior + 1 == mine && (mine & 15) != 0);
  for (unsigned long long begins = ~follows & ((2ull << n) - 2); begins != 0; begins &= begins - 1) {
    const int at = __builtin_ctzll(begins), j = at - 1;
    const int64_t slot = lane_of(mine, at);
    const int o = (int)(slot & 15);
    const int m = slot < 0 ? 1 : __builtin_ctzll(~(follows >> at >> 1)) + 1;
    const int64_t p = slot < 0 ? 0 : slot >> c.log_page;
    const float scale = slot < 0 ? 0.0f : c.v_scale[p * c.vs_stride + head];
    const uint8_t* codes = c.v + p * c.v_stride + in_page + (slot < 0 ? 0 : (slot & (page - 1)) >> 4) * 16 * D;
    for (int unit = lane; unit < D >> 1; unit += 64) {
      const int upper = unit >= D >> 2 ? 1 : 0, quad = unit - upper * (D >> 2);   // eights of tokens, four columns
      float x[4][8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint2 u = *(const uint2*)(codes + (quad * 4 + i) * 16 + upper * 8);
        if (slot < 0) u = make_uint2(0, 0);
        decode4<HELD>(x[i], u.x);
        decode4<HELD>(x[i] + 4, u.y);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int k = upper * 8 + e - o;   // of the neighbours
        if (k < 0 || k >= m) continue;
        T* to = dst + (int64_t)(j + k) * r.v_token + quad * 4;
        const float y[4] = {x[0][e] * scale, x[1][e] * scale, x[2][e] * scale, x[3][e] * scale};
        if (vec) {
          union { T e[4]; uint2 u[sizeof(T) / 2]; } z;
#pragma unroll
          for (int i = 0; i < 4; ++i) z.e[i] = (T)y[i];
          if constexpr (sizeof(T) == 2) *(uint2*)to = z.u[0];
          else *(uint4*)to = make_uint4(z.u[0].x, z.u[0].y, z.u[1].x, z.u[1].y);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) to[i] = (T)y[i];
        }
      }
    }
  }
}

}  // namespace

hipError_t fx_launch_kv_plan(const FxKvPlanArgs& a, hipStream_t stream) {
  const unsigned grid = (unsigned)((a.tokens + kPlanTokens - 1) / kPlanTokens);
  FxKvPlanArgs args = a;
  void* kargs[1] = {(void*)&args};
  return hipLaunchKernel((const void*)fx_kv_plan_kernel, dim3(grid ? grid : 1), dim3(kThreads), kargs, 0, stream);
}

hipError_t fx_launch_kv_store(const FxKvCache& c, const FxKvRows& r, int held, hipStream_t stream) {
  static const void* const kernels[2][3] = {
      {(const void*)fx_kv_store_kernel<0, float>, (const void*)fx_kv_store_kernel<0, _Float16>, (const void*)fx_kv_store_kernel<0, __bf16>},
      {(const void*)fx_kv_store_kernel<1, float>, (const void*)fx_kv_store_kernel<1, _Float16>, (const void*)fx_kv_store_kernel<1, __bf16>}};
  StoreShape shape = store_shape(c, r);
  FxKvCache cache = c;
  FxKvRows rows = r;
  void* kargs[4] = {(void*)&cache, (void*)&rows, (void*)&shape.per, (void*)&shape.vec};
  return hipLaunchKernel(kernels[held][r.dtype == FX_DT_F32 ? 0 : r.dtype == FX_DT_F16 ? 1 : 2], dim3((unsigned)shape.blocks), dim3(kThreads), kargs, 0, stream);
}

hipError_t fx_launch_kv_read(const FxKvCache& c, const FxKvRows& r, int held, hipStream_t stream) {
  static const void* const kernels[2][3] = {
      {(const void*)fx_kv_read_kernel<0, float>, (const void*)fx_kv_read_kernel<0, _Float16>, (const void*)fx_kv_read_kernel<0, __bf16>},
      {(const void*)fx_kv_read_kernel<1, float>, (const void*)fx_kv_read_kernel<1, _Float16>, (const void*)fx_kv_read_kernel<1, __bf16>}};
  const size_t size = r.dtype == FX_DT_F32 ? 4 : 2;
  // (one token a wave took 17.1 us where four take 13.7: a step of 96 requests stored and 816 tokens read)
  int per = std::max(tokens_a_wave(c, r, 16), 4), chunks = (r.tokens + per - 1) / per;
  int vec = aligned16(r.k, r.k_token, r.k_head, size) && aligned16(r.v, r.v_token, r.v_head, size);
  FxKvCache cache = c;
  FxKvRows rows = r;
  void* kargs[5] = {(void*)&cache, (void*)&rows, (void*)&per, (void*)&chunks, (void*)&vec};
  const int64_t waves = (int64_t)chunks * c.heads * 2;
  return hipLaunchKernel(kernels[held][r.dtype == FX_DT_F32 ? 0 : r.dtype == FX_DT_F16 ? 1 : 2],
                         dim3((unsigned)((waves + kStoreWaves - 1) / kStoreWaves)), dim3(kThreads), kargs, 0, stream);
}
