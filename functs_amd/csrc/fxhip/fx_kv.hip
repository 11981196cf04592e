// The paged 8-bit key / value cache: where tokens go (fx_kv_plan), how they get there (fx_kv_store) and what is
// there (fx_kv_read).  Attention over it is fx_kv_attn.h.
//
// A value is code * scale, the scale a power of two for each page and head: the least 2^e with
// amax <= top * 2^e (top: 448 for e4m3, 127 for int8), -100 <= e <= 119 (e4m3) or 121 (int8), which keeps
// top * 2^e finite.  Powers of two cost e4m3 no precision, make dividing and multiplying exact (so codes are
// exactly defined), and a page whose scale grows keeps its e4m3 codes but for underflow.
#include "fx_kv.h"
#include "fx_kv_device.h"

namespace {
constexpr int kThreads = 256;

// ---- fx_kv_plan ----
// Bound: latency (a few bytes a request and twelve a token).  One launch, nothing crosses workgroups: each
// takes kPlanTokens tokens and adds up the lengths of all requests by itself (kPlanRequests a round).  The
// request of a token: the workgroup's requests leave their number at their first token, and a maximum over
// the tokens before spreads it.
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

// ---- fx_kv_store ----
// Bound: HBM (2 or 4 bytes read and 1 written for each number); single tokens: latency.
// A run is the neighbours in `slots` that lie in one page; a wave takes the keys or the values of one head of a
// run, so a page's scale and codes have one writer and nothing is locked.  Two passes over the run's numbers,
// the second from the caches: their largest magnitude gives the scale, then codes.  The old tokens of a page whose scale
// grows are rounded again to the new one.
constexpr int kStoreWaves = kThreads / 64;

template <class T>
__device__ __forceinline__ void load8(float (&x)[8], const T* p, bool vec) {
  if (vec) {
    if constexpr (sizeof(T) == 2) {
      union { uint4 u; T e[8]; } w;
      w.u = *(const uint4*)p;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = (float)w.e[i];
    } else {
      union { uint4 u[2]; T e[8]; } w;
      w.u[0] = *(const uint4*)p;
      w.u[1] = *(const uint4*)(p + 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = (float)w.e[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)p[i];
  }
}
__device__ __forceinline__ float finite_abs(float x) {
  const float m = __builtin_fabsf(x);
  return m <= 3.402823466e38f ? m : 0.0f;   // (infinities become the largest code, NaN a code of its own or 0: neither sets the scale)
}
__device__ __forceinline__ float wave_max64(float v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v = fmaxf(v, __shfl_xor(v, d, 64));
  return v;
}

// 16 codes under a scale `ratio` times as large, those before `n` of them
template <int HELD>
__device__ __forceinline__ uint4 again16(uint4 w, float ratio, int n) {
  unsigned* u = (unsigned*)&w;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x[4];
    decode4<HELD>(x, u[i]);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] *= ratio;
    const unsigned fresh = encode4<HELD>(x);
    const int left = n - 4 * i;
    const unsigned keep = left >= 4 ? 0u : left <= 0 ? ~0u : ~0u << (8 * left);
    u[i] = (u[i] & keep) | (fresh & ~keep);
  }
  return w;
}

template <int HELD, class T>
__global__ __launch_bounds__(kThreads) void fx_kv_store_kernel(const FxKvCache c, const FxKvRows r, int per_wave, int n_chunks, int vec) {
  const int lane = (int)threadIdx.x & 63;
  const int64_t w = (int64_t)blockIdx.x * kStoreWaves + ((int)threadIdx.x >> 6);
  const int half = (int)(w % 2), head = (int)((w / 2) % c.heads);
  const int64_t chunk = w / 2 / c.heads;
  if (chunk >= n_chunks) return;
  const int D = c.depth, page = 1 << c.log_page, cpt = D >> 3;   // (8 numbers a lane and load)
  const int64_t n_slots = (int64_t)c.pages << c.log_page;
  const T* src = (const T*)(half ? r.v : r.k) + (int64_t)head * (half ? r.v_head : r.k_head);
  const int64_t stride = half ? r.v_token : r.k_token;
  const int t0 = (int)chunk * per_wave, t1 = min(r.tokens, t0 + per_wave);
  auto page_of = [&](int t) -> int64_t {   // -1: nowhere
    const int64_t s = r.slots[t];
    return s >= 0 && s < n_slots ? s >> c.log_page : -1;
  };
  for (int t = t0; t < t1; ++t) {
    const int64_t p = page_of(t);
    if (p < 0 || (t > 0 && page_of(t - 1) == p)) continue;   // (uniform: every lane reads the same slots)
    // the run's length, and whether its slots rise by one
    int n = 0;
    bool straight = true;
    const int64_t s0 = r.slots[t];
    for (;;) {
      const int u = t + n + lane;
      const bool mine = u < r.tokens && page_of(u) == p;
      const unsigned long long same = __ballot(mine), rising = __ballot(mine && r.slots[u] == s0 + n + lane);
      const int more = ~same == 0 ? 64 : __builtin_ctzll(~same);
      const unsigned long long part = more == 64 ? ~0ull : (1ull << more) - 1;
      straight = straight && (rising & part) == part;
      n += more;
      if (more < 64) break;
    }
    const int o0 = (int)(s0 & (page - 1));
    uint8_t* codes = (half ? c.v + p * c.v_stride : c.k + p * c.k_stride) + (int64_t)head * page * D;
    float* scales = half ? c.v_scale + p * c.vs_stride + head : c.k_scale + p * c.ks_stride + head;
    const T* rows = src + (int64_t)t * stride;
    // the scale
    float top = 0.0f;
    const int64_t n8 = (int64_t)n * cpt;
    for (int64_t i = lane; i < n8; i += 64) {
      const int64_t j = i / cpt;
      float x[8];
      load8(x, rows + j * stride + (i - j * cpt) * 8, vec);
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, finite_abs(x[e]));
    }
    float scale = scale_of<HELD>(wave_max64(top));
    if (o0 > 0) {
      const float old = *scales;
      if (old > scale && old <= 3.402823466e38f) {
        scale = old;
      } else if (old < scale && old > 0.0f) {
        // what the page holds below o0: as many whole columns of 16 as there are, the last one in part
        const float ratio = old / scale;
        const int words = half ? ((o0 + 15) >> 4) * D : (o0 * D) >> 4;
        for (int i = lane; i < words; i += 64) {
          uint4* at = (uint4*)codes + i;
          *at = again16<HELD>(*at, ratio, half ? o0 - (i / D) * 16 : 16);
        }
      }
    }
    if (lane == 0) *scales = scale;
    const float inv = 1.0f / scale;   // (a power of two: exact)
    if (straight && !half) {
      for (int64_t i = lane; i < n8; i += 64) {
        const int64_t j = i / cpt;
        float x[8];
        load8(x, rows + j * stride + (i - j * cpt) * 8, vec);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= inv;
        uint2 u;
        u.x = encode4<HELD>(x);
        u.y = encode4<HELD>(x + 4);
        *(uint2*)(codes + (int64_t)(o0 + j) * D + (i - j * cpt) * 8) = u;
      }
      continue;
    }
    // values, or slots in any order: whole groups of 16 tokens that lie as in the cache, the others token by token (in order,
    // so that of two rows for one slot the later one stays)
    for (int i = 0; i < n;) {
      const int o = (int)(r.slots[t + i] & (page - 1));
      if (half && straight && (o & 15) == 0 && n - i >= 16) {
        for (int d = lane; d < D; d += 64) {
          unsigned u[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = (float)rows[(int64_t)(i + 4 * q + e) * stride + d] * inv;
            u[q] = encode4<HELD>(x);
          }
          *(uint4*)(codes + (int64_t)(o >> 4) * 16 * D + (int64_t)d * 16) = make_uint4(u[0], u[1], u[2], u[3]);
        }
        i += 16;
        continue;
      }
      for (int d = lane; d < D; d += 64) {
        const float x[4] = {(float)rows[(int64_t)i * stride + d] * inv, 0.0f, 0.0f, 0.0f};
        const uint8_t code = (uint8_t)encode4<HELD>(x);
        if (half) codes[(int64_t)(o >> 4) * 16 * D + (int64_t)d * 16 + (o & 15)] = code;
        else codes[(int64_t)o * D + d] = code;
      }
      ++i;
    }
  }
}

// ---- fx_kv_read ----
// Bound: HBM (1 byte read and 2 or 4 written for each number).  A wave takes the keys or the values of one head for
// up to 16 entries of `slots`; values by the group of 16 tokens that neighbours share, a lane a column.
template <int HELD, class T>
__global__ __launch_bounds__(kThreads) void fx_kv_read_kernel(const FxKvCache c, const FxKvRows r, int per_wave, int n_chunks) {
  const int lane = (int)threadIdx.x & 63;
  const int64_t w = (int64_t)blockIdx.x * kStoreWaves + ((int)threadIdx.x >> 6);
  const int half = (int)(w % 2), head = (int)((w / 2) % c.heads);
  const int64_t chunk = w / 2 / c.heads;
  if (chunk >= n_chunks) return;
  const int D = c.depth, page = 1 << c.log_page;
  const int64_t n_slots = (int64_t)c.pages << c.log_page;
  T* dst = (T*)(half ? r.v : r.k) + (int64_t)head * (half ? r.v_head : r.k_head);
  const int64_t stride = half ? r.v_token : r.k_token;
  const int t0 = (int)chunk * per_wave, t1 = min(r.tokens, t0 + per_wave);
  for (int t = t0; t < t1;) {
    const int64_t s = r.slots[t];
    T* row = dst + (int64_t)t * stride;
    if (s < 0 || s >= n_slots) {
      for (int d = lane; d < D; d += 64) row[d] = (T)0.0f;
      ++t;
      continue;
    }
    const int64_t p = s >> c.log_page;
    const int o = (int)(s & (page - 1));
    const float scale = half ? c.v_scale[p * c.vs_stride + head] : c.k_scale[p * c.ks_stride + head];
    if (!half) {
      const uint8_t* codes = c.k + p * c.k_stride + ((int64_t)head * page + o) * D;
      for (int d = lane * 4; d < D; d += 256) {
        float x[4];
        decode4<HELD>(x, *(const unsigned*)(codes + d));
#pragma unroll
        for (int e = 0; e < 4; ++e) row[d + e] = (T)(x[e] * scale);
      }
      ++t;
      continue;
    }
    int n = 1;
    while (t + n < t1 && (o & 15) + n < 16 && r.slots[t + n] == s + n) ++n;
    const uint8_t* codes = c.v + p * c.v_stride + (int64_t)head * page * D + (int64_t)(o >> 4) * 16 * D;
    for (int d = lane; d < D; d += 64) {
      const uint4 u = *(const uint4*)(codes + (int64_t)d * 16);
      const unsigned word[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float x[4];
        decode4<HELD>(x, word[q]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = 4 * q + e - (o & 15);
          if (j >= 0 && j < n) row[(int64_t)j * stride + d] = (T)(x[e] * scale);
        }
      }
    }
    t += n;
  }
}

// tokens a wave takes: as many as leave some 8 192 waves (32 a CU), 16 at most
int tokens_a_wave(const FxKvCache& c, const FxKvRows& r) {
  int64_t per = (int64_t)r.tokens * c.heads * 2 / 8192;
  return (int)(per < 1 ? 1 : per > 16 ? 16 : per);
}
bool aligned16(const void* p, int64_t a, int64_t b, size_t size) {
  return ((uintptr_t)p & 15u) == 0 && a * (int64_t)size % 16 == 0 && b * (int64_t)size % 16 == 0;
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
  const size_t size = r.dtype == FX_DT_F32 ? 4 : 2;
  int per = tokens_a_wave(c, r), chunks = (r.tokens + per - 1) / per;
  int vec = aligned16(r.k, r.k_token, r.k_head, size) && aligned16(r.v, r.v_token, r.v_head, size);
  FxKvCache cache = c;
  FxKvRows rows = r;
  void* kargs[5] = {(void*)&cache, (void*)&rows, (void*)&per, (void*)&chunks, (void*)&vec};
  const int64_t waves = (int64_t)chunks * c.heads * 2;
  return hipLaunchKernel(kernels[held][r.dtype == FX_DT_F32 ? 0 : r.dtype == FX_DT_F16 ? 1 : 2],
                         dim3((unsigned)((waves + kStoreWaves - 1) / kStoreWaves)), dim3(kThreads), kargs, 0, stream);
}

hipError_t fx_launch_kv_read(const FxKvCache& c, const FxKvRows& r, int held, hipStream_t stream) {
  static const void* const kernels[2][3] = {
      {(const void*)fx_kv_read_kernel<0, float>, (const void*)fx_kv_read_kernel<0, _Float16>, (const void*)fx_kv_read_kernel<0, __bf16>},
      {(const void*)fx_kv_read_kernel<1, float>, (const void*)fx_kv_read_kernel<1, _Float16>, (const void*)fx_kv_read_kernel<1, __bf16>}};
  int per = tokens_a_wave(c, r), chunks = (r.tokens + per - 1) / per;
  FxKvCache cache = c;
  FxKvRows rows = r;
  void* kargs[4] = {(void*)&cache, (void*)&rows, (void*)&per, (void*)&chunks};
  const int64_t waves = (int64_t)chunks * c.heads * 2;
  return hipLaunchKernel(kernels[held][r.dtype == FX_DT_F32 ? 0 : r.dtype == FX_DT_F16 ? 1 : 2],
                         dim3((unsigned)((waves + kStoreWaves - 1) / kStoreWaves)), dim3(kThreads), kargs, 0, stream);
}
