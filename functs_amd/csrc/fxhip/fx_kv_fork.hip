// Pages of the paged cache behind a beam search's selection: whose they are (fx_kv_fork), and what has to be copied (fx_kv_copy).
//
// fx_kv_fork: bound by latency (a few bytes a row and a page).  Three launches, in which nothing waits for another workgroup.  fx_kv_fork_plan,
// one workgroup for all rows, decides who gets which page where a page is partly filled; fx_kv_fork_tables, a workgroup for 256 columns of a group's rows,
// moves the tables and finds the pages that nobody has any more; fx_kv_fork_pack puts those side by side.  Small tables: one workgroup does all three
// (fx_kv_fork_small).  32 groups of 4 beams, 33 columns: 9.5 us, and 13.4 in three launches; 61 of 8 beams, 938 columns: 5.3 + 5.5 + 3.2 us.
#include <algorithm>

#include "fx_kv_fork.h"

namespace {
constexpr int kPlanThreads = 1024, kThreads = 256;
// Entries of the table that one workgroup takes, of groups of so many beams (LDS), all of them filled: 4 096 in 9.2 us, and 11.4 in three launches; 16 384 in 19 to 23, and 14
constexpr int kSmallBeams = 8, kSmall = 6144;

// Who gets which page.  HERE: at most kPlanThreads / K * K rows; what is said of row r stays in LDS (tail: last, len: held, want: tokens, flags: 1 alive, 2 reused, from).
struct Plan {
  int tail[kPlanThreads], len[kPlanThreads], want[kPlanThreads], flags[kPlanThreads], spare[kPlanThreads], from[kPlanThreads];
  int64_t sum[kPlanThreads / 64];
  __device__ __forceinline__ FxKvForkRow row(int r) const { return {from[r], tail[r], want[r], len[r], flags[r] & 1, flags[r] >> 1, {0, 0}}; }
};
template <bool HERE>
__device__ __forceinline__ void plan_rows(const FxKvForkArgs& a, Plan& s) {
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6, K = a.beams, page = 1 << a.log_page;
  const int rows = a.groups * K, a_round = kPlanThreads / K * K;
  const int own = tid < a_round ? tid % K : 0, first = tid - own;   // place in the group, and the group's first place here
  const int64_t from = a.free_start ? min(max((int64_t)*a.free_start, (int64_t)0), (int64_t)a.n_free) : 0;
  const int64_t room = (int64_t)a.columns << a.log_page;
  int64_t asked = 0;   // free pages of the groups before this round's
  for (int r0 = 0; r0 < rows; r0 += a_round) {
    const int r = r0 + tid;
    const bool here = tid < a_round && r < rows;
    int held = 0, tail = -1, parent = -1;
    if (here) {
      parent = a.parents[r];
      held = a.lens[r];
      if (held < 0 || held > room) held = 0;
      if ((held & (page - 1)) != 0) tail = a.table[(int64_t)r * a.table_stride + (held >> a.log_page)];
    }
    const bool has = here && parent >= 0 && parent < K;
    __syncthreads();   // (the round before has been read)
    s.tail[tid] = tail;
    s.len[tid] = held;
    __syncthreads();
    const int tokens = has ? s.len[first + parent] : 0, want = has ? s.tail[first + parent] : -1;
    s.want[tid] = want;
    __syncthreads();
    // of the rows that continue a partly filled page the first has it; a page that nobody continues is spare (of rows that share one: once)
    bool need = false, spare = here && tail >= 0;
    if (here) {
#pragma unroll 4
      for (int j = 0; j < K; ++j) {
        const int w = s.want[first + j], t = s.tail[first + j];
        need |= (j < own) & (want >= 0) & (w == want);
        spare &= (w != tail) & !((j < own) & (t == tail));
      }
    }
    s.flags[tid] = (need ? 1 : 0) | (spare ? 2 : 0);
    __syncthreads();
    int needs = 0, spares = 0, needs_before = 0, spares_before = 0;
    if (here) {
#pragma unroll 4
      for (int j = 0; j < K; ++j) {
        const int f = s.flags[first + j];
        needs += f & 1;
        spares += f >> 1;
        needs_before += j < own ? f & 1 : 0;
        spares_before += j < own ? f >> 1 : 0;
      }
    }
    if (spare) s.spare[first + spares_before] = tail;
    // free pages of this round's groups before this one
    int64_t before = own == 0 && here ? max(needs - spares, 0) : 0;
    const int64_t mine = before;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t o = (int64_t)__shfl_up((unsigned long long)before, (unsigned)d, 64);
      if (lane >= d) before += o;
    }
    if (lane == 63) s.sum[wave] = before;
    __syncthreads();
    int64_t all = 0;
    before -= mine;
#pragma unroll 4
    for (int w = 0; w < kPlanThreads / 64; ++w) {
      if (w < wave) before += s.sum[w];
      all += s.sum[w];
    }
    if (own == 0) s.len[tid] = (int)min(before, (int64_t)0x7fffffff);   // (lengths have been read)
    __syncthreads();
    before = s.len[first];
    int last = want;
    bool granted = has;
    if (need) {
      if (needs_before < spares) {
        last = s.spare[first + needs_before];
      } else {
        const int64_t index = from + asked + before + (needs_before - spares);
        granted = index < a.n_free;
        last = granted ? a.free_pages[index] : -1;
      }
    }
    s.from[tid] = granted ? parent : -1;
    __syncthreads();
    if (here) {
      bool alive = false;
#pragma unroll 4
      for (int j = 0; j < K; ++j) alive |= s.from[first + j] == own;
      const bool reused = spare && spares_before < needs;
      if constexpr (HERE) {
        s.tail[tid] = last;
        s.len[tid] = held;   // (own == 0: `before` has been read)
        s.want[tid] = tokens;
        s.flags[tid] = (alive ? 1 : 0) | (reused ? 2 : 0);
      } else {
        a.rows[r] = FxKvForkRow{granted ? parent : -1, last, tokens, held, alive ? 1 : 0, reused ? 1 : 0, {0, 0}};
      }
      a.out_lens[r] = granted ? tokens : 0;
      const bool copied = need && granted;
      a.copies[3 * (int64_t)r] = copied ? want : -1;
      a.copies[3 * (int64_t)r + 1] = copied ? last : -1;
      a.copies[3 * (int64_t)r + 2] = copied ? tokens & (page - 1) : 0;
    }
    asked += all;
  }
  if (tid == 0) *a.taken = (int)min(asked, (int64_t)a.n_free - from);
}

// One column of a group's rows, whose table begins at `table`: the new rows' pages.  Says which old rows' pages nobody has any more; pages: LDS of this thread alone, a row's `apart`.
template <class Rows>
__device__ __forceinline__ unsigned move_column(const FxKvForkArgs& a, const Rows& rows, int32_t* table, int c, int* pages, int apart) {
  const int K = a.beams, page = 1 << a.log_page;
  // what the group's rows have: pages up to the one in which their tokens end (-1 behind).  (Loops are without branches, so that their reads do not wait for each other.)
  uint32_t alive = 0;
#pragma unroll 4
  for (int i = 0; i < K; ++i) {
    const FxKvForkRow row = rows(i);
    const bool has = c < (row.held + page - 1) >> a.log_page;
    pages[i * apart] = has ? table[(int64_t)i * a.table_stride + c] : -1;
    alive |= (row.alive != 0 ? 1u : 0u) << i;
  }
#pragma unroll 4
  for (int j = 0; j < K; ++j) {
    const FxKvForkRow row = rows(j);
    const int whole = row.tokens >> a.log_page, moved = pages[max(row.from, 0) * apart];
    const bool ends = (c == whole) & ((row.tokens & (page - 1)) != 0);
    if ((row.from >= 0) & (((c < whole) & (row.from != j)) | ends)) table[(int64_t)j * a.table_stride + c] = ends ? row.last : moved;
  }
  unsigned gone = 0;
  for (int i = 0; i < K; ++i) {
    if ((alive >> i & 1) != 0) continue;
    const int p = pages[i * apart];
    const FxKvForkRow row = rows(i);
    if (p < 0 || (row.reused && c == row.held >> a.log_page)) continue;
    const unsigned others = alive | ((1u << i) - 1);   // that keep it, or have said so (i is not among them)
    bool kept = false;
#pragma unroll 8
    for (int o = 0; o < K; ++o) kept |= ((others >> o & 1) != 0) & (pages[o * apart] == p);
    gone |= kept ? 0u : 1u << i;
  }
  return gone;
}
// the sum of a wave's values up to each lane's
__device__ __forceinline__ int sum_up_to(int v, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(v, (unsigned)d, 64);
    v += lane >= d ? o : 0;
  }
  return v;
}

__global__ __launch_bounds__(kPlanThreads) void fx_kv_fork_plan(const FxKvForkArgs a) {
  __shared__ Plan s;
  plan_rows<false>(a, s);
  if (threadIdx.x == 0 && a.groups * a.blocks == 0) *a.n_freed = 0;   // (nothing else is launched)
}

// All of it, for few rows and columns
__global__ __launch_bounds__(kPlanThreads) void fx_kv_fork_small(const FxKvForkArgs a) {
  extern __shared__ int s_pages[];   // [beams][kPlanThreads]
  __shared__ Plan s;
  __shared__ int s_upto[2][kPlanThreads / 64];
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6, K = a.beams;
  plan_rows<true>(a, s);
  __syncthreads();
  int most = tid < a.groups * K ? s.len[tid] : 0;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) most = max(most, __shfl_xor(most, d, 64));
  if (lane == 0) s_upto[0][wave] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kPlanThreads / 64; ++w) most = max(most, s_upto[0][w]);
  __syncthreads();
  // (a column in which no row has a page stays as it is)
  const int columns = (most + (1 << a.log_page) - 1) >> a.log_page, items = a.groups * columns;
  int freed = 0;
  for (int i0 = 0, turn = 0; i0 < items; i0 += kPlanThreads, turn ^= 1) {
    const int i = i0 + tid, g = i / columns, c = i - g * columns;
    unsigned gone = 0;
    if (i < items) gone = move_column(a, [&](int j) { return s.row(g * K + j); }, a.table + (int64_t)g * K * a.table_stride, c, s_pages + tid, kPlanThreads);
    const int mine = __builtin_popcount(gone), upto = sum_up_to(mine, lane);
    if (lane == 63) s_upto[turn][wave] = upto;
    __syncthreads();
    int at = freed + upto - mine;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 64; ++w) {
      at += w < wave ? s_upto[turn][w] : 0;
      freed += s_upto[turn][w];
    }
    for (; gone != 0; gone &= gone - 1) a.freed[at++] = s_pages[__builtin_ctz(gone) * kPlanThreads + tid];
  }
  for (int i = freed + tid; i < a.groups * K * a.columns; i += kPlanThreads) a.freed[i] = -1;
  if (tid == 0) *a.n_freed = freed;
}

__global__ __launch_bounds__(kThreads) void fx_kv_fork_tables(const FxKvForkArgs a) {
  extern __shared__ int s_pages[];   // [beams][FX_KV_FORK_COLUMNS]
  __shared__ FxKvForkRow s_row[FX_BEAM_MAX_BEAMS];
  __shared__ int s_sum[kThreads / 64];
  static_assert(FX_KV_FORK_COLUMNS == kThreads, "a column each");
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6, K = a.beams;
  const int group = (int)(blockIdx.x / (unsigned)a.blocks), block = (int)(blockIdx.x % (unsigned)a.blocks);
  if (tid < K * (int)(sizeof(FxKvForkRow) / 4)) ((int*)s_row)[tid] = ((const int*)(a.rows + (int64_t)group * K))[tid];
  __syncthreads();
  int most = 0;
#pragma unroll 4
  for (int i = 0; i < K; ++i) most = max(most, s_row[i].held);
  if (((int64_t)block * kThreads << a.log_page) >= most) {   // (no row has a page here)
    if (tid == 0) a.counts[blockIdx.x] = 0;
    return;
  }
  unsigned gone = move_column(a, [&](int j) { return s_row[j]; }, a.table + (int64_t)group * K * a.table_stride, block * kThreads + tid, s_pages + tid, kThreads);
  // column by column
  const int mine = __builtin_popcount(gone), upto = sum_up_to(mine, lane);
  if (lane == 63) s_sum[wave] = upto;
  __syncthreads();
  int at = upto - mine, all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    if (w < wave) at += s_sum[w];
    all += s_sum[w];
  }
  int32_t* list = a.lists + (int64_t)blockIdx.x * K * kThreads;
  for (; gone != 0; gone &= gone - 1) list[at++] = s_pages[__builtin_ctz(gone) * kThreads + tid];
  if (tid == 0) a.counts[blockIdx.x] = all;
}

__global__ __launch_bounds__(kThreads) void fx_kv_fork_pack(const FxKvForkArgs a) {
  __shared__ int64_t s_sum[2][kThreads / 64];
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6, units = a.groups * a.blocks, unit = (int)blockIdx.x;
  int64_t before = 0, all = 0;
  for (int u = tid; u < units; u += kThreads) {
    const int n = a.counts[u];
    all += n;
    before += u < unit ? n : 0;
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    before += (int64_t)__shfl_xor((unsigned long long)before, d, 64);
    all += (int64_t)__shfl_xor((unsigned long long)all, d, 64);
  }
  if (lane == 0) s_sum[0][wave] = before, s_sum[1][wave] = all;
  __syncthreads();
  before = all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) before += s_sum[0][w], all += s_sum[1][w];
  const int n = a.counts[unit];
  const int32_t* list = a.lists + (int64_t)unit * a.beams * kThreads;
  for (int i = tid; i < n; i += kThreads) a.freed[before + i] = list[i];
  // places behind the last
  const int64_t places = (int64_t)a.groups * a.beams * a.columns, a_unit = (places + units - 1) / units;
  const int64_t to = min(places, (unit + 1) * a_unit);
  for (int64_t i = max(all, unit * a_unit) + tid; i < to; i += kThreads) a.freed[i] = -1;
  if (unit == 0 && tid == 0) *a.n_freed = (int)all;
}

// ---- fx_kv_copy ----
// Bound: HBM, each code read and written once.  A unit is some heads of one page's keys or values in one layer: up to 16 KiB, whose filled part is
// copied 16 bytes a lane.  Every workgroup lists the rows that copy (most have none) and takes units in turn.
// 56 copies of 8 partly filled pages in 24 layers (8 heads of 128, 64 tokens): 32 us for 95 MB written, which the stores' way is full with (2 048 to 16 384 workgroups: 32 to
// 34); a step's, of 16 x 4 beams, pages of 16 tokens in 12 layers: 5.3 us, a chain of launch, list, loads.
constexpr int kRows = 1024;   // looked at together
typedef unsigned fx_words __attribute__((ext_vector_type(4)));

__global__ __launch_bounds__(kThreads) void fx_kv_copy_kernel(const FxKvCopyArgs a) {
  __shared__ int s_list[3][kRows];
  __shared__ int s_count[kThreads / 64];
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int D = a.c.depth, page = 1 << a.c.log_page, H = a.c.heads;
  for (int r0 = 0; r0 < a.rows; r0 += kRows) {
    int listed = 0;
    __syncthreads();   // (the list before has been read)
    for (int i = 0; i < kRows; i += kThreads) {
      const int r = r0 + i + tid;
      bool live = false;
      int from = -1, to = -1, tokens = 0;
      if (r < a.rows) {
        from = a.copies[3 * (int64_t)r];
        to = a.copies[3 * (int64_t)r + 1];
        tokens = a.copies[3 * (int64_t)r + 2];
        live = from >= 0 && from < a.c.pages && to >= 0 && to < a.c.pages && from != to;
      }
      const uint64_t lanes = __ballot(live);
      if (lane == 0) s_count[wave] = __builtin_popcountll(lanes);
      __syncthreads();
      int at = listed + __builtin_popcountll(lanes & ((1ull << lane) - 1));
#pragma unroll
      for (int w = 0; w < kThreads / 64; ++w) {
        if (w < wave) at += s_count[w];
        listed += s_count[w];
      }
      if (live) s_list[0][at] = from, s_list[1][at] = to, s_list[2][at] = min(max(tokens, 0), page);
      __syncthreads();
    }
    const unsigned units = (unsigned)(listed * a.layers * 2 * a.units_a_page);   // (at most 1 024 * 32 * 2 * 64)
    for (unsigned u = blockIdx.x; u < units; u += gridDim.x) {
      const unsigned page_unit = u / (unsigned)a.units_a_page, copy_layer = page_unit >> 1;
      const int part = (int)(u - page_unit * (unsigned)a.units_a_page), half = (int)(page_unit & 1);
      const int copy = (int)(copy_layer / (unsigned)a.layers), layer = (int)(copy_layer - (unsigned)copy * (unsigned)a.layers);
      const int64_t from = __builtin_amdgcn_readfirstlane(s_list[0][copy]), to = __builtin_amdgcn_readfirstlane(s_list[1][copy]);
      const int filled = __builtin_amdgcn_readfirstlane(s_list[2][copy]);
      const int h0 = part * a.heads_a_unit, heads = min(a.heads_a_unit, H - h0);
      const int stride = page * D >> 4, words = (half == 0 ? filled : (filled + 15) & ~15) * D >> 4;   // 16 bytes of a head, and those that are filled
      uint8_t* const codes = half == 0 ? a.layer[layer].k : a.layer[layer].v;
      const uint32_t page_stride = half == 0 ? a.c.k_stride : a.c.v_stride, scale_stride = half == 0 ? a.c.ks_stride : a.c.vs_stride;
      const fx_words* src = (const fx_words*)(codes + from * page_stride) + (int64_t)h0 * stride;
      fx_words* dst = (fx_words*)(codes + to * page_stride) + (int64_t)h0 * stride;
      float* const scales = half == 0 ? a.layer[layer].ks : a.layer[layer].vs;
      for (int h = tid; h < heads; h += kThreads) scales[to * scale_stride + h0 + h] = scales[from * scale_stride + h0 + h];
      const int n = heads * words;
      // (i + 1/2) / words is half a word's share away from whole numbers at least, h 2^-22 off at most
      const float share = 1.0f / (float)words;
      const bool exact = n < 1 << 20;
      constexpr int kBatch = 4;
      for (int i0 = tid; i0 < n; i0 += kThreads * kBatch) {
        fx_words w[kBatch];
        int at[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
          const int i = min(i0 + b * kThreads, n - 1), h = exact ? (int)(((float)i + 0.5f) * share) : i / words;
          at[b] = h * stride + (i - h * words);
          w[b] = src[at[b]];
        }
#pragma unroll
        for (int b = 0; b < kBatch; ++b)
          if (i0 + b * kThreads < n) dst[at[b]] = w[b];
      }
    }
  }
}
}  // namespace

hipError_t fx_launch_kv_fork(const FxKvForkArgs& a, hipStream_t stream, int* launched) {
  FxKvForkArgs args = a;
  void* kargs[1] = {(void*)&args};
  *launched = 0;
  hipError_t e;
  if (a.beams <= kSmallBeams && a.groups <= kPlanThreads / a.beams && (int64_t)a.groups * a.beams * a.columns <= kSmall) {
    e = hipLaunchKernel((const void*)fx_kv_fork_small, dim3(1), dim3(kPlanThreads), kargs, (size_t)a.beams * kPlanThreads * sizeof(int), stream);
    *launched = e == hipSuccess ? 1 : 0;
    return e;
  }
  e = hipLaunchKernel((const void*)fx_kv_fork_plan, dim3(1), dim3(kPlanThreads), kargs, 0, stream);
  if (e != hipSuccess) return e;
  const unsigned units = (unsigned)a.groups * (unsigned)a.blocks;
  *launched = 1;
  if (units == 0) return e;
  e = hipLaunchKernel((const void*)fx_kv_fork_tables, dim3(units), dim3(kThreads), kargs, (size_t)a.beams * kThreads * sizeof(int), stream);
  if (e != hipSuccess) return e;
  e = hipLaunchKernel((const void*)fx_kv_fork_pack, dim3(units), dim3(kThreads), kargs, 0, stream);
  *launched = e == hipSuccess ? 3 : 2;
  return e;
}

hipError_t fx_launch_kv_copy(const FxKvCopyArgs& a, hipStream_t stream) {
  FxKvCopyArgs args = a;
  void* kargs[1] = {(void*)&args};
  // as many workgroups as there may be units, 16 a CU at most (eight are there at once; the others start as these end)
  const int64_t units = (int64_t)a.rows * a.layers * 2 * a.units_a_page;
  return hipLaunchKernel((const void*)fx_kv_copy_kernel, dim3((unsigned)std::min<int64_t>(units, 4096)), dim3(kThreads), kargs, 0, stream);
}
