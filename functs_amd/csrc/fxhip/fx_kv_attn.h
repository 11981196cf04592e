// Attention over the paged 8-bit cache (fx_kv_attention).
//   row i of request b (n rows, len cached tokens): position p = len - n + i, sees tokens j <= p, j > p - window, page in the cache
//   s_j = scale * q . k_j;  out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  lse = m + log sum_j e^(s_j - m)
// in one pass over the cached tokens with a running maximum, sum and output.
//
// Both products run on the matrix cores, transposed: S^T = K Q^T and O^T = V^T P^T.  The scores of S^T lie in the
// registers in which P^T is read (a lane holds 16 tokens of one row of queries), so they never cross lanes or
// LDS.  Which token is which row of K's operand is free: token (m / 4) * 16 + 4 r + m % 4 in row m of product r gives each
// lane the 16 neighbouring tokens of one group, so one page, one scale of keys (on the scores) and one of values (on the
// weights) a lane.  The depth of the first product is contracted in the order in which lanes load 16 bytes each.
// Codes become bf16 (or f16) exactly; fp32 queries and the weights are sums of two or three such numbers:
//   queries  bf16, f16: as they are;  fp32: three bf16 (24 bits)
//   weights  fp32 results: three bf16;  f16: two (16 bits);  bf16: two in fx_kv_rows, which waits for memory anyway, one in
//            fx_kv_tiles: weights of one bf16 are off by half a step each, no more than the result's own rounding is (2-norm of
//            the error of prompts, against 64 bits: 0.0019, the result's rounding alone 0.0016), and two, as f16 calls have them,
//            take 491 us where one takes 377.  Sums of the weights are fp32, of weights as they were
#pragma once
#include <type_traits>

#include "fx_kv.h"
#include "fx_kv_device.h"

typedef __bf16 fx_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 fx_bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 fx_f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 fx_f16x2 __attribute__((ext_vector_type(2)));
typedef float fx_f32x4 __attribute__((ext_vector_type(4)));

namespace fxkv {
typedef const __attribute__((address_space(4))) FxKvAttnArgs KernelArgs;   // where a kernel's arguments are
constexpr float kInf = __builtin_inff(), kLn2 = 0.693147180559945309f;
constexpr float kTiny = 1.17549435e-38f;   // in place of scales of 0 (memory that nobody has written): -inf and 0 stay what they are under it
// Weights are 2^(score - m) in base 2, at most 1: m is kHead above the largest score when it is set, and raised where a score is above it
constexpr float kHead = 8.0f;
constexpr float kMost = 3.402823466e38f;   // of values' scales of infinity: the weight of a token that a row does not see stays 0
// Weights have the values' scale in their exponent.  Their sum is taken from them where the scale lies in this range, so that no weight that
// counts leaves the range of normal numbers; under other scales from exponentials of its own (weight_sum)
constexpr float kFoldLeast = 0x1p-64f, kFoldMost = 0x1p64f;
enum { kBf16 = 0, kF16 = 1, kF32 = 2 };   // types of queries and results

union Frag {   // eight 16-bit numbers of an operand
  unsigned u[4];
  fx_bf16x8 b;
  fx_f16x8 h;
};

// two codes of a word (its lower or upper half) as two 16-bit floats
template <int HELD, bool F16, bool HI>
__device__ __forceinline__ unsigned two(unsigned w) {
  if constexpr (HELD == 0) {
    if constexpr (F16) return __builtin_bit_cast(unsigned, (fx_f16x2)__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
    else return __builtin_bit_cast(unsigned, (fx_bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
  } else {
    const float x = (float)(signed char)(w >> (HI ? 16 : 0)), y = (float)(signed char)(w >> (HI ? 24 : 8));
    if constexpr (F16) return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pkrtz(x, y));
    else return __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);   // (at most 7 bits: the upper halves are exact)
  }
}
template <int HELD, bool F16>
__device__ __forceinline__ Frag eight(unsigned lo, unsigned hi) {
  Frag f;
  f.u[0] = two<HELD, F16, false>(lo);
  f.u[1] = two<HELD, F16, true>(lo);
  f.u[2] = two<HELD, F16, false>(hi);
  f.u[3] = two<HELD, F16, true>(hi);
  return f;
}
// the bytes of a word that are e4m3's NaN: 0x80 in each
__device__ __forceinline__ unsigned nan_codes(unsigned w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
template <bool F16>
__device__ __forceinline__ fx_f32x4 mfma16(const Frag& a, const Frag& b, fx_f32x4 c) {
  if constexpr (F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(a.h, b.h, c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.b, b.b, c, 0, 0, 0);
}
// x as the sum of N bf16 numbers: all but the last cut off (so that what is left is exact), the last rounded
template <int N>
__device__ __forceinline__ void split8(Frag (&f)[N], const float* x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      if (k == N - 1) {
        fx_bf16x2 r;
        r[0] = (__bf16)a;
        r[1] = (__bf16)b;
        f[k].u[i] = __builtin_bit_cast(unsigned, r);
      } else {
        f[k].u[i] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
        a -= __uint_as_float(__float_as_uint(a) & 0xffff0000u);
        b -= __uint_as_float(__float_as_uint(b) & 0xffff0000u);
      }
    }
  }
}

// ---- which workgroup does what (fx_kv_split.h) ----
struct Unit {
  FxKvRequest r;
  int request, head, tile, split, splits, part, item;
};
// (a request whose rows are the other kernel's has no tiles here)
__device__ __forceinline__ FxKvRequest request_of(const FxKvAttnArgs& a, int start, int end, int len, int tile_rows) {
  FxKvRequest r = fx_kv_request(start, end, len, a.tokens, a.columns << a.c.log_page, a.group, a.window, tile_rows);
  if ((int64_t)r.rows * a.group <= a.rows_above || (int64_t)r.rows * a.group > a.rows_upto) r.tiles = 0;
  return r;
}
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int v) { return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false); }
// sum over the lanes up to this one
__device__ __forceinline__ int sum_upto(int v) {
  v = dpp_add<0x111, 0xf>(v);   // row_shr: 1, 2, 4, 8
  v = dpp_add<0x112, 0xf>(v);
  v = dpp_add<0x114, 0xf>(v);
  v = dpp_add<0x118, 0xf>(v);
  v = dpp_add<0x142, 0xa>(v);   // row_bcast: 15, 31
  return dpp_add<0x143, 0xc>(v);
}
// 43-bit numbers of the lanes, added up in two parts; one that is larger (no call has so many steps) counts as endless: nothing is cut then
__device__ __forceinline__ int64_t wave_total(int64_t v) {
  const bool endless = v >= int64_t{1} << 43;
  const int low = sum_upto((int)(v & 0xfffff)), high = sum_upto(endless ? 0 : (int)(v >> 20));
  const int64_t all = ((int64_t)__builtin_amdgcn_readlane(high, 63) << 20) + __builtin_amdgcn_readlane(low, 63);
  return __any(endless) ? FX_KV_ENDLESS : all;
}
__device__ __forceinline__ int64_t all_steps(const FxKvAttnArgs& a, int64_t steps) {   // of all heads
  return steps >= FX_KV_ENDLESS ? steps : steps * a.c.heads;
}

// Unit u of the call, or false behind the last one: every wave finds it by itself, in scalar registers, without a barrier.  Up
// to kScanned requests are added up here, one a lane; of more, fx_kv_offsets has left the sums (130 requests of 300 tokens took 35 us so,
// 39 with rounds of 64 here; 250 took 51 and 64, 700 of 100 tokens 86 and 211).
// SORTED: of up to 64 requests those of more steps come first, so that what is left at the end of a call is short: fx_kv_tiles (prompts
// 415 us without, 391 with); fx_kv_rows, of many workgroups a CU, took 71 us for 64 requests of up to 4 000 tokens with it and 62 without.
constexpr int kScanned = 64;
// Chunks are multiples of so many steps: fx_kv_rows, of one for each wave; fx_kv_tiles, so that what a part costs by itself (some 8 us) stays
// small: 4 requests of 256 rows on 3 000 cached tokens, 12 heads of 64, took 67 us with 4, 68 with 8 and 86 with 2; one of 8 000 37, 39 and 37
constexpr int kRowLeast = 4, kTileLeast = 4;
template <bool SORTED>
__device__ __forceinline__ bool unit_at(const FxKvAttnArgs& a, int tile_rows, int least, int u, Unit& x, int* shared_items) {
  const int lane = (int)threadIdx.x & 63;
  int chunk, rest, parts;   // rest: the unit's number in its request; parts: items << 16 | parts before the request
  if (a.requests <= kScanned) {
    // (all three loads at once, whatever the lane)
    const int c = max(min(lane, a.requests - 1), 0), start = a.starts[c], end = a.starts[c + (a.requests > 0 ? 1 : 0)], len = a.requests > 0 ? a.lens[c] : 0;
    const int behind = lane < a.requests ? end : start;
    const FxKvRequest r = request_of(a, start, behind, len, tile_rows);
    chunk = fx_kv_chunk(all_steps(a, wave_total(fx_kv_work(start, behind, r))), least);
    const int splits = fx_kv_parts(r.steps, chunk), items = r.tiles * a.c.heads, mine = items * splits, cut = splits > 1 ? (items << 16) + mine : 0;
    const int cuts = sum_upto(cut);
    int before = 0;
    if constexpr (SORTED) {
      for (int c = 0; c < a.requests; ++c) {
        const int n = __builtin_amdgcn_readlane(r.steps, c), add = __builtin_amdgcn_readlane(mine, c);
        if (n > r.steps || (n == r.steps && c < lane)) before += add;
      }
    } else {
      before = sum_upto(mine) - mine;
    }
    *shared_items = (unsigned)__builtin_amdgcn_readlane(cuts, 63) >> 16;
    const unsigned long long owner = __ballot(u >= before && u < before + mine);
    if (owner == 0) return false;
    const int L = __builtin_ctzll(owner);
    x.request = L;
    x.r.start = __builtin_amdgcn_readlane(r.start, L);
    x.r.rows = __builtin_amdgcn_readlane(r.rows, L);
    x.r.len = __builtin_amdgcn_readlane(r.len, L);
    x.r.tiles = __builtin_amdgcn_readlane(r.tiles, L);
    x.r.steps = __builtin_amdgcn_readlane(r.steps, L);
    rest = u - __builtin_amdgcn_readlane(before, L);
    parts = __builtin_amdgcn_readlane(cuts - cut, L);
  } else {
    const int32_t* units = a.offsets + 2;   // [requests + 1], then [requests] of parts
    chunk = a.offsets[0];
    *shared_items = a.offsets[1];
    int lo = 0, hi = a.requests;
    if (u < 0 || u >= units[hi]) return false;
    while (hi - lo > 1) {
      const int step = (hi - lo + 63) >> 6, at = min(lo + lane * step, hi);
      const int last = 63 - __builtin_clzll(__ballot(at < hi && units[at] <= u));   // (lane 0 always)
      lo += last * step;
      hi = min(lo + step, hi);
    }
    x.request = __builtin_amdgcn_readfirstlane(lo);
    rest = u - __builtin_amdgcn_readfirstlane(units[lo]);
    parts = __builtin_amdgcn_readfirstlane(units[a.requests + 1 + lo]);
    x.r = request_of(a, __builtin_amdgcn_readfirstlane(a.starts[lo]), __builtin_amdgcn_readfirstlane(a.starts[lo + 1]), __builtin_amdgcn_readfirstlane(a.lens[lo]), tile_rows);
  }
  // (the compiler does not know them as the same in all lanes)
  auto scalar = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
  x.request = scalar(x.request), rest = scalar(rest), parts = scalar(parts), chunk = scalar(chunk);
  x.r = FxKvRequest{scalar(x.r.start), scalar(x.r.rows), scalar(x.r.len), scalar(x.r.tiles), scalar(x.r.steps)};
  x.splits = scalar(fx_kv_parts(x.r.steps, chunk));
  int item;
  if (!fx_kv_item(x.r, a.c.heads, x.splits, rest, &item, &x.tile, &x.head)) return false;
  item = scalar(item), x.tile = scalar(x.tile), x.head = scalar(x.head);
  x.split = rest - item * x.splits;
  x.part = (parts & 0xffff) + item * x.splits;
  x.item = (int)((unsigned)parts >> 16) + item;
  return true;
}
__device__ __forceinline__ FxKvSpan scalars(const FxKvSpan& s) {
  return FxKvSpan{__builtin_amdgcn_readfirstlane(s.low),      __builtin_amdgcn_readfirstlane(s.high), __builtin_amdgcn_readfirstlane(s.all_low),
                  __builtin_amdgcn_readfirstlane(s.all_high), __builtin_amdgcn_readfirstlane(s.from), __builtin_amdgcn_readfirstlane(s.to)};
}
static_assert(2 * FX_KV_TARGET < 1 << 15 && FX_KV_TARGET < 1 << 15, "parts and items in 16 bits each");

template <class T>
__device__ __forceinline__ void store4(T* p, const float* x) {
  T y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = (T)x[i];
  if constexpr (sizeof(T) == 4) *(float4*)p = *(const float4*)y;
  else *(uint2*)p = *(const uint2*)y;
}
template <int TQ> struct TypeOf;
template <> struct TypeOf<kBf16> { typedef __bf16 type; };
template <> struct TypeOf<kF16> { typedef _Float16 type; };
template <> struct TypeOf<kF32> { typedef float type; };

// Eight numbers of a row of queries at depth d as operands (zeros where `in` is false: what is loaded then is the row's first ones)
template <int TQ, int NQ, class T>
__device__ __forceinline__ void load_query(Frag* const (&f)[NQ], const T* src, int d, bool in, bool vec) {
  const T* p = src + (in ? d : 0);
  union { uint4 u[sizeof(T) / 2]; T e[8]; } w;
  if (vec) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) w.u[i] = ((const uint4*)p)[i];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) w.e[e] = p[e];
  }
  if constexpr (TQ == kF32) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = in ? w.e[e] : 0.0f;
    Frag s[NQ];
    split8<NQ>(s, v);
#pragma unroll
    for (int k = 0; k < NQ; ++k) *f[k] = s[k];
  } else {
    f[0]->u[0] = in ? w.u[0].x : 0u;
    f[0]->u[1] = in ? w.u[0].y : 0u;
    f[0]->u[2] = in ? w.u[0].z : 0u;
    f[0]->u[3] = in ? w.u[0].w : 0u;
  }
}

// Rows of no request: zeros, and nothing under the logarithm
template <class T>
__device__ __forceinline__ void fill_rest(const FxKvAttnArgs& a) {
  const int lo = a.requests > 0 ? min(max(a.starts[0], 0), a.tokens) : 0, hi = a.requests > 0 ? min(max(a.starts[a.requests], 0), a.tokens) : 0;
  const int per = a.q_heads * a.c.depth;
  for (int t = (int)blockIdx.x; t < a.tokens; t += (int)gridDim.x) {
    if (t >= lo && t < hi) continue;
    for (int i = (int)threadIdx.x; i < per; i += (int)blockDim.x) ((T*)a.out)[(int64_t)t * a.out_token + i] = (T)0.0f;
    for (int i = (int)threadIdx.x; i < a.q_heads; i += (int)blockDim.x) a.lse[(int64_t)t * a.q_heads + i] = -kInf;
  }
}

// The sum of a lane's 16 weights without the values' scale
template <class Scores>
__device__ __forceinline__ float weight_sum(const Scores& s, float cs, float sub) {
  float sum = 0.0f;
#pragma unroll
  for (int e = 0; e < 16; ++e) sum += __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], cs, -sub));
  return sum;
}
__device__ __forceinline__ bool folds(float scale) { return scale >= kFoldLeast && scale <= kFoldMost; }

// the larger one; a NaN loses (fmaxf does the same and quiets what the matrix cores give it, an instruction for each)
__device__ __forceinline__ float larger(float a, float b) { return __builtin_amdgcn_fmed3f(a, b, __builtin_inff()); }

// ---- 16 rows a tile: single tokens and few rows ----
// Bound: HBM, each key and value is read once by one wave, straight into the registers of its operand; 64 tokens a
// step, the four waves of a workgroup in turn.  The loads of the next step's keys are under way during the softmax and the second
// product, those of the values during the first.
// Measured (e4m3, depth 128, 8 heads): one request of 130 000 tokens, 8 query heads to each, fp16, 49.5 us, 5.4 TB/s, as a large copy,
// and 4.6 of fx_kv_join; 64 requests of up to 4 000, 4 query heads, bf16, 58 to 62, 4.3 TB/s: units of unequal length.  A single
// request of 50 tokens 6.8 us, a chain of launch, lengths, table, codes and join within the workgroup.
template <int HELD, int TQ, int DP, bool EXACT>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void fx_kv_rows(const FxKvAttnArgs a) {
  typedef typename TypeOf<TQ>::type T;
  constexpr int W = 4, NQ = TQ == kF32 ? 3 : 1, NP = TQ == kF32 ? 3 : 2, C = DP / 64, DT = DP / 16, LD = DP + 4;
  constexpr bool F16 = TQ == kF16;
  __shared__ __align__(16) float s_acc[W][FX_KV_ROWS][LD];
  __shared__ float s_ml[W][FX_KV_ROWS][2];
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int col = lane & 15, kg = lane >> 4;
  const int D = EXACT ? DP : a.c.depth, G = a.group, lp = a.c.log_page, pm = (1 << lp) - 1;
  for (int u = (int)blockIdx.x;; u += (int)gridDim.x) {
    Unit x;
    int shared_items = 0;
    const bool live = unit_at<false>(a, FX_KV_ROWS, kRowLeast, u, x, &shared_items);
    if (u == 0 && threadIdx.x == 0) *a.parts.n_items = shared_items;
    if (!live) break;
    if (u != (int)blockIdx.x) __syncthreads();   // (LDS is free again)
    // rows
    const int r0 = x.tile * FX_KV_ROWS, row = r0 + col;
    const bool valid = row < x.r.rows * G;
    const int i = valid ? row / G : 0, g = valid ? row - i * G : 0;
    const int hi_row = valid ? x.r.len - x.r.rows + i + 1 : 0;                             // tokens [lo_row, hi_row)
    const int lo_row = a.window > 0 ? max(hi_row - a.window, 0) : 0;
    const FxKvSpan span = scalars(fx_kv_span(x.r, G, a.window, r0, FX_KV_ROWS, x.split, x.splits));
    const int from = span.from, to = span.to;
    // queries: lane kg holds depths 64 c + 16 kg ... + 15 of its row
    Frag q[NQ][2 * C];
    {
      const T* src = (const T*)a.q + (int64_t)(x.r.start + i) * a.q_token + (int64_t)(x.head * G + g) * a.q_head;
#pragma unroll
      for (int c = 0; c < 2 * C; ++c) {
        const int d = (c >> 1) * 64 + kg * 16 + (c & 1) * 8;
        Frag* f[NQ];
#pragma unroll
        for (int k = 0; k < NQ; ++k) f[k] = &q[k][c];
        load_query<TQ, NQ, T>(f, src, d, valid && d < D, a.q_vec != 0);
      }
    }
    fx_f32x4 acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d] = fx_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -kInf, l = 0.0f;
    bool nans = false;   // a step had values that are NaN and rows that do not see all its tokens
    const int32_t* table = a.table + (int64_t)x.request * a.table_stride;
    const int k_group = (col >> 2) * 16, k_row = col & 3;
    const int64_t head_at = (int64_t)x.head * (pm + 1) * D;
    auto entry_of = [&](int token) { return table[min(token >> lp, a.columns - 1)]; };   // as it is: looked at when it is used, a step later
    uint4 kr[4][C];
    // a lane beyond the depth takes its row's first numbers again: its queries there are 0
    int k_at[C];
#pragma unroll
    for (int c = 0; c < C; ++c) k_at[c] = c * 64 + kg * 16 < D ? c * 64 : -kg * 16;
    auto load_keys = [&](int step, int page) {
      const int at = (step * FX_KV_STEP + k_group) & pm;
      const uint8_t* p = a.c.k + (int64_t)page * a.c.k_stride + head_at + (int64_t)(at + k_row) * D + kg * 16;
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < C; ++c)
          kr[r][c] = *(const uint4*)(p + r * 4 * D + (EXACT ? c * 64 : k_at[c]));
    };
        // entries of the step after this one, and the page of this one's values
    int step = from + wave, entry = 0, next_k = 0, next_v = 0, pv = 0;
    if (step < to) {
      entry = entry_of(step * FX_KV_STEP + k_group);
      const int ev = entry_of(step * FX_KV_STEP + kg * 16);
      next_k = entry_of((step + W) * FX_KV_STEP + k_group);
      next_v = entry_of((step + W) * FX_KV_STEP + kg * 16);
      load_keys(step, max(fx_kv_page(entry, a.c.pages), 0));
      pv = fx_kv_page(ev, a.c.pages);
    }
    for (; step < to; step += W) {
      const int base = step * FX_KV_STEP;
      const bool ok = pv >= 0;
      const int page = max(pv, 0);
      const float ks = a.c.k_scale[(int64_t)page * a.c.ks_stride + x.head], vs = a.c.v_scale[(int64_t)page * a.c.vs_stride + x.head];
      uint4 vr[DT];
      {
        const uint8_t* p = a.c.v + (int64_t)page * a.c.v_stride + head_at + (int64_t)(((base + kg * 16) & pm) >> 4) * 16 * D + col * 16;
#pragma unroll
        for (int d = 0; d < DT; ++d) vr[d] = *(const uint4*)(p + (EXACT ? d * 256 : min(d * 16, D - 16) * 16));   // (beyond the depth: not used)
      }
      // (the last step loads its own keys once more: with a load that may not happen the compiler waits for the values and the next
      // keys together)
      const bool more = step + W < to;
      const int pk = max(fx_kv_page(more ? next_k : entry, a.c.pages), 0);
      pv = fx_kv_page(next_v, a.c.pages);
      entry = next_k;
      next_k = entry_of(base + 2 * W * FX_KV_STEP + k_group);
      next_v = entry_of(base + 2 * W * FX_KV_STEP + kg * 16);
      // scores
      float s[16];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        fx_f32x4 t = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const Frag k0 = eight<HELD, F16>(kr[r][c].x, kr[r][c].y), k1 = eight<HELD, F16>(kr[r][c].z, kr[r][c].w);
#pragma unroll
          for (int k = NQ - 1; k >= 0; --k) {
            t = mfma16<F16>(k0, q[k][2 * c], t);
            t = mfma16<F16>(k1, q[k][2 * c + 1], t);
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) s[r * 4 + e] = t[e];
      }
      load_keys(more ? step + W : step, pk);
      float cs = fmaxf(ks * a.scale, kTiny), vscale = __builtin_amdgcn_fmed3f(vs, kTiny, kMost);   // (NaN: kTiny)
      const bool inside = base >= span.all_low && base + FX_KV_STEP <= span.all_high && __all(ok);
      if (!inside) {
        int hi_row_ = hi_row, lo_row_ = lo_row;
        asm volatile("" : "+v"(hi_row_), "+v"(lo_row_));   // (compared here, not ahead of the branch)
        const int t0 = base + kg * 16;
        if (!ok || span.high <= t0 || t0 + 16 <= span.low) cs = vscale = 1.0f;   // (what lies there may be anything)
        const int h = ok ? hi_row_ - t0 : 0, b = lo_row_ - t0;
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = e < h && e >= b ? s[e] : -kInf;
        if constexpr (HELD == 0) {
          // a value that is NaN would reach the rows that do not see its token, as 0 * NaN: see below
          unsigned any = 0;
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            unsigned* v = (unsigned*)&vr[d];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const unsigned n = nan_codes(v[w]);
              any |= n;
              v[w] &= ~((n >> 7) * 0xffu);
            }
          }
          nans = nans || __any(any != 0);
        }
      }
      // running maximum: see kHead
      float top = larger(s[0], s[1]);
#pragma unroll
      for (int e = 2; e < 16; ++e) top = larger(top, s[e]);
      top *= cs;
      if (__any(top > m)) {
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float now = fmaxf(m, top + kHead);
        const float by = now == -kInf ? 1.0f : __builtin_amdgcn_exp2f(m - now);
        m = now;
        l *= by;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[d][e] *= by;
      }
      const float sub = m == -kInf ? 0.0f : m;
      // weights times the values' scale, a power of two: part of the exponent (see kFoldLeast), and taken out of their sum again
      Frag p[2][NP];
      float w[16], sum[2] = {0.0f, 0.0f};
      const float off = __builtin_amdgcn_logf(vscale) - sub;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], cs, off));
        sum[e & 1] += w[e];
      }
      float add = (sum[0] + sum[1]) * __builtin_amdgcn_rcpf(vscale);
      if (!__all(folds(vscale))) add = weight_sum(s, cs, sub);
      l += add;
      split8<NP>(p[0], w);
      split8<NP>(p[1], w + 8);
#pragma unroll
      for (int d = 0; d < DT; ++d)
        if (EXACT || d * 16 < D) {
          const Frag v0 = eight<HELD, false>(vr[d].x, vr[d].y), v1 = eight<HELD, false>(vr[d].z, vr[d].w);
#pragma unroll
          for (int k = NP - 1; k >= 0; --k) {
            acc[d] = mfma16<false>(v0, p[0][k], acc[d]);
            acc[d] = mfma16<false>(v1, p[1][k], acc[d]);
          }
        }
    }
    if constexpr (HELD == 0) {
      if (nans) {   // the rows that see a NaN get it here: in which column of the values, by a product of ones
        for (int again = from + wave; again < to; again += W) {
          const int t0 = again * FX_KV_STEP + kg * 16, page = fx_kv_page(entry_of(t0), a.c.pages), h = page >= 0 ? hi_row - t0 : 0, b = lo_row - t0;
          Frag sees[2];
#pragma unroll
          for (int k = 0; k < 8; ++k)
            sees[k >> 2].u[k & 3] = (2 * k < h && 2 * k >= b ? 0x3f80u : 0u) | (2 * k + 1 < h && 2 * k + 1 >= b ? 0x3f800000u : 0u);
          const uint8_t* v = a.c.v + (int64_t)max(page, 0) * a.c.v_stride + head_at + (int64_t)((t0 & pm) >> 4) * 16 * D;
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            uint4 is = *(const uint4*)(v + min(d * 16 + col, D - 1) * 16);
            unsigned* k = (unsigned*)&is;
#pragma unroll
            for (int w = 0; w < 4; ++w) k[w] = (nan_codes(k[w]) >> 7) * 0x38u;   // e4m3's 1
            fx_f32x4 n = {0.0f, 0.0f, 0.0f, 0.0f};
            n = mfma16<false>(eight<0, false>(is.x, is.y), sees[0], n);
            n = mfma16<false>(eight<0, false>(is.z, is.w), sees[1], n);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (n[e] > 0.0f) acc[d][e] = __builtin_nanf("");
          }
        }
      }
    }
    // the four waves' results into one
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (kg == 0) {
      s_ml[wave][col][0] = m;
      s_ml[wave][col][1] = l;
    }
#pragma unroll
    for (int d = 0; d < DT; ++d) *(fx_f32x4*)&s_acc[wave][col][d * 16 + kg * 4] = acc[d];
    __syncthreads();
    const int c = (int)threadIdx.x >> 4, part = (int)threadIdx.x & 15;
    if (r0 + c < x.r.rows * G) {
      float top = s_ml[0][c][0], f[W], sum = 0.0f;
#pragma unroll
      for (int w = 1; w < W; ++w) top = fmaxf(top, s_ml[w][c][0]);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        f[w] = s_ml[w][c][0] == -kInf ? 0.0f : __builtin_amdgcn_exp2f(s_ml[w][c][0] - top);
        sum += s_ml[w][c][1] * f[w];
      }
      const int ri = (r0 + c) / G, rg = r0 + c - ri * G;
      const int64_t t = x.r.start + ri;
      const int h = x.head * G + rg;
      const float per = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
      for (int k = 0; k < C; ++k) {
        const int d = (part + 16 * k) * 4;
        if (!EXACT && d >= D) continue;
        float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < W; ++w)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(s_acc[w][c][d + e], f[w], o[e]);
        if (x.splits == 1) {
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] *= per;
          store4((T*)a.out + t * a.out_token + (int64_t)h * D + d, o);
        } else {
          *(float4*)(a.parts.acc + ((int64_t)(x.part + x.split) * FX_KV_ROWS + c) * D + d) = make_float4(o[0], o[1], o[2], o[3]);
        }
      }
      if (part == 0) {
        if (x.splits == 1) {
          a.lse[t * a.q_heads + h] = sum == 0.0f ? -kInf : (top + __builtin_amdgcn_logf(sum)) * kLn2;
        } else {
          float* ml = a.parts.ml + ((int64_t)(x.part + x.split) * FX_KV_ROWS + c) * 2;
          ml[0] = top;
          ml[1] = sum;
        }
      }
    }
    if (x.splits > 1 && x.split == 0 && threadIdx.x == 0)
      a.parts.items[x.item] = FxKvItem{x.request, x.head, x.tile, x.part, x.splits};
  }
  if (a.fill) fill_rest<T>(a);
}

// ---- 32 rows a wave: prompts ----
// Queries of 16 bits.  Bound: the matrix cores and the vector units, which turn scores into weights, side by side.  The waves of a workgroup take 32 rows
// each and share the cached tokens, 64 a step: together they turn a step's codes into 16-bit floats and leave them in LDS.  32 x 32
// products; as above the scores stay where the second product reads them: row 8 g + 4 h + j of K's operand is token
// 16 h + 4 g + j, so a lane holds the 16 tokens of one group.
// Two groups of four waves, one of each on every SIMD, half a step apart: while one is at its products (those of the
// step before with the values, then the next scores) the other one makes its weights and its share of the operands, and a barrier
// changes them over.  Products go first (their waves' priority): what they wait for is longer.  Where a wave's registers are more than
// half of a SIMD's (depths above 128) there is one group, which does one after the other.
// Measured at 4 requests of 511 to 2 047 rows behind up to 6 001 cached tokens, 32 query heads on 8, depth 128, e4m3, bf16 (0.33
// TFLOP): 375 to 384 us, 880 TFLOP/s, of 1 430 that a large library product reaches here.  Without the second group 438 us (before the next
// two steps), with a page a lane and group of 16 tokens (below) in place of one a step 421, without the priority 397.  A step takes about
// 2 300 clocks for either half of its work: 1 024 of the matrix cores and their operands' way from LDS (32 reads of 16 bytes a
// lane), or 1 750 of the vector units (265 instructions, 32 exponentials among them), the longer half.
// Registers that do not fit, a lane: none at depth 64 and, with pages of 64 tokens and more, of bf16 calls at depth 128; f16 on e4m3 4; up to 143 in the
// other forms (pages of 16 and 32, f16 on int8, depths that are not 64, 128 or 256, depth 256): 670 us for bf16 on int8 with pages of 16 where pages of 64 take 383.
// In LDS a key's row of 16-byte pieces is permuted by its token (key_piece), which spreads the 32 rows of an operand over the banks; values
// lie as [group][8 tokens of it][depth][8 tokens].
typedef float fx_f32x16 __attribute__((ext_vector_type(16)));
template <bool F16>
__device__ __forceinline__ fx_f32x16 mfma32(const Frag& a, const Frag& b, fx_f32x16 c) {
  if constexpr (F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(a.h, b.h, c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.b, b.b, c, 0, 0, 0);
}
template <int DP>
__device__ __forceinline__ int key_piece(int token, int piece) {   // where 8 numbers of a key lie in its row
  constexpr int kMask = DP / 8 - 1 < 15 ? DP / 8 - 1 : 15;
  return piece ^ (((token & 3) | ((token >> 2) & 4) | ((token << 1) & 8)) & kMask);
}
// N operands from LDS, four at a time, each four on their way while the four before are used: read(i) gives operand i, use(i, operand)
// takes it; meanwhile() comes while the first four are awaited.  (Left to itself the compiler reads each one right before its product, to save registers.)
template <int N, class Read, class Use, class Meanwhile>
__device__ __forceinline__ void piped(Read read, Use use, Meanwhile meanwhile) {
  Frag f[2][4];
#pragma unroll
  for (int e = 0; e < 4; ++e) f[0][e] = read(e);
  __builtin_amdgcn_sched_barrier(0);
  meanwhile();
#pragma unroll
  for (int b = 0; b < N / 4; ++b) {
    __builtin_amdgcn_sched_barrier(0);
    if (b + 1 < N / 4)
#pragma unroll
      for (int e = 0; e < 4; ++e) f[(b + 1) & 1][e] = read((b + 1) * 4 + e);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int e = 0; e < 4; ++e) use(b * 4 + e, f[b & 1][e]);
  }
}
constexpr int tile_waves(int dp) { return dp <= 128 ? 8 : 4; }   // (fx_kv_tile_rows)

// WIDE: pages of 64 tokens and more, so that a step lies in one page and all about its page is the same in all lanes; smaller pages
// need a page for each group of 16 tokens, and took 421 us instead of 397 in the call above
template <int HELD, int TQ, int DP, bool EXACT, bool WIDE>
__global__ __launch_bounds__(64 * tile_waves(DP), tile_waves(DP) / 4) void fx_kv_tiles(const FxKvAttnArgs a) {
  typedef typename TypeOf<TQ>::type T;
  constexpr int W = tile_waves(DP), kGroups = W / 4, kRows = 32 * W;
  constexpr int NP = TQ == kF16 ? 2 : 1, C = DP / 16, DT = DP / 32;
  constexpr int kShare = DP / 8 / W;   // KB of a step's keys and values that a wave takes
  constexpr int kTile = FX_KV_STEP * DP * 2;
  constexpr bool F16 = TQ == kF16;
  __shared__ __align__(16) uint8_t s_k[2][kTile], s_v[2][kTile];
  __shared__ int s_nan;   // e4m3: there were NaN among the values
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int late = kGroups == 2 ? wave >> 2 : 0;   // the group that is half a step behind
  const int col = lane & 31, half = lane >> 5;
  const int D = EXACT ? DP : a.c.depth, G = a.group, lp = a.c.log_page, pm = (1 << lp) - 1;
  for (int u = (int)blockIdx.x;; u += (int)gridDim.x) {
    Unit x;
    int shared_items = 0;
    const bool live = unit_at<true>(a, kRows, kTileLeast, u, x, &shared_items);
    if (u == 0 && threadIdx.x == 0) *a.parts.n_items = shared_items;
    if (!live) break;
    __syncthreads();   // (LDS is free again)
    if (threadIdx.x == 0) s_nan = 0;
    __syncthreads();
    x.tile = x.r.tiles - 1 - x.tile;   // (the last rows see most: they begin first)
    const int r0 = x.tile * kRows, w0 = r0 + wave * 32, row = w0 + col, n_rows = x.r.rows * G;
    const bool valid = row < n_rows;
    const int i = valid ? row / G : 0, g = valid ? row - i * G : 0;
    const int hi_row = valid ? x.r.len - x.r.rows + i + 1 : 0;
    const int lo_row = a.window > 0 ? max(hi_row - a.window, 0) : 0;
    const FxKvSpan span = scalars(fx_kv_span(x.r, G, a.window, r0, kRows, x.split, x.splits));
    FxKvSpan mine = scalars(fx_kv_span(x.r, G, a.window, min(w0, n_rows - 1), 32, 0, 1));   // of this wave's rows
    if (w0 >= n_rows) mine.high = 0;
    const int from = span.from, n = span.to - span.from;
    Frag q[C];
    {
      const T* src = (const T*)a.q + (int64_t)(x.r.start + i) * a.q_token + (int64_t)(x.head * G + g) * a.q_head;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int d = c * 16 + half * 8;
        Frag* f[1] = {&q[c]};
        load_query<TQ, 1, T>(f, src, d, valid && d < D, a.q_vec != 0);
      }
    }
    fx_f32x16 acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[d][e] = 0.0f;
    float m = -kInf, l = 0.0f;
    const int32_t* table = a.table + (int64_t)x.request * a.table_stride;
    const uint32_t head_at = (uint32_t)x.head * (uint32_t)(pm + 1) * (uint32_t)D;
    // A lane's two groups of a step are `half` and 2 + half.  Their entries are taken as they are, and looked at when they are used, a step later
    constexpr int kP = WIDE ? 1 : 2;   // pages of a lane and step
    auto entry_of = [&](int s, int which) { return table[min(((from + s) * FX_KV_STEP + (WIDE ? 0 : which * 32 + half * 16)) >> lp, a.columns - 1)]; };
    auto page_of = [&](int entry) { return fx_kv_page(WIDE ? __builtin_amdgcn_readfirstlane(entry) : entry, a.c.pages); };
    // A wave's share: blocks of 1 KB, first of the keys, then of the values; block b is 64 bytes of depth for the 16 tokens of a group
    constexpr int kHalf = DP / 16, kPieces = DP / 16, kRowsOf = 1024 / DP, kParts = DP / 64;
    uint4 raw[kShare];
    auto is_keys = [&](int k) { return kShare >= 2 ? k < kShare / 2 : wave < W / 2; };
    auto block_of = [&](int k) { return (k * W + wave) % kHalf; };
    uint32_t key_at[kShare], to_at[kShare][2];   // of a lane: bytes from its group's first key or value, and in LDS
#pragma unroll
    for (int k = 0; k < kShare; ++k) {
      const int group = block_of(k) / kParts, part = block_of(k) % kParts;
      if (is_keys(k)) {
        const int token = part * kRowsOf + lane / kPieces, piece = lane % kPieces, row_at = (group * 16 + token) * DP * 2;
        key_at[k] = token * D + (EXACT || piece * 16 < D ? piece : 0) * 16;   // (queries beyond the depth are 0)
        to_at[k][0] = row_at + key_piece<DP>(group * 16 + token, piece * 2) * 16;
        to_at[k][1] = row_at + key_piece<DP>(group * 16 + token, piece * 2 + 1) * 16;
      } else {
        key_at[k] = (EXACT ? part * 64 + lane : min(part * 64 + lane, D - 1)) * 16;
        to_at[k][0] = (group * 2 * DP + part * 64 + lane) * 16;
        to_at[k][1] = to_at[k][0] + DP * 16;
      }
    }
    // Round r: the keys of step r + 1 and the values of step r, on their way in registers and then to LDS.  (Steps behind the last one
    // are the table's last entries again, and are not used.)
    auto load_round = [&](int r, const int (&key_pages)[kP], const int (&value_pages)[kP]) {
#pragma unroll
      for (int k = 0; k < kShare; ++k) {
        const int group = block_of(k) / kParts;
        const bool keys = is_keys(k);
        uint32_t page;
        if constexpr (WIDE) {
          page = (uint32_t)max(keys ? key_pages[0] : value_pages[0], 0);
        } else {
          const int lane_of = (group & 1) * 32, first = __builtin_amdgcn_readlane(keys ? key_pages[0] : value_pages[0], lane_of),
                    second = __builtin_amdgcn_readlane(keys ? key_pages[1] : value_pages[1], lane_of);
          page = (uint32_t)max(group < 2 ? first : second, 0);
        }
        const uint32_t at = (uint32_t)(((from + r + (keys ? 1 : 0)) * FX_KV_STEP + group * 16) & pm);
        const uint8_t* base = (keys ? a.c.k : a.c.v) + ((uint64_t)page * (keys ? a.c.k_stride : a.c.v_stride) + (head_at + at * (uint32_t)D));
        raw[k] = *(const uint4*)(base + key_at[k]);
      }
    };
    auto write_round = [&](int r) {
#pragma unroll
      for (int k = 0; k < kShare; ++k) {
        if (is_keys(k)) {
          uint8_t* to = s_k[(r + 1) & 1];
          *(Frag*)(to + to_at[k][0]) = eight<HELD, F16>(raw[k].x, raw[k].y);
          *(Frag*)(to + to_at[k][1]) = eight<HELD, F16>(raw[k].z, raw[k].w);
        } else if (r >= 0) {
          if constexpr (HELD == 0) {
            if (__any((nan_codes(raw[k].x) | nan_codes(raw[k].y) | nan_codes(raw[k].z) | nan_codes(raw[k].w)) != 0)) {   // (see below)
              if (lane == 0) s_nan = 1;
              unsigned* w = (unsigned*)&raw[k];
#pragma unroll
              for (int e = 0; e < 4; ++e) w[e] &= ~((nan_codes(w[e]) >> 7) * 0xffu);
            }
          }
          uint8_t* to = s_v[r & 1];
          *(Frag*)(to + to_at[k][0]) = eight<HELD, false>(raw[k].x, raw[k].y);
          *(Frag*)(to + to_at[k][1]) = eight<HELD, false>(raw[k].z, raw[k].w);
        }
      }
    };
    int pg[kP];           // pages of the lane's groups of a step (-1: none), and their scales
    float ks[kP], vs[kP];
#pragma unroll
    for (int t = 0; t < kP; ++t) pg[t] = -1, ks[t] = vs[t] = 1.0f;
    const float *k_scales = a.c.k_scale + x.head, *v_scales = a.c.v_scale + x.head;
    auto scales_of = [&](const int (&pages)[kP]) {
#pragma unroll
      for (int t = 0; t < kP; ++t) {
        pg[t] = pages[t];
        const uint32_t page = (uint32_t)max(pages[t], 0);
        ks[t] = *(const float*)((const char*)k_scales + (uint64_t)page * (a.c.ks_stride * 4));
        vs[t] = *(const float*)((const char*)v_scales + (uint64_t)page * (a.c.vs_stride * 4));
      }
    };
    // pages of steps s and s + 1, and entries of step s + 2, of the products of step s
    int pages0[kP], pages1[kP], entries2[kP];
#pragma unroll
    for (int t = 0; t < kP; ++t) pages0[t] = pages1[t] = entries2[t] = -1;
    if (n > 0) {
#pragma unroll
      for (int t = 0; t < kP; ++t) {
        pages0[t] = page_of(entry_of(0, t));
        pages1[t] = page_of(entry_of(1, t));
        entries2[t] = entry_of(2, t);
      }
      load_round(-1, pages0, pages0);
      write_round(-1);
      if (late) load_round(0, pages1, pages0);
    }
    __syncthreads();
    fx_f32x16 r[2];     // scores of a step
    Frag p[2][2][NP];   // its weights
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) r[t][e] = 0.0f;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int k = 0; k < NP; ++k) p[t >> 1][t & 1][k].u[0] = p[t >> 1][t & 1][k].u[1] = p[t >> 1][t & 1][k].u[2] = p[t >> 1][t & 1][k].u[3] = 0;
    auto sees = [&](int s) { return (from + s) * FX_KV_STEP < mine.high && (from + s + 1) * FX_KV_STEP > mine.low; };   // a row of this wave does
    // The weights of step s - 1 with its values, and the scores of step s.  While its first operands are awaited the next round and the
    // scales of step s are sent for: round s, which this group writes with the weights of step s, and of the late group round s + 1.
    auto products = [&](int s, auto is_late) {
      auto send = [&]() {
        int pages2[kP];
#pragma unroll
        for (int t = 0; t < kP; ++t) pages2[t] = page_of(entries2[t]);
        if constexpr (is_late) load_round(s + 1, pages2, pages1);
        else load_round(s, pages1, pages0);
        scales_of(pages0);
#pragma unroll
        for (int t = 0; t < kP; ++t) {
          pages0[t] = pages1[t];
          pages1[t] = pages2[t];
          entries2[t] = entry_of(s + 3, t);
        }
      };
      if (s > 0 && sees(s - 1)) {
        const uint8_t* vt = s_v[(s - 1) & 1];
        piped<4 * DT>([&](int k) { return *(const Frag*)(vt + (((k / DT / 2 * 2 + half) * 2 + k / DT % 2) * DP + k % DT * 32 + col) * 16); },
                      [&](int k, const Frag& v) {
#pragma unroll
                        for (int e = NP - 1; e >= 0; --e) acc[k % DT] = mfma32<false>(v, p[k / DT / 2][k / DT % 2][e], acc[k % DT]);
                      }, send);
        __builtin_amdgcn_sched_barrier(0);
      } else {
        send();
      }
      if (s < n && sees(s)) {
        const uint8_t* kt = s_k[s & 1];
        int krow = ((col >> 2) & 1) * 16 + (col >> 3) * 4 + (col & 3);
        int kpiece = key_piece<DP>(krow, half) * 16;
        krow *= DP * 2;
        asm volatile("" : "+v"(krow), "+v"(kpiece));   // (16 addresses that are not worth a register each)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) r[t][e] = 0.0f;
        piped<2 * C>([&](int k) { return *(const Frag*)(kt + k % 2 * 32 * DP * 2 + krow + (kpiece ^ (k / 2 * 32))); },
                     [&](int k, const Frag& kf) { r[k % 2] = mfma32<F16>(kf, q[k / 2], r[k % 2]); }, []() {});
      }
    };
    // the weights of step s, and a share of round `round`
    auto weights = [&](int s, int round) {
      const int p0 = pg[0], p1 = pg[kP - 1];
      float cs[2], cv[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        cs[t] = fmaxf(ks[t % kP] * a.scale, kTiny);
        cv[t] = __builtin_amdgcn_fmed3f(vs[t % kP], kTiny, kMost);   // (NaN: kTiny)
      }
      if (round < n) write_round(round);
      __builtin_amdgcn_sched_barrier(0);   // (what is loaded later stays out of registers that are not there)
      if (s >= 0 && sees(s)) {
        const int base = (from + s) * FX_KV_STEP;
        const bool inside = base >= mine.all_low && base + FX_KV_STEP <= mine.all_high && __all(p0 >= 0 && p1 >= 0);
        if (!inside) {
          int hi_row_ = hi_row, lo_row_ = lo_row;
          asm volatile("" : "+v"(hi_row_), "+v"(lo_row_));   // (compared here, not ahead of the branch)
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int t0 = base + (t * 2 + half) * 16;
            const bool ok = (t ? p1 : p0) >= 0;
            if (!ok || mine.high <= t0 || t0 + 16 <= mine.low) cs[t] = cv[t] = 1.0f;   // (what lies there may be anything)
            const int h = ok ? hi_row_ - t0 : 0, b = lo_row_ - t0;
#pragma unroll
            for (int e = 0; e < 16; ++e) r[t][e] = e < h && e >= b ? r[t][e] : -kInf;
          }
        }
        float top[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          top[t] = larger(r[t][0], r[t][1]);
#pragma unroll
          for (int e = 2; e < 16; ++e) top[t] = larger(top[t], r[t][e]);
          top[t] *= cs[t];
        }
        float up = fmaxf(top[0], top[1]);
        if (__any(up > m)) {
          up = fmaxf(up, __shfl_xor(up, 32, 64));
          const float to_m = fmaxf(m, up + kHead);
          const float by = to_m == -kInf ? 1.0f : __builtin_amdgcn_exp2f(m - to_m);
          m = to_m;
          l *= by;
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[d][e] *= by;
        }
        const float sub = m == -kInf ? 0.0f : m;
        float add = 0.0f;
        // weights times the values' scale, a power of two: part of the exponent (see kFoldLeast), and taken out of their sum again
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const float off = __builtin_amdgcn_logf(cv[t]) - sub;
          float w[16], sum[2] = {0.0f, 0.0f};
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(r[t][e], cs[t], off));
            sum[e & 1] += w[e];
          }
          add = __builtin_fmaf(sum[0] + sum[1], __builtin_amdgcn_rcpf(cv[t]), add);
          split8<NP>(p[t][0], w);
          split8<NP>(p[t][1], w + 8);
        }
        if (!__all(folds(cv[0]) && folds(cv[1]))) add = weight_sum(r[0], cs[0], sub) + weight_sum(r[1], cs[1], sub);
        l += add;
      }
    };
    // (a part without steps, the same in all waves: its rows see nothing, and there may be no table to send for)
    if (n <= 0) {
    } else if (!late) {
      for (int s = 0; s <= n; ++s) {
        __builtin_amdgcn_s_setprio(1);
        products(s, std::false_type());
        __builtin_amdgcn_s_setprio(0);
        __syncthreads();
        if (s < n) weights(s, s);
        __syncthreads();
      }
    } else {
      for (int s = 0; s <= n; ++s) {
        weights(s - 1, s);
        __syncthreads();
        __builtin_amdgcn_s_setprio(1);
        products(s, std::true_type());
        __builtin_amdgcn_s_setprio(0);
        __syncthreads();
      }
    }
    if constexpr (HELD == 0) {
      // Values that are NaN were left out of LDS, because 0 * NaN would reach the rows that do not see their tokens: the
      // rows that do get their NaN here, from the cache itself.
      if (__builtin_amdgcn_readfirstlane(s_nan)) {
        for (int s = 0; s < n; ++s)
          for (int t = 0; t < 2; ++t) {
            const int t0 = (from + s) * FX_KV_STEP + (t * 2 + half) * 16;
            const int page = fx_kv_page(table[min(t0 >> lp, a.columns - 1)], a.c.pages), hi = page >= 0 ? hi_row - t0 : 0, lo = lo_row - t0;
            Frag see[2];
#pragma unroll
            for (int w = 0; w < 8; ++w)
              see[w >> 2].u[w & 3] = (2 * w < hi && 2 * w >= lo ? 0x3f80u : 0u) | (2 * w + 1 < hi && 2 * w + 1 >= lo ? 0x3f800000u : 0u);
            const uint8_t* v = a.c.v + (int64_t)max(page, 0) * a.c.v_stride + head_at + (int64_t)((t0 & pm) >> 4) * 16 * D;
#pragma unroll
            for (int d = 0; d < DT; ++d) {
              uint4 is = *(const uint4*)(v + min(d * 32 + col, D - 1) * 16);
              unsigned* w = (unsigned*)&is;
#pragma unroll
              for (int e = 0; e < 4; ++e) w[e] = (nan_codes(w[e]) >> 7) * 0x38u;   // e4m3's 1
              fx_f32x16 y;
#pragma unroll
              for (int e = 0; e < 16; ++e) y[e] = 0.0f;
              y = mfma32<false>(eight<0, false>(is.x, is.y), see[0], y);
              y = mfma32<false>(eight<0, false>(is.z, is.w), see[1], y);
#pragma unroll
              for (int e = 0; e < 16; ++e)
                if (y[e] > 0.0f) acc[d][e] = __builtin_nanf("");
            }
          }
      }
    }
    // (read again from memory rather than kept in scalar registers all along)
    const KernelArgs* z = (const KernelArgs*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(z));
    l += __shfl_xor(l, 32, 64);
    if (valid) {
      const int64_t t = x.r.start + i;
      const int h = x.head * G + g;
      const float per = l == 0.0f ? 0.0f : 1.0f / l;
      const int64_t at = (int64_t)(x.part + x.split) * kRows + wave * 32 + col;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int depth = d * 32 + e * 8 + half * 4;
          if (!EXACT && depth >= D) continue;
          float o[4];
          if (x.splits == 1) {
#pragma unroll
            for (int k = 0; k < 4; ++k) o[k] = acc[d][e * 4 + k] * per;
            store4((T*)z->out + t * z->out_token + (int64_t)h * D + depth, o);
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) o[k] = acc[d][e * 4 + k];
            store4(z->parts.acc + at * D + depth, o);
          }
        }
      if (half == 0) {
        if (x.splits == 1) {
          z->lse[t * z->q_heads + h] = l == 0.0f ? -kInf : (m + __builtin_amdgcn_logf(l)) * kLn2;
        } else {
          z->parts.ml[at * 2] = m;
          z->parts.ml[at * 2 + 1] = l;
        }
      }
    }
    if (x.splits > 1 && x.split == 0 && threadIdx.x == 0)
      z->parts.items[x.item] = FxKvItem{x.request, x.head, x.tile, x.part, x.splits};
  }
  if (a.fill) fill_rest<T>(a);
}

// What several workgroups found for the same rows, added up, of fx_kv_tiles and fx_kv_rows in one launch.  A workgroup takes a row of
// an item: 16 bytes of the result a lane, the parts in turn over the groups of lanes that are left, whose sums meet in LDS in a fixed order.
// Bound: latency, 4.6 us whatever there is to add up.  (Done by the last workgroup to arrive, at counters, it gained nothing: 54 and 56 us
// for the long request above.)
template <class T>
__global__ __launch_bounds__(256) void fx_kv_join(const FxKvAttnArgs a, const FxKvParts tiles, const FxKvParts rows) {
  __shared__ float s_m[64], s_l[64];
  __shared__ __align__(16) float s_o[256 * 4];
  const int64_t of_tiles = tiles.n_items ? (int64_t)*tiles.n_items * tiles.tile_rows : 0, all = of_tiles + (rows.n_items ? (int64_t)*rows.n_items * rows.tile_rows : 0);
  const int D = a.c.depth, G = a.group, lanes = D / 4, groups = 256 / lanes;
  const int group = (int)threadIdx.x / lanes, d = ((int)threadIdx.x - group * lanes) * 4;
  for (int64_t w = blockIdx.x; w < all; w += gridDim.x) {
    const FxKvParts& from = w < of_tiles ? tiles : rows;
    const int tile_rows = from.tile_rows, at_row = (int)(w < of_tiles ? w : w - of_tiles), c = at_row % tile_rows;
    const FxKvItem it = from.items[at_row / tile_rows];
    const int row = it.tile * tile_rows + c;
    const int s = min(max(a.starts[it.request], 0), a.tokens), e = min(max(a.starts[it.request + 1], 0), a.tokens);
    if (row >= (e - s) * G) continue;
    float m = -kInf, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (group < groups) {
#pragma unroll 4
      for (int p = group; p < it.parts; p += groups) {
        const int64_t at = (int64_t)(it.first + p) * tile_rows + c;
        const float2 ml = *(const float2*)(from.ml + at * 2);
        const float4 v = *(const float4*)(from.acc + at * D + d);
        const float now = fmaxf(m, ml.x), f = m == -kInf ? 0.0f : __builtin_amdgcn_exp2f(m - now),
                    g = ml.x == -kInf ? 0.0f : __builtin_amdgcn_exp2f(ml.x - now);
        m = now;
        l = __builtin_fmaf(l, f, ml.y * g);
        o[0] = __builtin_fmaf(o[0], f, v.x * g);
        o[1] = __builtin_fmaf(o[1], f, v.y * g);
        o[2] = __builtin_fmaf(o[2], f, v.z * g);
        o[3] = __builtin_fmaf(o[3], f, v.w * g);
      }
      if (d == 0) {
        s_m[group] = m;
        s_l[group] = l;
      }
      *(float4*)&s_o[(group * lanes) * 4 + d] = make_float4(o[0], o[1], o[2], o[3]);
    }
    __syncthreads();
    if (group == 0) {
      float top = -kInf, sum = 0.0f;
      for (int k = 0; k < groups; ++k) top = fmaxf(top, s_m[k]);
      o[0] = o[1] = o[2] = o[3] = 0.0f;
      for (int k = 0; k < groups; ++k) {
        const float f = s_m[k] == -kInf ? 0.0f : __builtin_amdgcn_exp2f(s_m[k] - top);
        sum = __builtin_fmaf(s_l[k], f, sum);
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = __builtin_fmaf(s_o[(k * lanes) * 4 + d + j], f, o[j]);
      }
      const int64_t t = s + row / G;
      const int h = it.head * G + row % G;
      const float per = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] *= per;
      store4((T*)a.out + t * a.out_token + (int64_t)h * D + d, o);
      if (d == 0) a.lse[t * a.q_heads + h] = sum == 0.0f ? -kInf : (top + __builtin_amdgcn_logf(sum)) * kLn2;
    }
    __syncthreads();
  }
}

struct Kernels {
  const void *rows, *tiles;
};
template <int HELD, int TQ>
Kernels kernels_of(int depth, bool wide) {
  // (fp32 queries: fx_kv_rows alone)
#define FX_KV_TILES(DP, EXACT) (wide ? (const void*)fx_kv_tiles<HELD, TQ == kF32 ? kBf16 : TQ, DP, EXACT, true> : (const void*)fx_kv_tiles<HELD, TQ == kF32 ? kBf16 : TQ, DP, EXACT, false>)
#define FX_KV_PAIR(DP, EXACT) Kernels{(const void*)fx_kv_rows<HELD, TQ, DP, EXACT>, TQ == kF32 ? nullptr : FX_KV_TILES(DP, EXACT)}
  if (depth == 64) return FX_KV_PAIR(64, true);
  if (depth == 128) return FX_KV_PAIR(128, true);
  if (depth == 256) return FX_KV_PAIR(256, true);
  if (depth < 128) return FX_KV_PAIR(128, false);
  return FX_KV_PAIR(256, false);
#undef FX_KV_PAIR
#undef FX_KV_TILES
}
template <int HELD>
Kernels kernels_of(int type, int depth, bool wide) {
  return type == kBf16 ? kernels_of<HELD, kBf16>(depth, wide) : type == kF16 ? kernels_of<HELD, kF16>(depth, wide) : kernels_of<HELD, kF32>(depth, wide);
}
}  // namespace fxkv

fxkv::Kernels fx_kv_kernels_e4m3(int type, int depth, bool wide);
fxkv::Kernels fx_kv_kernels_int8(int type, int depth, bool wide);
