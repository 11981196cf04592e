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
//   weights  bf16, f16 results: two bf16 (16 bits);  fp32 results: three
#pragma once
#include "fx_kv.h"
#include "fx_kv_device.h"

typedef __bf16 fx_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 fx_bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 fx_f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 fx_f16x2 __attribute__((ext_vector_type(2)));
typedef float fx_f32x4 __attribute__((ext_vector_type(4)));

namespace fxkv {
constexpr float kInf = __builtin_inff(), kLn2 = 0.693147180559945309f;
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
__device__ __forceinline__ FxKvRequest request_at(const FxKvAttnArgs& a, int b, int tile_rows) {
  if (b >= a.requests) return FxKvRequest{0, 0, 0, 0, 0};
  return fx_kv_request(a.starts[b], a.starts[b + 1], a.lens[b], a.tokens, a.columns << a.c.log_page, a.group, a.window, tile_rows);
}
template <int THREADS>
__device__ __forceinline__ int64_t sum_before(int64_t v, int64_t* scratch, int64_t* total) {
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  int64_t s = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t o = (int64_t)__shfl_up((unsigned long long)s, (unsigned)d, 64);
    if (lane >= d) s += o;
  }
  if (lane == 63) scratch[wave] = s;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    if (w < wave) before += scratch[w];
    all += scratch[w];
  }
  __syncthreads();
  *total = all;
  return before + s - v;
}
template <int THREADS>
__device__ int chunk_of(const FxKvAttnArgs& a, int tile_rows, int least, int64_t* scratch) {
  int64_t work = 0, all = 0;
  for (int b0 = 0; b0 < a.requests; b0 += THREADS) {
    const FxKvRequest r = request_at(a, b0 + (int)threadIdx.x, tile_rows);
    work += (int64_t)r.tiles * r.steps;
  }
  sum_before<THREADS>(work, scratch, &all);
  return fx_kv_chunk(all * a.c.heads, least);
}
// Unit u of the call, or false behind the last one; *shared_items: how many items several workgroups share
template <int THREADS>
__device__ bool unit_at(const FxKvAttnArgs& a, int tile_rows, int chunk, int u, Unit& out, Unit* s_unit, int64_t* scratch, int* shared_items) {
  int64_t carry_units = 0, carry_parts = 0;   // carry_parts: items << 32 | parts
  if (threadIdx.x == 0) s_unit->r.rows = 0;
  for (int b0 = 0; b0 < a.requests; b0 += THREADS) {
    const int b = b0 + (int)threadIdx.x;
    const FxKvRequest r = request_at(a, b, tile_rows);
    const int splits = fx_kv_parts(r.steps, chunk);
    const int64_t items = (int64_t)r.tiles * a.c.heads, units = items * splits;
    int64_t all_units, all_parts;
    const int64_t before = carry_units + sum_before<THREADS>(units, scratch, &all_units);
    const int64_t parts = carry_parts + sum_before<THREADS>(splits > 1 ? (items << 32) + units : 0, scratch, &all_parts);
    if (u >= before && u < before + units) {
      const int i = (int)(u - before), item = i / splits;
      Unit x;
      x.r = r;
      x.request = b;
      x.head = item % a.c.heads;
      x.tile = item / a.c.heads;
      x.split = i - item * splits;
      x.splits = splits;
      x.part = (int)(parts & 0xffffffff) + item * splits;
      x.item = (int)(parts >> 32) + item;
      *s_unit = x;
    }
    carry_units += all_units;
    carry_parts += all_parts;
  }
  __syncthreads();
  out = *s_unit;
  *shared_items = (int)(carry_parts >> 32);
  return out.r.rows > 0;
}

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

// ---- 16 rows a tile: single tokens and few rows ----
// Bound: HBM, each key and value is read once by one wave, straight into the registers of its operand; 64 tokens a
// step, the four waves of a workgroup in turn.  The loads of the next step's keys are under way during the softmax and the second
// product, those of the values during the first.
template <int HELD, int TQ, int DP, bool EXACT>
__global__ __launch_bounds__(256) void fx_kv_rows(const FxKvAttnArgs a) {
  typedef typename TypeOf<TQ>::type T;
  constexpr int W = 4, NQ = TQ == kF32 ? 3 : 1, NP = TQ == kF32 ? 3 : 2, C = DP / 64, DT = DP / 16, LD = DP + 4;
  constexpr bool F16 = TQ == kF16;
  __shared__ __align__(16) float s_acc[W][FX_KV_ROWS][LD];
  __shared__ float s_ml[W][FX_KV_ROWS][2];
  __shared__ int64_t s_scan[W];
  __shared__ Unit s_unit;
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  const int col = lane & 15, kg = lane >> 4;
  const int D = EXACT ? DP : a.c.depth, G = a.group, lp = a.c.log_page, pm = (1 << lp) - 1;
  if (a.fill) fill_rest<T>(a);
  const int chunk = chunk_of<256>(a, FX_KV_ROWS, W, s_scan);
  for (int u = (int)blockIdx.x;; u += (int)gridDim.x) {
    Unit x;
    int shared_items;
    if (u != (int)blockIdx.x) __syncthreads();
    const bool live = unit_at<256>(a, FX_KV_ROWS, chunk, u, x, &s_unit, s_scan, &shared_items);
    if (u == 0 && threadIdx.x == 0) *a.n_items = shared_items;
    if (!live) return;
    // rows
    const int r0 = x.tile * FX_KV_ROWS, row = r0 + col;
    const bool valid = row < x.r.rows * G;
    const int i = valid ? row / G : 0, g = valid ? row - i * G : 0;
    const int hi_row = valid ? x.r.len - x.r.rows + i + 1 : 0;                             // tokens [lo_row, hi_row)
    const int lo_row = a.window > 0 ? max(hi_row - a.window, 0) : 0;
    const FxKvSpan span = fx_kv_span(x.r, G, a.window, r0, FX_KV_ROWS, x.split, x.splits);
    const int from = span.from, to = span.to;
    // queries: lane kg holds depths 64 c + 16 kg ... + 15 of its row
    Frag q[NQ][2 * C];
    {
      const T* src = (const T*)a.q + (int64_t)(x.r.start + i) * a.q_token + (int64_t)(x.head * G + g) * a.q_head;
#pragma unroll
      for (int c = 0; c < 2 * C; ++c) {
        const int d = (c >> 1) * 64 + kg * 16 + (c & 1) * 8;
        const bool in = valid && d < D;
        if constexpr (TQ == kF32) {
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = in ? src[d + e] : 0.0f;
          Frag f[NQ];
          split8<NQ>(f, v);
#pragma unroll
          for (int k = 0; k < NQ; ++k) q[k][c] = f[k];
        } else {
          T v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = in ? src[d + e] : (T)0.0f;
          q[0][c] = *(const Frag*)v;
        }
      }
    }
    fx_f32x4 acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d] = fx_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -kInf, l = 0.0f;
    const int32_t* table = a.table + (int64_t)x.request * a.table_stride;
    const int k_group = (col >> 2) * 16, k_row = col & 3;
    const int64_t head_at = (int64_t)x.head * (pm + 1) * D;
    auto page_of = [&](int token) { return fx_kv_page(table[min(token >> lp, a.columns - 1)], a.c.pages); };   // -1: none
    uint4 kr[4][C];
    auto load_keys = [&](int step, int page) {
      const int at = (step * FX_KV_STEP + k_group) & pm;
      const uint8_t* p = a.c.k + (int64_t)page * a.c.k_stride + head_at + (int64_t)(at + k_row) * D + kg * 16;
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < C; ++c)
          if (EXACT || c * 64 + kg * 16 < D) kr[r][c] = *(const uint4*)(p + r * 4 * D + c * 64);
          else kr[r][c] = make_uint4(0, 0, 0, 0);
    };
        int step = from + wave, pk = 0, pv = 0;
    if (step < to) {
      pk = page_of(step * FX_KV_STEP + k_group);
      pv = page_of(step * FX_KV_STEP + kg * 16);
      load_keys(step, max(pk, 0));
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
        for (int d = 0; d < DT; ++d)
          if (EXACT || d * 16 < D) vr[d] = *(const uint4*)(p + d * 256);
      }
      const bool more = step + W < to;
      if (more) {
        pk = page_of(base + W * FX_KV_STEP + k_group);
        pv = page_of(base + W * FX_KV_STEP + kg * 16);
      }
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
      if (more) load_keys(step + W, max(pk, 0));
      float cs = ks * a.scale, vscale = vs;
      const bool inside = base >= span.all_low && base + FX_KV_STEP <= span.all_high && __all(ok);
      if (!inside) {
        const int t0 = base + kg * 16;
        const int n_any = ok ? min(max(span.high - t0, 0), 16) : 0;   // tokens of this group that some row may see
        if (n_any == 0) cs = vscale = 1.0f;                      // (what lies there may be anything)
        const int h = ok ? hi_row - t0 : 0, b = lo_row - t0;
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = e < h && e >= b ? s[e] : -kInf;
        const int skip = min(max(span.low - t0, 0), 16);
        unsigned keep[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {   // bytes of tokens that some row may see
          const int up = min(max(n_any - 4 * w, 0), 4), down = min(max(skip - 4 * w, 0), 4);
          const unsigned upper = up == 4 ? ~0u : (1u << (8 * up)) - 1, lower = down == 4 ? ~0u : (1u << (8 * down)) - 1;
          keep[w] = upper & ~lower;
        }
        unsigned nans = 0;
#pragma unroll
        for (int d = 0; d < DT; ++d)
          if (EXACT || d * 16 < D) {
            unsigned* v = (unsigned*)&vr[d];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              v[w] &= keep[w];
              if constexpr (HELD == 0) nans |= ((v[w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
            }
          }
        if constexpr (HELD == 0) {
          // A value that is NaN must not reach the rows that do not see its token, and 0 * NaN would: such codes
          // are taken out, and the rows that see them get their NaN here.
          if (__any(nans != 0)) {
            Frag sees[2];
            float y[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) y[e] = e < h && e >= b ? 1.0f : 0.0f;
            Frag one[1];
            split8<1>(one, y);
            sees[0] = one[0];
            split8<1>(one, y + 8);
            sees[1] = one[0];
#pragma unroll
            for (int d = 0; d < DT; ++d)
              if (EXACT || d * 16 < D) {
                unsigned* v = (unsigned*)&vr[d];
                unsigned is[4];
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                  const unsigned n = (((v[w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
                  is[w] = n * 0x38u;   // e4m3's 1
                  v[w] &= ~(n * 0xffu);
                }
                fx_f32x4 t = {0.0f, 0.0f, 0.0f, 0.0f};
                t = mfma16<false>(eight<0, false>(is[0], is[1]), sees[0], t);
                t = mfma16<false>(eight<0, false>(is[2], is[3]), sees[1], t);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (t[e] > 0.0f) acc[d][e] = __builtin_nanf("");
              }
          }
        }
      }
      // running maximum: raised only where a score is 8 or more above it (weights stay below 2^8)
      float top = s[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) top = fmaxf(top, s[e]);
      top *= cs;
      if (__any(top > m + 8.0f || (m == -kInf && top > -kInf))) {
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float now = fmaxf(m, top);
        const float by = now == -kInf ? 1.0f : __builtin_amdgcn_exp2f(m - now);
        m = now;
        l *= by;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[d][e] *= by;
      }
      const float sub = m == -kInf ? 0.0f : m;
      Frag p[2][NP];
      float w[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], cs, -sub));
        l += w[e];
        w[e] *= vscale;
      }
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
          *(float4*)(a.part_acc + ((int64_t)(x.part + x.split) * FX_KV_ROWS + c) * D + d) = make_float4(o[0], o[1], o[2], o[3]);
        }
      }
      if (part == 0) {
        if (x.splits == 1) {
          a.lse[t * a.q_heads + h] = sum == 0.0f ? -kInf : (top + __builtin_amdgcn_logf(sum)) * kLn2;
        } else {
          float* ml = a.part_ml + ((int64_t)(x.part + x.split) * FX_KV_ROWS + c) * 2;
          ml[0] = top;
          ml[1] = sum;
        }
      }
    }
    if (x.splits > 1 && x.split == 0 && threadIdx.x == 0)
      a.items[x.item] = FxKvItem{x.request, x.head, x.tile, x.part, x.splits};
  }
}

// What several workgroups found for the same rows, added up in their order.  A workgroup takes a row of an item, a wave the
// depths of it.
template <class T>
__global__ __launch_bounds__(256) void fx_kv_join(const FxKvAttnArgs a, int tile_rows) {
  const int items = *a.n_items;
  const int D = a.c.depth, G = a.group, d = (int)threadIdx.x;
  for (int64_t w = blockIdx.x; w < (int64_t)items * tile_rows; w += gridDim.x) {
    const FxKvItem it = a.items[w / tile_rows];
    const int c = (int)(w % tile_rows), row = it.tile * tile_rows + c;
    const int s = min(max(a.starts[it.request], 0), a.tokens), e = min(max(a.starts[it.request + 1], 0), a.tokens);
    if (row >= (e - s) * G) continue;
    float top = -kInf;
    for (int p = 0; p < it.parts; ++p) top = fmaxf(top, a.part_ml[((int64_t)(it.first + p) * tile_rows + c) * 2]);
    float sum = 0.0f, o = 0.0f;
    for (int p = 0; p < it.parts; ++p) {
      const int64_t at = (int64_t)(it.first + p) * tile_rows + c;
      const float m = a.part_ml[at * 2], f = m == -kInf ? 0.0f : __builtin_amdgcn_exp2f(m - top);
      sum = __builtin_fmaf(a.part_ml[at * 2 + 1], f, sum);
      if (d < D) o = __builtin_fmaf(a.part_acc[at * D + d], f, o);
    }
    const int64_t t = s + row / G;
    const int h = it.head * G + row % G;
    if (d < D) ((T*)a.out)[t * a.out_token + (int64_t)h * D + d] = (T)(sum == 0.0f ? 0.0f : o / sum);
    if (d == 0) a.lse[t * a.q_heads + h] = sum == 0.0f ? -kInf : (top + __builtin_amdgcn_logf(sum)) * kLn2;
  }
}

template <int HELD, int TQ>
const void* rows_kernel(int depth) {
  if (depth == 64) return (const void*)fx_kv_rows<HELD, TQ, 64, true>;
  if (depth == 128) return (const void*)fx_kv_rows<HELD, TQ, 128, true>;
  if (depth == 256) return (const void*)fx_kv_rows<HELD, TQ, 256, true>;
  if (depth < 128) return (const void*)fx_kv_rows<HELD, TQ, 128, false>;
  return (const void*)fx_kv_rows<HELD, TQ, 256, false>;
}
template <int HELD>
const void* rows_kernel(int type, int depth) {
  return type == kBf16 ? rows_kernel<HELD, kBf16>(depth) : type == kF16 ? rows_kernel<HELD, kF16>(depth) : rows_kernel<HELD, kF32>(depth);
}
}  // namespace fxkv

const void* fx_kv_rows_kernel_e4m3(int type, int depth);
const void* fx_kv_rows_kernel_int8(int type, int depth);
hipError_t fx_launch_kv_attention(const FxKvAttnArgs& a, int held, int type, int64_t grid, int64_t join_grid, hipStream_t stream);
