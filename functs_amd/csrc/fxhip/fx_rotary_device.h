// Rotary positions on the device.
//
// A pair (a, b) of a token at position p with frequency f becomes m (a cos pf - b sin pf, b cos pf + a sin pf); backward the
// transposed matrix, which is sin with the other sign.  The angle is a product of 64 bits, less whole quarter turns: positions of
// 2^31 are as exact as small ones (1e-7 of a turn at most).  What is left, up to pi / 4 either way, goes through polynomials in 32 bits
// (least maximum error, found by exchange: sine 0.7 ulp, cosine 1.3 * 2^-24); products are 32 bits, rounded once at the end.
#pragma once
#include "fx_rotary.h"

namespace {
struct Turn { float c, s; };

// (g: frequency times 2 / pi, quarter turns a token)
__device__ __forceinline__ Turn turn_of(double p, double g, float magnitude, bool back) {
  const double t = p * g, q = __builtin_rint(t);
  const float r = (float)((t - q) * 1.57079632679489661923);
  const int k = (int)(q - 4.0 * __builtin_rint(q * 0.25)) & 3;   // -2 .. 2
  const float z = r * r;
  float s = __builtin_fmaf(z, __builtin_fmaf(z, -0.000195169778f, 0.00833217613f), -0.166666552f);
  s = __builtin_fmaf(r, z * s, r);
  float c = __builtin_fmaf(z, __builtin_fmaf(z, 2.44380917e-05f, -0.00138873642f), 0.0416666456f);
  c = __builtin_fmaf(z * z, c, __builtin_fmaf(z, -0.5f, 1.0f));
  Turn w;
  w.c = (k & 1) ? s : c;
  w.s = (k & 1) ? c : s;
  w.c = k == 1 || k == 2 ? -w.c : w.c;
  w.s = (k >= 2) != back ? -w.s : w.s;
  w.c *= magnitude;
  w.s *= magnitude;
  return w;
}
__device__ __forceinline__ double position_of(const FxTurns& t, int64_t i) {
  return t.wide ? (double)((const int64_t*)t.positions)[i] : (double)((const int32_t*)t.positions)[i];
}
__device__ __forceinline__ double quarters_of(const FxTurns& t, int pair) {
  return (t.narrow ? (double)((const float*)t.frequencies)[pair] : ((const double*)t.frequencies)[pair]) * 0.63661977236758134308;
}
__device__ __forceinline__ void turn_pair(float& a, float& b, const Turn& w) {
  const float u = __builtin_fmaf(a, w.c, -(b * w.s)), v = __builtin_fmaf(b, w.c, a * w.s);
  a = u;
  b = v;
}

__device__ __forceinline__ unsigned divided(unsigned n, unsigned d, unsigned magic) { return magic ? __umulhi(n, magic) : n / d; }

// N numbers from any address (rows of odd sizes begin anywhere), in whole words: halves would take a register each
template <class T, int N>
struct Some {
  unsigned u[N * sizeof(T) / 4];
  __device__ __forceinline__ void load(const T* p) { __builtin_memcpy(u, p, sizeof u); }
  __device__ __forceinline__ void store(T* p) const { __builtin_memcpy(p, u, sizeof u); }
  __device__ __forceinline__ float at(int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(u[i]);
    else return (float)__builtin_bit_cast(T, (unsigned short)(i % 2 ? u[i / 2] >> 16 : u[i / 2]));
  }
  __device__ __forceinline__ void set(int i, float a, float b) {   // numbers i and i + 1, i even
    if constexpr (sizeof(T) == 4) u[i] = __float_as_uint(a), u[i + 1] = __float_as_uint(b);
    else u[i / 2] = __builtin_bit_cast(unsigned short, (T)a) | (unsigned)__builtin_bit_cast(unsigned short, (T)b) << 16;
  }
};
template <class T>
struct Some<T, 1> {
  T e;
  __device__ __forceinline__ void load(const T* p) { e = *p; }
  __device__ __forceinline__ void store(T* p) const { *p = e; }
};

// A workgroup's share of the rows.  A unit is PV pairs of a head, or 2 PV of the columns that do not turn, in two halves as well: two loads and two stores of
// 16 bytes a lane where PV is 8 (16-bit types) or 4.  Where the units do not fit, the last one begins earlier and does some numbers
// again.  Angles are computed once for all heads and kept in LDS, behind the first loads.  Both kinds of units go one way, but for the turn itself (10 565 tokens of 32 heads
// of 128 columns, half of them turning, fp16: 32 us; 37 with loads and stores of their own).
template <class T, int PV, bool INTER>
__device__ __forceinline__ void rotary_rows(const FxRotary& a, int block, int slice, Turn* s_turn) {
  constexpr int kThreadsHere = 256, kUnits = 2;
  const int tid = (int)threadIdx.x, pairs = a.turns.pairs, rest = a.depth - 2 * pairs, half = (rest + 1) / 2, total = a.batch * a.tokens;
  const int g0 = block * a.per, n = min(a.per, total - g0), row = a.units * a.heads, all = n * row;
  T* const y = (T*)a.y;
  const auto apart = [&](int angle) { return INTER ? PV : angle >= 0 ? pairs : rest - half; };   // a unit's halves
  bool first = true;
  for (int base = slice * kThreadsHere; base < all; base += a.slices * kThreadsHere * kUnits) {
    Some<T, PV> lo[kUnits], hi[kUnits];
    int64_t to[kUnits];              // the head's place in y
    int at[kUnits], angle[kUnits];   // at: first column; angle: place of the first pair's, -1: columns that do not turn, -2: few of them, -3: nothing
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
      const int i = base + k * a.slices * kThreadsHere + tid;
      angle[k] = -3;
      if (i >= all) continue;
      const int j = (int)divided((unsigned)i, (unsigned)row, a.magic_token), in_row = i - j * row;
      const int h = (int)divided((unsigned)in_row, (unsigned)a.units, a.magic_head), u = in_row - h * a.units;
      const int g = g0 + j, b = a.batch == 1 ? 0 : g / a.tokens, t = g - b * a.tokens;
      const T* x = (const T*)a.x + (int64_t)b * a.x_batch + (int64_t)t * a.x_token + (int64_t)h * a.x_head;
      to[k] = (int64_t)b * a.y_batch + (int64_t)t * a.y_token + (int64_t)h * a.y_head;
      const bool turns = u < a.turning;
      if (turns || rest >= 2 * PV) {
        if constexpr (INTER) {
          const int p = turns ? min(u * PV, pairs - PV) : pairs;
          at[k] = turns ? 2 * p : 2 * pairs + min((u - a.turning) * 2 * PV, rest - 2 * PV);
          angle[k] = turns ? j * pairs + p : -1;
        } else {
          const int p = min((turns ? u : u - a.turning) * PV, (turns ? pairs : half) - PV);
          at[k] = turns ? p : 2 * pairs + p;
          angle[k] = turns ? j * pairs + p : -1;
        }
        lo[k].load(x + at[k]);
        hi[k].load(x + at[k] + apart(angle[k]));
      } else {
        angle[k] = -2;
        for (int c = 2 * pairs; c < a.depth; ++c) y[to[k] + c] = x[c];
      }
    }
    if (first) {
      first = false;
      for (int i = tid; i < n * pairs; i += kThreadsHere) {
        const int j = (int)divided((unsigned)i, (unsigned)pairs, a.magic_pair), g = g0 + j, b = a.batch == 1 ? 0 : g / a.tokens;
        s_turn[i] = turn_of(position_of(a.turns, (int64_t)b * a.position_batch + (g - b * a.tokens)), quarters_of(a.turns, i - j * pairs), a.turns.magnitude, a.turns.back != 0);
      }
      __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
      if (angle[k] < -1) continue;
      if (angle[k] >= 0) {
        const Turn* const w = s_turn + angle[k];
        if constexpr (PV == 1) {
          float u = (float)lo[k].e, v = (float)hi[k].e;
          turn_pair(u, v, w[0]);
          lo[k].e = (T)u;
          hi[k].e = (T)v;
        } else {
#pragma unroll
          for (int i = 0; i < PV; i += 2) {
            float a0 = lo[k].at(i), a1 = lo[k].at(i + 1), b0 = hi[k].at(i), b1 = hi[k].at(i + 1);
            if constexpr (INTER) {
              turn_pair(a0, a1, w[i / 2]);
              turn_pair(b0, b1, w[(PV + i) / 2]);
            } else {
              turn_pair(a0, b0, w[i]);
              turn_pair(a1, b1, w[i + 1]);
            }
            lo[k].set(i, a0, a1);
            hi[k].set(i, b0, b1);
          }
        }
      }
      lo[k].store(y + to[k] + at[k]);
      hi[k].store(y + to[k] + at[k] + apart(angle[k]));
    }
  }
}
}  // namespace
