// How rows of keys and values become codes of the paged cache: the kernel of fx_kv_store (fx_kv.hip) and of
// fx_kv_append (fx_kv_append.hip), whose keys turn on the way.
#pragma once
#include <algorithm>
#include <type_traits>

#include "fx_kv.h"
#include "fx_kv_device.h"
#include "fx_rotary_device.h"

namespace {
constexpr int kThreads = 256;

// ---- fx_kv_store ----
// Bound: HBM (2 or 4 bytes read and 1 written for each number); single tokens: latency.
// A run is the neighbours in `slots` that lie in one page; a workgroup takes the keys or the values of one head of the runs that
// begin in its chunk of tokens, so a page's scale and codes have one writer and nothing is locked.  The run's numbers are read, their
// largest magnitude gives the scale, then they become codes.  Of a run of more than 16 tokens each of the four waves takes a
// quarter, which stays in registers between the two (beyond those it is read a second time, from the caches), and the
// magnitudes meet in LDS; shorter ones, and those in no order, are the waves' in turn.  Keys: 8 numbers of a token a lane.  Values: 2 columns
// of a group of 16 tokens a lane, which are 32 neighbouring bytes of the cache.
// Measured: 19 000 tokens of 9 prompts, 8 heads of 128, pages of 64, fp16 to int8: 36 us, 3.3 TB/s (a large copy: 5.4); whole runs a wave: 46.
// 96 single tokens: 8 us, most of it the way to slots, rows and codes, one after the other.
// Magnitudes are compared as the integers that their bits are.  Where the largest one is finite and below the largest scale, no number
// needs to be held to the range of the codes or looked at for NaN (PLAIN).
constexpr int kStoreWaves = kThreads / 64;
typedef unsigned short fx_u16x2 __attribute__((ext_vector_type(2)));

// 2 and 8 numbers as they are loaded; the magnitudes' bits (16-bit types: two to a word)
template <class T> struct Pack {   // 16 bits
  typedef unsigned two;
  typedef uint4 eight;
  static __device__ __forceinline__ unsigned larger(unsigned m, unsigned w) {
    return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(fx_u16x2, m), __builtin_bit_cast(fx_u16x2, w & 0x7fff7fffu)));
  }
  static __device__ __forceinline__ unsigned see(unsigned m, two w) { return larger(m, w); }
  static __device__ __forceinline__ unsigned see(unsigned m, const eight& w) { return larger(larger(larger(larger(m, w.x), w.y), w.z), w.w); }
  static __device__ __forceinline__ float value(unsigned m) {   // of the larger half; infinity or NaN where there is one
    const unsigned short u = (unsigned short)max(m & 0xffffu, m >> 16);
    return (float)__builtin_bit_cast(T, u);
  }
};
template <> struct Pack<float> {
  typedef uint2 two;
  typedef struct { uint4 a, b; } eight;
  static __device__ __forceinline__ unsigned larger(unsigned m, unsigned w) { return max(m, w & 0x7fffffffu); }
  static __device__ __forceinline__ unsigned see(unsigned m, const two& w) { return larger(larger(m, w.x), w.y); }
  static __device__ __forceinline__ unsigned see(unsigned m, const eight& w) {
    m = larger(larger(larger(larger(m, w.a.x), w.a.y), w.a.z), w.a.w);
    return larger(larger(larger(larger(m, w.b.x), w.b.y), w.b.z), w.b.w);
  }
  static __device__ __forceinline__ float value(unsigned m) { return __uint_as_float(m); }
};
template <class T, int N, class P>
__device__ __forceinline__ P load_numbers(const T* p, bool vec) {
  union { P u; T e[N]; } w;
  if (vec) {
    w.u = *(const P*)p;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) w.e[i] = p[i];
  }
  return w.u;
}
template <class T, int N, class P>
__device__ __forceinline__ void floats(float (&x)[N], const P& p) {
  union { P u; T e[N]; } w;
  w.u = p;
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = (float)w.e[i];
}
// the largest of a wave's words, each half by itself where HALVES
template <bool HALVES>
__device__ __forceinline__ unsigned wave_largest(unsigned m) {
  auto larger = [](unsigned a, unsigned b) {
    return HALVES ? __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(fx_u16x2, a), __builtin_bit_cast(fx_u16x2, b))) : max(a, b);
  };
  m = larger(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x111, 0xf, 0xf, false));   // row_shr: 1, 2, 4, 8
  m = larger(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x112, 0xf, 0xf, false));
  m = larger(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x114, 0xf, 0xf, false));
  m = larger(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x118, 0xf, 0xf, false));
  m = larger(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x142, 0xa, 0xf, false));   // row_bcast: 15, 31
  m = larger(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x143, 0xc, 0xf, false));
  return (unsigned)__builtin_amdgcn_readlane((int)m, 63);
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
// codes of x * inv
template <int HELD, bool PLAIN>
__device__ __forceinline__ unsigned codes4(const float* x, float inv) {
  float y[4];
  if constexpr (PLAIN && HELD == 1) {   // the sum with 1.5 * 2^23 rounds to whole numbers: its last byte is the code
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = __builtin_fmaf(x[i], inv, 12582912.0f);
    return __builtin_amdgcn_perm(__float_as_uint(y[1]), __float_as_uint(y[0]), 0x0c0c0400u) |
           __builtin_amdgcn_perm(__float_as_uint(y[3]), __float_as_uint(y[2]), 0x04000c0cu);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = x[i] * inv;
    if constexpr (PLAIN) {
      const int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
      return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
    }
    return encode4<HELD>(y);
  }
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

__device__ __forceinline__ int64_t lane_of(int64_t v, int lane) {   // in scalar registers
  return ((int64_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32) | (unsigned)__builtin_amdgcn_readlane((int)v, lane);
}
// One run, or a wave's share of it: rows [0, n) of `rows` go to offsets o0 on of a page (straight), or to those that `slots` says.
// TURN: keys turn by their tokens' positions ahead of all else, and are fp32 from then on.  A lane has 8 pairs of a row (16 of its columns, or 16
// that do not turn), forms their angles by itself and keeps the turned numbers of two iterations; where the units of a row do not fit, the last one
// begins earlier and does some columns again.  INTER: pairs are neighbours.  Angles are formed for each head anew: 2 us of the chip's vector units for
// 10 565 tokens, 8 heads and 32 pairs, of 59 (fx_kv_append with its queries).  Slower there: 8 columns a lane, angles shared by a wave in LDS and
// numbers in registers 82 us, numbers in LDS as well 88; 16 columns a lane as numbers of 16 bits, each in a register of its own, three waves a SIMD 69, four 76.
template <int HELD, class T, bool VALUES, bool TURN = false, bool INTER = false>
struct StoreRun {
  static_assert(!(VALUES && TURN), "values do not turn");
  typedef std::conditional_t<TURN, float, T> N;   // what is kept of a number
  typedef typename Pack<N>::eight P8;
  typedef typename Pack<T>::two P2;
  const T* rows;
  int64_t stride;
  int n, o0, D, lane;
  uint8_t* codes;
  bool vec;
  const FxTurns* turns;    // TURN: what turns, and the place of row 0's position
  int64_t token;
  const double* quarters;  // (LDS) of all pairs
  int pair0;               // the lane's first
  int lo, hi, n_lo, n_hi;  // the lane's columns: n_lo from lo on, n_hi from hi on, 8 each but at the ends
  bool turning;
  // lane -> (row of an iteration, eight of its depth), or (group of an iteration, pair of columns)
  int width, abreast, sub, at, blocks, g0, count, iterations;

  __device__ __forceinline__ void shape() {
    width = VALUES ? D >> 1 : D >> 3;
    if constexpr (TURN) {
      const int pairs = turns->pairs, rest = D - 2 * pairs;
      width = ((pairs + 7) >> 3) + ((rest + 15) >> 4);
    }
    abreast = width >= 64 ? 1 : 64 / width;
    sub = lane / width;
    at = lane - sub * width;
    blocks = width > 64 ? (width + 63) >> 6 : 1;   // (values of depth above 128)
    g0 = o0 >> 4;
    count = VALUES ? ((o0 + n + 15) >> 4) - g0 : n;
    iterations = (count + abreast - 1) / abreast * blocks;
    if constexpr (TURN) {
      const int pairs = turns->pairs, rest = D - 2 * pairs, units = (pairs + 7) >> 3;
      turning = at < units;
      if (turning) {
        const int first = max(min(at * 8, pairs - 8), 0), some = min(pairs, 8);
        lo = INTER ? 2 * first : first;
        hi = INTER ? lo + 8 : first + pairs;
        n_lo = INTER ? min(2 * some, 8) : some;
        n_hi = INTER ? 2 * some - n_lo : some;
        pair0 = first;
      } else {
        const int some = min(rest, 16);
        lo = 2 * pairs + max(min((at - units) * 16, rest - 16), 0);
        hi = lo + 8;
        n_lo = min(some, 8);
        n_hi = some - n_lo;
        pair0 = 0;
      }
    }
  }
  // column d of row j, as it is stored
  __device__ __forceinline__ float number(int j, int d) const {
    const T* p = rows + (int64_t)j * stride;
    if constexpr (TURN) {
      const int pairs = turns->pairs;
      if (d < 2 * pairs) {
        const bool upper = turns->interleaved ? (d & 1) != 0 : d >= pairs;
        const int step = turns->interleaved ? 1 : pairs, pair = turns->interleaved ? d >> 1 : upper ? d - pairs : d;
        float a = (float)p[upper ? d - step : d], b = (float)p[upper ? d : d + step];
        turn_pair(a, b, turn_of(position_of(*turns, token + j), quarters_of(*turns, pair), turns->magnitude, false));
        return upper ? b : a;
      }
    }
    return (float)p[d];
  }
  // rows beyond the run: its last or first one again, which is in the maximum anyway and not written
  __device__ __forceinline__ typename Pack<T>::eight load_eight(int k) const {
    typedef typename Pack<T>::eight P;
    const T* p = rows + at * 8;
    if ((k + 1) * abreast <= n) return load_numbers<T, 8, P>(p + (int64_t)(k * abreast) * stride + (int64_t)sub * stride, vec);
    return load_numbers<T, 8, P>(p + (int64_t)min(k * abreast + sub, n - 1) * stride, vec);
  }
  // TURN: the lane's columns of a row as they are loaded
  struct Raw { unsigned u[sizeof(T) * 4]; };   // (whole words: halves would take a register each)
  __device__ __forceinline__ int row_of(int k) const { return min(k * abreast + sub, n - 1); }
  __device__ __forceinline__ void load_sixteen(Raw& raw, int k) const {
    const T* p = rows + (int64_t)row_of(k) * stride;
    if (n_lo + n_hi == 16) {
      __builtin_memcpy(raw.u, p + lo, sizeof raw.u / 2);
      __builtin_memcpy(raw.u + sizeof(T) * 2, p + hi, sizeof raw.u / 2);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const bool there = i < 8 ? i < n_lo : i - 8 < n_hi;
        const T* from = p + (i < 8 ? lo + i : hi + i - 8);
        if constexpr (sizeof(T) == 4) {
          raw.u[i] = there ? __builtin_bit_cast(unsigned, *from) : 0u;
        } else {
          const unsigned w = there ? (unsigned)__builtin_bit_cast(unsigned short, *from) : 0u;
          raw.u[i / 2] = i % 2 == 0 ? w : raw.u[i / 2] | w << 16;
        }
      }
    }
  }
  // x: the first of each pair, then the others (of columns that do not turn: in the same order)
  __device__ __forceinline__ void turn_sixteen(float (&x)[16], Raw& raw, double position) const {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) * 4; ++i) asm volatile("" : "+v"(raw.u[i]));
    float u[8], v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (sizeof(T) == 4) {
        u[i] = __uint_as_float(raw.u[i]);
        v[i] = __uint_as_float(raw.u[8 + i]);
      } else {
        u[i] = (float)__builtin_bit_cast(T, (unsigned short)(raw.u[i / 2] >> (i % 2 * 16)));
        v[i] = (float)__builtin_bit_cast(T, (unsigned short)(raw.u[4 + i / 2] >> (i % 2 * 16)));
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = INTER ? (i < 4 ? u[2 * i % 8] : v[2 * i % 8]) : u[i];
      x[8 + i] = INTER ? (i < 4 ? u[(2 * i + 1) % 8] : v[(2 * i + 1) % 8]) : v[i];
    }
    if (turning) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        turn_pair(x[i], x[8 + i], turn_of(position, quarters[pair0 + i], turns->magnitude, false));
        if (i % 2 == 1) __builtin_amdgcn_sched_barrier(0);   // (eight angles at once take 40 registers more)
      }
    }
  }
  template <bool PLAIN>
  __device__ __forceinline__ void write_sixteen(int k, const float (&x)[16], float inv) const {
    const int j = k * abreast + sub;
    if (j >= n || sub >= abreast) return;
    float y[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      y[INTER ? 2 * i : i] = x[i];
      y[INTER ? 2 * i + 1 : 8 + i] = x[8 + i];
    }
    uint8_t* to = codes + (o0 + j) * D;
    const unsigned u[4] = {codes4<HELD, PLAIN>(y, inv), codes4<HELD, PLAIN>(y + 4, inv), codes4<HELD, PLAIN>(y + 8, inv), codes4<HELD, PLAIN>(y + 12, inv)};
    if (n_lo + n_hi == 16) {
      __builtin_memcpy(to + lo, u, 8);
      __builtin_memcpy(to + hi, u + 2, 8);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i < n_lo) to[lo + i] = (uint8_t)(u[i >> 2] >> (8 * (i & 3)));
        if (i < n_hi) to[hi + i] = (uint8_t)(u[2 + (i >> 2)] >> (8 * (i & 3)));
      }
    }
  }
  static constexpr int kTurned = 2;   // iterations whose turned numbers stay in registers
  static __device__ __forceinline__ unsigned largest_of(unsigned m, const float (&x)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
    return m;
  }
  __device__ __forceinline__ int group_of(int k) const { return blocks > 1 ? k / blocks : k * abreast + sub; }
  __device__ __forceinline__ int pair_of(int k) const { return blocks > 1 ? at + (k % blocks) * 64 : at; }
  __device__ __forceinline__ bool whole(int k) const {   // all rows of the iteration's groups are in the run
    const int g = blocks > 1 ? k / blocks : k * abreast;
    return (g0 + g) * 16 >= o0 && (g0 + g + abreast) * 16 <= o0 + n;
  }
  __device__ __forceinline__ void load_column(P2 (&c)[16], int k) const {
    const int first = (g0 + group_of(k)) * 16 - o0;
    const T* p = rows + min(pair_of(k), width - 1) * 2;
    if (whole(k)) {
      p += (int64_t)first * stride;
#pragma unroll
      for (int e = 0; e < 16; ++e) c[e] = load_numbers<T, 2, P2>(p + e * stride, vec);
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) c[e] = load_numbers<T, 2, P2>(p + (int64_t)min(max(first + e, 0), n - 1) * stride, vec);
    }
  }
  template <bool PLAIN>
  __device__ __forceinline__ void write_eight(int k, const P8& p, float inv) const {
    const int j = k * abreast + sub;
    if (j >= n) return;
    float x[8];
    floats<N, 8>(x, p);
    *(uint2*)(codes + (o0 + j) * D + at * 8) = make_uint2(codes4<HELD, PLAIN>(x, inv), codes4<HELD, PLAIN>(x + 4, inv));
  }
  template <bool PLAIN>
  __device__ __forceinline__ void write_column(int k, const P2 (&c)[16], float inv, float ratio) const {
    const int g = group_of(k), pair = pair_of(k);
    if (g >= count || pair >= width) return;
    uint4* to = (uint4*)(codes + ((g0 + g) * D + pair * 2) * 16);
    uint4 u[2];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float x[4], y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float z[2];
        floats<T, 2>(z, c[q * 4 + e]);
        x[e] = z[0];
        y[e] = z[1];
      }
      ((unsigned*)&u[0])[q] = codes4<HELD, PLAIN>(x, inv);
      ((unsigned*)&u[1])[q] = codes4<HELD, PLAIN>(y, inv);
    }
    if (!whole(k)) {
      const int low = o0 - (g0 + g) * 16, high = low + n;   // tokens of the group that are written: [low, high)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint4 was = to[h];
        if (ratio != 1.0f && low > 0) was = again16<HELD>(was, ratio, low);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int up = min(max(high - 4 * q, 0), 4), down = min(max(low - 4 * q, 0), 4);
          const unsigned fresh = (up == 4 ? ~0u : (1u << (8 * up)) - 1) & ~(down == 4 ? ~0u : (1u << (8 * down)) - 1);
          ((unsigned*)&u[h])[q] = (((unsigned*)&u[h])[q] & fresh) | (((unsigned*)&was)[q] & ~fresh);
        }
      }
    }
    to[0] = u[0];
    to[1] = u[1];
  }
  static constexpr int kKept = VALUES ? 1 : 4;   // iterations whose numbers stay in registers: more of them cost waves
  template <bool PLAIN>
  __device__ __forceinline__ void write(const P8 (&kept8)[VALUES ? 1 : kKept], const P2 (&kept2)[VALUES ? kKept : 1][16], const float (&turned16)[TURN ? kTurned : 1][16], bool keep, float inv, float ratio) const {
    if constexpr (TURN) {
      if (iterations <= kTurned) {
#pragma unroll
        for (int k = 0; k < kTurned; ++k)
          if (k < iterations) write_sixteen<PLAIN>(k, turned16[k], inv);
        return;
      }
#pragma unroll 1
      for (int k = 0; k < iterations; ++k) {
        Raw raw;
        load_sixteen(raw, k);
        float x[16];
        turn_sixteen(x, raw, position_of(*turns, token + row_of(k)));
        write_sixteen<PLAIN>(k, x, inv);
      }
    } else {
    if (keep) {
#pragma unroll
      for (int k = 0; k < kKept; ++k) {
        if (k < iterations) {
          if constexpr (VALUES) write_column<PLAIN>(k, kept2[k], inv, ratio);
          else write_eight<PLAIN>(k, kept8[k], inv);
        }
      }
      return;
    }
#pragma unroll 2
    for (int k = 0; k < iterations; ++k) {
      if constexpr (VALUES) {
        P2 c[16];
        load_column(c, k);
        write_column<PLAIN>(k, c, inv, ratio);
      } else {
        write_eight<PLAIN>(k, load_eight(k), inv);
      }
    }
    }
  }

  // tops: of a run that the workgroup shares, where its waves' largest magnitudes meet (nullptr: the run is this wave's)
  __device__ __forceinline__ void run(bool straight, const int64_t* slots, int page_mask, float* scale_at, unsigned* tops) {
    lane = (int)threadIdx.x & 63;
    const int wave = tops ? __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) : 0, first = o0;   // (of the run)
    const float old = first > 0 ? *scale_at : 0.0f;
    if (tops) {   // a quarter of the groups of 16 tokens
      const int before = o0 >> 4, groups = ((o0 + n + 15) >> 4) - before, per = (groups + kStoreWaves - 1) / kStoreWaves;
      const int from = max((before + wave * per) * 16 - o0, 0), to = min((before + (wave + 1) * per) * 16 - o0, n);
      n = max(to - from, 0);
      o0 += from;
      rows += (int64_t)from * stride;
      if constexpr (TURN) token += from;
    }
    shape();
    P8 kept8[VALUES ? 1 : kKept];
    P2 kept2[VALUES ? kKept : 1][16];
    float turned16[TURN ? kTurned : 1][16];
    const bool keep = iterations <= kKept, used = sub < abreast;
    unsigned m = 0;
    if (straight && used) {
      if constexpr (TURN) {
        if (iterations <= kTurned) {
          Raw raw[kTurned];
          double position[kTurned];
#pragma unroll
          for (int k = 0; k < kTurned; ++k) {
            if (k < iterations) {
              load_sixteen(raw[k], k);
              position[k] = position_of(*turns, token + row_of(k));
            }
          }
#pragma unroll
          for (int k = 0; k < kTurned; ++k) {
            if (k < iterations) {
              turn_sixteen(turned16[k], raw[k], position[k]);
              m = largest_of(m, turned16[k]);
            }
          }
        } else {
#pragma unroll 1
          for (int k = 0; k < iterations; ++k) {
            Raw raw;
            load_sixteen(raw, k);
            turn_sixteen(turned16[0], raw, position_of(*turns, token + row_of(k)));
            m = largest_of(m, turned16[0]);
          }
        }
      } else if (keep) {
#pragma unroll
        for (int k = 0; k < kKept; ++k) {
          if (k < iterations) {
            if constexpr (VALUES) load_column(kept2[k], k);
            else kept8[k] = load_eight(k);
          }
        }
#pragma unroll
        for (int k = 0; k < kKept; ++k) {
          if (k < iterations) {
            if constexpr (VALUES) {
#pragma unroll
              for (int e = 0; e < 16; ++e) m = Pack<T>::see(m, kept2[k][e]);
            } else {
              m = Pack<T>::see(m, kept8[k]);
            }
          }
        }
      } else {
#pragma unroll 2
        for (int k = 0; k < iterations; ++k) {
          if constexpr (VALUES) {
            P2 c[16];
            load_column(c, k);
#pragma unroll
            for (int e = 0; e < 16; ++e) m = Pack<T>::see(m, c[e]);
          } else {
            m = Pack<T>::see(m, load_eight(k));
          }
        }
      }
    }
    m = wave_largest<sizeof(N) == 2>(m);
    if (tops) {
      if (lane == 0) tops[wave] = m;
      __syncthreads();   // (and the scale has been read)
      m = 0;
#pragma unroll
      for (int w = 0; w < kStoreWaves; ++w) m = Pack<N>::larger(m, tops[w]);
    }
    float top = Pack<N>::value(m);
    constexpr float kMost = HELD == 0 ? 448.0f * 0x1p119f : 127.0f * 0x1p121f;
    const bool plain = straight && top <= kMost;
    if (!plain) {   // infinities or NaN (or slots in any order): the largest finite one
      float t = 0.0f;
      for (int j = 0; j < n; ++j)
        for (int d = lane; d < D; d += 64) t = fmaxf(t, finite_abs(number(j, d)));
      top = wave_max64(t);
      if (tops) {
        __syncthreads();
        if (lane == 0) tops[wave] = __float_as_uint(top);
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kStoreWaves; ++w) top = fmaxf(top, __uint_as_float(tops[w]));
      }
    }
    float scale = scale_of<HELD>(top);
    float ratio = 1.0f;   // of the page's scale before to the one from now on
    if (first > 0) {
      if (old > scale && old <= 3.402823466e38f) scale = old;
      else if (old > 0.0f && old < scale) ratio = old / scale;
    }
    if (lane == 0 && wave == 0) *scale_at = scale;
    if (ratio != 1.0f && wave == 0) {
      // what the page holds below o0; the group in which o0 lies, if it is written below, is done there
      const int words = VALUES ? (straight ? g0 : (o0 + 15) >> 4) * D : (o0 * D) >> 4;
      for (int i = lane; i < words; i += 64) {
        uint4* w = (uint4*)codes + i;
        *w = again16<HELD>(*w, ratio, VALUES ? o0 - (i / D) * 16 : 16);
      }
    }
    const float inv = 1.0f / scale;   // (a power of two: exact)
    if (straight) {
      if (!used) return;
      if (plain) write<true>(kept8, kept2, turned16, keep, inv, ratio);
      else write<false>(kept8, kept2, turned16, keep, inv, ratio);
      return;
    }
    // slots in any order: token by token, so that of two rows for one slot the later one stays
    __threadfence_block();   // (the words above and the bytes below come from different lanes)
    for (int j = 0; j < n; ++j) {
      const int o = (int)(slots[j] & page_mask);
      for (int d = lane; d < D; d += 64) {
        const float x[4] = {number(j, d) * inv, 0.0f, 0.0f, 0.0f};
        const uint8_t code = (uint8_t)encode4<HELD>(x);
        if (VALUES) codes[((o >> 4) * D + d) * 16 + (o & 15)] = code;
        else codes[o * D + d] = code;
      }
    }
  }
};

// A workgroup's keys or values of one head.  turns, quarters (LDS, kTurnPairs): of keys that turn (TURN), by the positions of all tokens
constexpr int kTurnPairs = FX_KV_MAX_DEPTH / 2 + 8;
template <int HELD, class T, bool TURN, bool INTER>
__device__ __forceinline__ void store_chunk(const FxKvCache& c, const FxKvRows& r, int per, int vec, unsigned block, const FxTurns* turns, double* quarters, unsigned (*s_tops)[kStoreWaves]) {
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const unsigned chunk_head = block >> 1;
  const int half = (int)(block & 1), chunk = (int)(chunk_head / (unsigned)c.heads), head = (int)(chunk_head - (unsigned)chunk * (unsigned)c.heads);
  const int D = c.depth, page = 1 << c.log_page;
  const int64_t n_slots = (int64_t)c.pages << c.log_page;
  const int t0 = chunk * per, t1 = min(r.tokens, t0 + per);
  if constexpr (TURN) {   // (with the pairs behind the last, which a lane reads of fewer than 8)
    if (half == 0) {
      for (int i = (int)threadIdx.x; i < turns->pairs + 8; i += kThreads) quarters[i] = quarters_of(*turns, min(i, turns->pairs - 1));
      __syncthreads();
    }
  }
  // lane i: the slot of token t0 - 1 + i, which a run that begins in the chunk needs (the first 64 - per of it, at least)
  auto slot_of = [&](int t) -> int64_t {
    const int64_t s = t >= 0 && t < r.tokens ? r.slots[min(max(t, 0), r.tokens - 1)] : -1;
    return s >= 0 && s < n_slots ? s : -1;
  };
  const int64_t mine = slot_of(t0 - 1 + lane);
  int alone = 0, shared = 0;   // runs of one wave, and of all of them, so far
  const int64_t prior = (int64_t)__shfl_up((unsigned long long)mine, 1u, 64);
  unsigned long long begins = __ballot(lane > 0 && lane <= t1 - t0 && mine >= 0 && !(prior >= 0 && prior >> c.log_page == mine >> c.log_page));
  for (; begins != 0; begins &= begins - 1) {
    const int at = __builtin_ctzll(begins), t = t0 + at - 1;
    const int64_t s0 = lane_of(mine, at), p = s0 >> c.log_page;
    // the run's length, and whether its slots rise by one
    int n = 0;
    bool straight = true;
    int64_t seen = mine;
    int first = at;   // the lane of the run's next token
    for (;;) {
      const bool here = lane >= first && seen >= 0 && seen >> c.log_page == p;
      const unsigned long long same = __ballot(here) >> first, rising = __ballot(here && seen == s0 + n + lane - first) >> first;
      const int most = 64 - first, more = ~same == 0 ? 64 : min(__builtin_ctzll(~same), most);
      const unsigned long long part = more == 64 ? ~0ull : (1ull << more) - 1;
      straight = straight && (rising & part) == part;
      n += more;
      if (more < most) break;
      first = 0;
      seen = slot_of(t + n + lane);
    }
    const bool together = straight && n > 16;   // (what decides is the same in all waves)
    if (!together && alone++ % kStoreWaves != wave) continue;
    unsigned* tops = together ? s_tops[shared++ & 1] : nullptr;
    const int o0 = (int)(s0 & (page - 1));
    const int64_t in_page = (int64_t)head * page * D;
    if (half == 0) {
      StoreRun<HELD, T, false, TURN, INTER> run;
      run.rows = (const T*)r.k + (int64_t)t * r.k_token + (int64_t)head * r.k_head;
      run.stride = r.k_token;
      run.n = n, run.o0 = o0, run.D = D, run.vec = vec != 0;
      run.codes = c.k + p * c.k_stride + in_page;
      if constexpr (TURN) run.turns = turns, run.token = t, run.quarters = quarters;
      run.run(straight, r.slots + t, page - 1, c.k_scale + p * c.ks_stride + head, tops);
    } else {
      StoreRun<HELD, T, true> run;
      run.rows = (const T*)r.v + (int64_t)t * r.v_token + (int64_t)head * r.v_head;
      run.stride = r.v_token;
      run.n = n, run.o0 = o0, run.D = D, run.vec = vec != 0;
      run.codes = c.v + p * c.v_stride + in_page;
      run.run(straight, r.slots + t, page - 1, c.v_scale + p * c.vs_stride + head, tops);
    }
  }
}

template <int HELD, class T>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 ? 5 : 4) void fx_kv_store_kernel(const FxKvCache c, const FxKvRows r, int per, int vec) {
  __shared__ unsigned s_tops[2][kStoreWaves];
  store_chunk<HELD, T, false, false>(c, r, per, vec, blockIdx.x, nullptr, nullptr, s_tops);
}

// tokens a wave takes: as many as leave some 8 192 waves (32 a CU), `most` at most
inline int tokens_a_wave(const FxKvCache& c, const FxKvRows& r, int most) {
  const int64_t per = (int64_t)r.tokens * c.heads * 2 / 8192;
  return (int)(per < 1 ? 1 : per > most ? most : per);
}
inline bool aligned16(const void* p, int64_t a, int64_t b, size_t size) {
  return ((uintptr_t)p & 15u) == 0 && a * (int64_t)size % 16 == 0 && b * (int64_t)size % 16 == 0;
}
// How the tokens of a call that stores are dealt out: `per` tokens a workgroup, a key head, keys and values apart
struct StoreShape {
  int per, vec;
  int64_t blocks;
};
inline StoreShape store_shape(const FxKvCache& c, const FxKvRows& r) {
  const size_t size = r.dtype == FX_DT_F32 ? 4 : 2;
  StoreShape s;
  // (a workgroup for each 32 tokens took 96 us where 63 take 73)
  s.per = std::max(std::min(tokens_a_wave(c, r, FX_KV_STORE_MOST) * kStoreWaves, FX_KV_STORE_MOST), kStoreWaves);
  s.vec = aligned16(r.k, r.k_token, r.k_head, size) && aligned16(r.v, r.v_token, r.v_head, size);
  s.blocks = (int64_t)((r.tokens + s.per - 1) / s.per) * c.heads * 2;
  return s;
}
}  // namespace
