// A beam search's selection: of each request the `count` best continuations of all its beams and words, by score + logit - log sum exp(logits).
//
// Two launches, or fx_beam_join alone for rows of one part.  fx_beam_scan reads the logits once; a wave leaves the sum of exponentials of its 2 048 (16-bit types) or 1 024 words and the largest of each
// eighth of them.  fx_beam_join, a workgroup a request and a wave a row, finds from these which few segments the best words can lie in, reads those again (from the caches, as a
// rule) and takes their best; then it ranks the rows' candidates.  (The best words of every part found by fx_beam_scan itself: 31 us for 488 rows of 128 001 words,
// half of them instructions of that search.)
//
// What is compared within a row are its logits; between rows score + (logit - lse) in 64 bits.  Sums of exponentials: eight at a time in fp32, these in
// 64 bits, so that lse is off by some 1e-8 and rows change places only where they are as near as that.
//
// The best `count` words: a bound is searched for, a quarter of what is left at a time, until at least `count` of 256 groups of segments, and hardly more, have a word at or
// above it; the words at or above it are a few more than `count`, and are ranked by counting.  Equal numbers: lower words go first, and so as many as there may be of them
// never need more than a list's places (it is cut to the best `count` when it fills up).
//
// 488 rows of 128 001 words, bf16, 390 of them alive: 24.5 us (4.1 TB/s; to read them and do nothing but the sum takes 18) and 10.6; 64 of 50 001: 4.6 and 8.6;
// 4 of 32 000, fp32: 3.3 and 7.0.  Rows that are masked with one finite number but for fewer words than `count`: the bound stays at that number, every segment has words at it, and
// fx_beam_join walks them all (4 rows of 128 001 words, 3 of them free, 8 wanted, bf16: 740 us a call, and 12 where the mask is -infinity).
#include <algorithm>

#include "fx_beam.h"

namespace {
constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kLoads = 4;    // of 16 bytes that a lane of fx_beam_scan has under way (read for the sum alone, without segments: 488 rows of 128 001 words 23 us with 8, 18 with 4)
constexpr int kMore = 128;   // candidates that a wave keeps besides the best `count`: two steps' of 64
constexpr int kList = FX_BEAM_MAX_COUNT + kMore;
constexpr int kSegments = 384;   // that it lists before it looks at them
constexpr int kPer = kLoads * 4 / FX_BEAM_SEGMENTS;   // loads of 16 lanes that are a segment (1: fx_beam_scan 25.4 us instead of 24.4; 4: 22.5, but fx_beam_join 2.5 us more)
constexpr int kUnder = 6;        // loads of a lane of fx_beam_join under way: 12 segments
constexpr int kJoinWaves = 16;   // rows of a request at a time, at most
constexpr int kLinear = 256;     // candidates of a request that are ranked against each other; more are joined in pairs of rows (450: 17 us instead of 22; 256: 14.5, and 15 in pairs)
constexpr float kLowest = -3.402823466e38f;   // (-infinity is none)

__device__ __forceinline__ float wave_max(float m) {
  const auto step = [](float m, int s) { return fmaxf(m, __uint_as_float((unsigned)s)); };
#define FX_STEP(ctrl, rows) m = step(m, __builtin_amdgcn_update_dpp((int)__float_as_uint(m), (int)__float_as_uint(m), ctrl, rows, 0xf, false));
  FX_STEP(0x111, 0xf) FX_STEP(0x112, 0xf) FX_STEP(0x114, 0xf) FX_STEP(0x118, 0xf) FX_STEP(0x142, 0xa) FX_STEP(0x143, 0xc)
#undef FX_STEP
  return __uint_as_float((unsigned)__builtin_amdgcn_readlane((int)__float_as_uint(m), 63));
}
// (of all lanes, in an order of its own that does not change; lanes that a step does not reach add 0)
__device__ __forceinline__ double wave_sum(double v) {
#define FX_STEP(ctrl, rows)                                                                                       \
  {                                                                                                               \
    const int low = __builtin_amdgcn_update_dpp(0, __double2loint(v), ctrl, rows, 0xf, false);                    \
    const int high = __builtin_amdgcn_update_dpp(0, __double2hiint(v), ctrl, rows, 0xf, false);                   \
    v += __hiloint2double(high, low);                                                                             \
  }
  FX_STEP(0x111, 0xf) FX_STEP(0x112, 0xf) FX_STEP(0x114, 0xf) FX_STEP(0x118, 0xf) FX_STEP(0x142, 0xa) FX_STEP(0x143, 0xc)
#undef FX_STEP
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), 63), __builtin_amdgcn_readlane(__double2loint(v), 63));
}
// a wave's accesses to LDS go in order: only the compiler has to keep it
__device__ __forceinline__ void in_wave() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
// whole numbers in the order of floats (no NaN)
__device__ __forceinline__ int ordered(float x) {
  const int i = (int)__float_as_uint(x);
  return i ^ ((i >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float unordered(int i) { return __uint_as_float((unsigned)(i ^ ((i >> 31) & 0x7fffffff))); }
// larger keys go first: larger numbers (-0 is 0), then lower words
__device__ __forceinline__ uint64_t key_of(float x, uint32_t word) { return ((uint64_t)((unsigned)ordered(x + 0.0f) ^ 0x80000000u) << 32) | (0xffffffffu - word); }
__device__ __forceinline__ float x_of(uint64_t key) { return unordered((int)((unsigned)(key >> 32) ^ 0x80000000u)); }
__device__ __forceinline__ uint32_t word_of(uint64_t key) { return 0xffffffffu - (unsigned)key; }
__device__ __forceinline__ int below(uint64_t mask) {   // set lanes below this one
  return (int)__builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask, 0u));
}

// How many of keys[0, n) are larger than each of a lane's (lane, lane + 64, ...)
__device__ __forceinline__ void rank_keys(const uint64_t* keys, int n, int lane, uint64_t (&mine)[kList / 64], int (&rank)[kList / 64]) {
#pragma unroll
  for (int i = 0; i < kList / 64; ++i) {
    mine[i] = lane + 64 * i < n ? keys[lane + 64 * i] : 0;
    rank[i] = 0;
  }
#pragma unroll 8
  for (int j = 0; j < n; ++j) {
    const uint64_t k = keys[j];
    rank[0] += k > mine[0] ? 1 : 0;
    if (n > 64) {
#pragma unroll
      for (int i = 1; i < kList / 64; ++i) rank[i] += k > mine[i] ? 1 : 0;
    }
  }
}

// 16 bytes as they are loaded, and the numbers in them (whole words throughout: halves would take a register each)
template <class T> struct Load;
template <> struct Load<float> {
  static constexpr unsigned kNone = 0xff800000u;   // -infinity, here and below two of them
  unsigned u[4];
  __device__ __forceinline__ float operator[](int e) const { return __uint_as_float(u[e]); }
};
template <> struct Load<_Float16> {
  static constexpr unsigned kNone = 0xfc00fc00u;
  unsigned u[4];
  __device__ __forceinline__ float operator[](int e) const { return (float)__builtin_bit_cast(_Float16, (unsigned short)(e % 2 ? u[e / 2] >> 16 : u[e / 2])); }
};
template <> struct Load<__bf16> {
  static constexpr unsigned kNone = 0xff80ff80u;
  unsigned u[4];
  __device__ __forceinline__ float operator[](int e) const { return __uint_as_float(e % 2 ? u[e / 2] & 0xffff0000u : u[e / 2] << 16); }
};
// A part's sum is of terms 2^(x c - r), r the whole number next to the largest x c: product and difference are rounded once.  c is log2 e (1 + 1.3e-8), which is 1e-8 in the terms
// that count.  From 2^22 on fp32 has no whole number so near (a product rounded to 2^31 or more is 128 and more from itself): such parts' terms are 2^((x - largest) c), a
// difference that is exact wherever the term is not 0, and their sum is brought to r, in 64 bits, behind.
constexpr float kC = 1.44269504088896340736f;
__device__ __forceinline__ bool far_from(float top) { return __builtin_fabsf(top) > 0x1p22f; }
__device__ __forceinline__ double scaled(float top) { return (double)top * (double)kC; }   // (48 bits: exact)
__device__ __forceinline__ double whole_of(float top) { return __builtin_rint(scaled(top)); }
// a part's sum under `whole`, the r of the row's largest logit (of no words: 0, or NaN)
__device__ __forceinline__ double part_of(const FxBeamPart& p, double whole) {
  return p.top > -INFINITY ? p.sum * __builtin_amdgcn_ldexp(1.0, (int)fmax(whole_of(p.top) - whole, -4000.0)) : p.sum;
}
// (the largest logit and what the others add to it: rounded at the logit's own size once, whatever that is)
__device__ __forceinline__ double lse_of(float most, double whole, double sum) { return (double)most + (log(sum) + (whole - scaled(most)) * 0.69314718055994530942); }

// Words of a row: load l of a part, in its lane.  Loads that would begin in a row's last words lie at its end (at), less the first ones, which are other lanes'
template <class T>
struct Words {
  static constexpr int kVec = 16 / (int)sizeof(T), kPart = 64 * kVec * kLoads;
  const T* x;
  int words;
  __device__ __forceinline__ int at(int place) const { return min(place, words - kVec); }
  // the numbers from `place` on, -infinity for those that are not the lane's
  __device__ __forceinline__ Load<T> load(int place) const {
    Load<T> v;
    __builtin_memcpy(v.u, (const char*)x + (unsigned)at(place) * (unsigned)sizeof(T), 16);
    return v;
  }
  __device__ __forceinline__ void mask(Load<T>& v, int place) const {
    const int skip = place - at(place);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (sizeof(T) == 4) v.u[i] = skip > i ? Load<T>::kNone : v.u[i];
      else v.u[i] = skip > 2 * i + 1 ? Load<T>::kNone : skip == 2 * i + 1 ? (v.u[i] & 0xffff0000u) | (Load<T>::kNone & 0xffffu) : v.u[i];
    }
  }
  // of a row that is shorter than a load: all of it
  __device__ __forceinline__ Load<T> load_tiny() const {
    T few[kVec];
#pragma unroll
    for (int e = 0; e < kVec; ++e) few[e] = e < words ? x[e] : (T)(-INFINITY);
    Load<T> v;
    __builtin_memcpy(v.u, few, 16);
    return v;
  }
};
template <class T>
__device__ __forceinline__ Words<T> words_of(const FxBeamArgs& a, int64_t row) {
  const int64_t request = row / a.beams;
  Words<T> w;
  w.x = (const T*)a.logits + request * a.l_request + (row - request * a.beams) * a.l_beam;
  w.words = a.words;
  return w;
}
// the largest of the lane's 16 lanes, in the last of them (of whole numbers the compiler makes one instruction a step)
__device__ __forceinline__ int segment_max(int m) {
#define FX_STEP(ctrl) m = max(m, __builtin_amdgcn_update_dpp((int)0x80000000, m, ctrl, 0xf, 0xf, false));
  FX_STEP(0x111) FX_STEP(0x112) FX_STEP(0x114) FX_STEP(0x118)
#undef FX_STEP
  return m;
}

// A wave's part of a row: its sum, and the largest word of each segment
template <class T>
__device__ __forceinline__ void scan_part(const FxBeamArgs& a, int row, int part, int unit, int lane) {
  typedef Words<T> W;
  const W w = words_of<T>(a, row);
  const int begin = part * W::kPart + lane * W::kVec;   // load l: words begin + l * 64 * kVec on
  Load<T> v[kLoads];
  if (w.words >= W::kVec) {
#pragma unroll
    for (int l = 0; l < kLoads; ++l) v[l] = w.load(begin + l * 64 * W::kVec);
    if ((part + 1) * W::kPart > w.words) {
#pragma unroll
      for (int l = 0; l < kLoads; ++l) w.mask(v[l], begin + l * 64 * W::kVec);
    }
  } else {
#pragma unroll
    for (int l = 0; l < kLoads; ++l) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[l].u[i] = Load<T>::kNone;
    }
    if (lane == 0) v[0] = w.load_tiny();
  }
  float x[kLoads][W::kVec];
  int all = (int)0x80000000;
  float pair = -INFINITY;
  int* const tops = a.tops + (int64_t)unit * FX_BEAM_SEGMENTS + (lane >> 4);
#pragma unroll
  for (int l = 0; l < kLoads; ++l) {
    float m = -INFINITY;
#pragma unroll
    for (int e = 0; e < W::kVec; ++e) {
      x[l][e] = v[l][e];
      m = fmaxf(m, x[l][e]);   // (NaN is passed over here, and is in the sum)
    }
    pair = fmaxf(pair, m);
    if (l % kPer == kPer - 1) {
      const int segment = segment_max(ordered(pair));
      if ((lane & 15) == 15) tops[l / kPer * 4] = segment;
      all = max(all, segment);
      pair = -INFINITY;
    }
  }
  const float most = unordered(max(max(__builtin_amdgcn_readlane(all, 15), __builtin_amdgcn_readlane(all, 31)), max(__builtin_amdgcn_readlane(all, 47), __builtin_amdgcn_readlane(all, 63))));
  const bool far = far_from(most);
  const float r = most > -INFINITY ? (float)whole_of(most) : 0.0f;
  double sum = 0.0;
  if (!far) {
#pragma unroll
    for (int l = 0; l < kLoads; ++l) {
      float some = 0.0f;
#pragma unroll
      for (int e = 0; e < W::kVec; ++e) some += __builtin_amdgcn_exp2f(__builtin_fmaf(x[l][e], kC, -r));
      sum += (double)some;
    }
  } else {
    const float least = most > -INFINITY ? most : 0.0f;
#pragma unroll
    for (int l = 0; l < kLoads; ++l) {
      float some = 0.0f;
#pragma unroll
      for (int e = 0; e < W::kVec; ++e) some += __builtin_amdgcn_exp2f((x[l][e] - least) * kC);
      sum += (double)some;
    }
  }
  sum = wave_sum(sum);
  if (far && most > -INFINITY) sum *= (double)__builtin_amdgcn_exp2f((float)(scaled(most) - whole_of(most)));
  if (lane == 0) {
    a.parts[unit].top = most;
    a.parts[unit].sum = sum;
  }
}

// Bound: HBM.  A wave a part; nothing is shared between waves.
template <class T>
__global__ __launch_bounds__(kThreads, 8) void fx_beam_scan(const FxBeamArgs a) {
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int unit = (int)blockIdx.x * kWaves + wave, row = unit / a.parts_a_row;
  if (row >= a.requests * a.beams) return;
  // (beams with no continuations of their own are not read)
  if ((a.ended && a.ended[row]) || !(a.scores[row] > -INFINITY)) return;
  scan_part<T>(a, row, unit - row * a.parts_a_row, unit, lane);
}

// Bound: latency.  A row is a chain of some ten steps, and the code of each arrives for the first time: loops are not unrolled where they need not be (16 segments' loads in
// registers, 28 KB of code, took 2 us more than this).
// ALONE: rows of one part, for which there was no fx_beam_scan (6 x 2 rows of 109 words: 8.2 us a call, 13.1 in two launches).
template <class T, bool ALONE>
__global__ __launch_bounds__(64 * kJoinWaves) void fx_beam_join(const FxBeamArgs a) {
  typedef Words<T> W;
  extern __shared__ uint4 s_join[];
  const int count = a.count, K = a.beams, lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), waves = (int)blockDim.x >> 6;
  uint4* loads = s_join + wave * 64;                               // [waves][64]
  double* score = (double*)(s_join + waves * 64);                  // [beams][count]
  const int room = count + kMore;
  uint64_t* keys = (uint64_t*)score + K * count + wave * room;     // [waves][room]
  uint32_t* word = (uint32_t*)((uint64_t*)score + K * count + waves * room);    // [beams][count]
  int* places = (int*)(word + K * count) + wave * 64;              // [waves][64]
  uint16_t* list = (uint16_t*)((int*)(word + K * count) + waves * 64) + wave * kSegments;   // [waves][kSegments]; a row of 2^18 words has 2 048 segments
  const int64_t request = blockIdx.x;
  const int fours = a.parts_a_row * (FX_BEAM_SEGMENTS / 4);        // of segments of a row
  for (int k = wave; k < K; k += waves) {
    const int64_t row = request * K + k;
    // (all loads at once: what beams with no candidates of their own have there is never looked at)
    const float before = a.scores[row];
    const bool over = a.ended && a.ended[row];
    if constexpr (ALONE) {
      if (!over && before > -INFINITY) scan_part<T>(a, (int)row, 0, (int)row, lane);
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
    }
    const int4* tops = (const int4*)a.tops + row * fours;
    const FxBeamPart* parts = a.parts + row * a.parts_a_row;
    const FxBeamPart none{-INFINITY, 0.0f, 0.0};
    const FxBeamPart first = lane < a.parts_a_row ? parts[lane] : none;
    float group[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};   // 256 groups of segments: four to a lane
#pragma unroll 1
    for (int i0 = 0; i0 < fours; i0 += 256) {
      int4 t[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) t[g] = tops[min(i0 + 64 * g + lane, fours - 1)];   // (the last one again)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const bool some = i0 + 64 * g + lane < fours;
        group[0] = fmaxf(group[0], some ? unordered(t[g].x) : -INFINITY);
        group[1] = fmaxf(group[1], some ? unordered(t[g].y) : -INFINITY);
        group[2] = fmaxf(group[2], some ? unordered(t[g].z) : -INFINITY);
        group[3] = fmaxf(group[3], some ? unordered(t[g].w) : -INFINITY);
      }
    }
    const bool live = before > -INFINITY;
    int n = 0;
    if (over) {
      if (lane == 0 && live) {
        score[k * count] = (double)before;
        word[k * count] = 0;   // (the end word, which need not be one of the vocabulary's)
      }
      n = live ? 1 : 0;
    } else if (live) {
      const float top = wave_max(fmaxf(fmaxf(group[0], group[1]), fmaxf(group[2], group[3])));
      if (top > -INFINITY) {
        const auto above = [&](float b) {
          int some = 0;
#pragma unroll
          for (int g = 0; g < 4; ++g) some += __builtin_popcountll(__ballot(group[g] >= b));
          return some;
        };
        // a bound with at least `count` groups at or above it and hopefully no more than `enough`; `low` is one to begin with, `high` the largest.
        // (quarters instead of halves, whose counts do not wait for each other)
        const auto raise = [&](float low, float high, int enough) {
          if (high - 64.0f > low && above(high - 64.0f) >= count) low = high - 64.0f;
#pragma unroll 1
          for (int i = 0; i < 10; ++i) {
            const float mid = 0.5f * low + 0.5f * high, one = 0.5f * low + 0.5f * mid, three = 0.5f * mid + 0.5f * high;
            if (!(mid > low)) break;
            const int at_one = above(one), at_mid = above(mid), at_three = above(three);
            int some = at_one;
            if (at_three >= count) low = three, some = at_three;
            else if (at_mid >= count) low = mid, high = three, some = at_mid;
            else if (at_one >= count) low = one, high = mid;
            else high = one;
            if (some >= count && some <= enough) break;
          }
          return low;
        };
        // (all groups are at or above the least; of long rows, fewer segments than 12 take as long as so many)
        const float low = raise(-wave_max(-fminf(fminf(group[0], group[1]), fminf(group[2], group[3]))), top, max(count + 2, min(12, fours)));
        float bound = fmaxf(low, kLowest);
        uint32_t last = 0xffffffffu;      // of words equal to the bound, those up to this one
        const W w = words_of<T>(a, row);
        const bool tiny = w.words < W::kVec;
        double lse = 0.0;
#pragma unroll 1
        for (int seen = 0; seen < fours;) {
          int listed = 0;
#pragma unroll 1
          for (; seen < fours && listed <= kSegments - 256; seen += 64) {
            const int i0 = seen;
            const int4 t = tops[min(i0 + lane, fours - 1)];
            const float each[4] = {unordered(t.x), unordered(t.y), unordered(t.z), unordered(t.w)};
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const bool some = i0 + lane < fours && each[q] >= bound;
              const uint64_t lanes = __ballot(some);
              if (some) list[listed + below(lanes)] = (i0 + lane) * 4 + q;
              listed += __builtin_popcountll(lanes);
            }
          }
          in_wave();
          // The words of the listed segments, 32 lanes a segment, six loads under way.  Of the loads those that have a word above the bound go to LDS, 64 at most,
          // and from there each of their words to a lane.  If they have more than 256 words (of rows with few segments, or equal words), the bound is raised
          // once, by the largest words of 256 groups of the loads; if that leaves more than 64 loads, all take that way, four segments at a time.  (101 x 11 rows of
          // 579 words, 22 wanted: 54 us without, 19 with it.)
          const auto place_of = [&](int i) {   // (of none: behind the last word, where nothing is the lane's)
            if (i >= listed) return a.words;
            const int s = list[i], part = s / FX_BEAM_SEGMENTS, first = s % FX_BEAM_SEGMENTS / 4 * kPer + ((lane >> 4) & (kPer - 1));   // the load of the part
            return part * W::kPart + (first * 64 + (s & 3) * 16 + (lane & 15)) * W::kVec;
          };
          const auto load = [&](int place) {
            if (!tiny) return w.load(place);
            Load<T> v = w.load_tiny();
            if (place != 0) v.u[0] = v.u[1] = v.u[2] = v.u[3] = Load<T>::kNone;
            return v;
          };
          int found = 0;
#pragma unroll 1
          for (int time = 0;; ++time) {
            found = 0;
#pragma unroll 1
            for (int i0 = 0; i0 < listed; i0 += kUnder * 4 / kPer) {
              Load<T> v[kUnder];
              int place[kUnder];
#pragma unroll
              for (int u = 0; u < kUnder; ++u) {
                place[u] = place_of(i0 + (4 * u + (lane >> 4)) / kPer);
                v[u] = load(place[u]);
              }
              if (lse == 0.0) {   // (the first time, while they are under way)
                const double whole = whole_of(top);
                double sum = part_of(first, whole);
#pragma unroll 1
                for (int i = lane + 64; i < a.parts_a_row; i += 64) sum += part_of(parts[i], whole);
                lse = lse_of(top, whole, wave_sum(sum));
                if (!(lse - lse == 0.0)) listed = 0, seen = fours;   // (a row with NaN or +infinity has no candidates)
              }
#pragma unroll
              for (int u = 0; u < kUnder; ++u) {
                float m = v[u][0];   // (of words that are other lanes', too: they are passed over below)
#pragma unroll
                for (int e = 1; e < W::kVec; ++e) m = fmaxf(m, v[u][e]);
                const bool some = m >= bound && place[u] < a.words;
                const uint64_t lanes = __ballot(some);
                const int to = found + below(lanes);
                if (some && to < 64) {
                  loads[to] = make_uint4(v[u].u[0], v[u].u[1], v[u].u[2], v[u].u[3]);
                  places[to] = place[u];
                }
                found += __builtin_popcountll(lanes);
              }
            }
            if (listed == 0) found = 0;
            if (found <= 256 / W::kVec || time == 1) break;
            group[0] = group[1] = group[2] = group[3] = -INFINITY;
#pragma unroll 1
            for (int i0 = 0; i0 < listed; i0 += 16 / kPer) {
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                const int place = place_of(i0 + (4 * u + (lane >> 4)) / kPer);
                Load<T> v = w.load(place);   // (a row of one load has not so many)
                w.mask(v, place);
#pragma unroll
                for (int e = 0; e < W::kVec; ++e) group[u] = fmaxf(group[u], v[e]);
              }
            }
            if (above(bound) < count) break;
            const float raised = raise(bound, top, count + 2);
            if (!(raised > bound)) break;
            bound = raised;
            last = 0xffffffffu;
          }
          const bool few = found <= 64;
          int i0 = 0;    // of the segments, where they come four at a time
#pragma unroll 1
          while (found > 0) {
            if (!few) {
              in_wave();
              const int place = place_of(i0 + (lane >> 4) / kPer);
              const Load<T> v = load(place);
              loads[lane] = make_uint4(v.u[0], v.u[1], v.u[2], v.u[3]);
              places[lane] = place;
              found = 64;
            }
            in_wave();
            int i1 = 0;
            if (found * W::kVec <= 256) {
              // few words: four to a lane, and the bound is raised by themselves if many of them are above it (15 beams of 247 words, 15 wanted: 14.4 us, by their
              // loads 17.6, not at all 21)
              uint32_t here[4];
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                const int i = (lane + 64 * g) / W::kVec, e = lane % W::kVec;
                group[g] = -INFINITY;
                here[g] = 0;
                if (i >= found) continue;
                const int place = places[i], at = tiny ? 0 : w.at(place);
                const float z = (float)((const T*)loads)[i * W::kVec + e];
                here[g] = (uint32_t)(at + e);
                if (at + e >= place && place < a.words && (z > bound || (z == bound && here[g] <= last))) group[g] = z;
              }
              int hits = above(kLowest);
              if (hits > count + 24) {
                const float raised = raise(bound, top, count + 2);
                if (raised > bound) {
                  bound = raised;
                  last = 0xffffffffu;
#pragma unroll
                  for (int g = 0; g < 4; ++g) group[g] = group[g] >= bound ? group[g] : -INFINITY;
                  hits = above(bound);
                }
              }
              if (n + hits <= room) {
                i1 = found;   // (no others: the list is ranked)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                  const uint64_t lanes = __ballot(group[g] >= kLowest);
                  if (group[g] >= kLowest) keys[n + below(lanes)] = key_of(group[g], here[g]);
                  n += __builtin_popcountll(lanes);
                }
              }
            }
#pragma unroll 1
            for (; i1 < found + 64 / W::kVec; i1 += 64 / W::kVec) {   // (and once more, for what is left in the list)
              if (n > room - 64 || i1 >= found) {
                // no room for a word of each lane, or the end: the best `count`, in order; what comes has to be better than the last of them
                uint64_t mine[kList / 64];
                int rank[kList / 64];
                in_wave();
                rank_keys(keys, n, lane, mine, rank);
                in_wave();
#pragma unroll
                for (int i = 0; i < kList / 64; ++i)
                  if (lane + 64 * i < n && rank[i] < count) keys[rank[i]] = mine[i];
                in_wave();
                n = min(n, count);
                if (n == count) {
                  const uint64_t worst = keys[n - 1];
                  bound = x_of(worst);
                  last = word_of(worst);
                }
              }
              const int i = i1 + lane / W::kVec, e = lane % W::kVec;
              float z = -INFINITY;
              uint32_t here = 0;
              if (i < found) {
                const int place = places[i], at = tiny ? 0 : w.at(place);
                here = (uint32_t)(at + e);
                if (at + e >= place && place < a.words) z = (float)((const T*)loads)[i * W::kVec + e];
              }
              const bool hit = z > bound || (z == bound && here <= last);
              const uint64_t lanes = __ballot(hit);
              if (hit) keys[n + below(lanes)] = key_of(z, here);
              n += __builtin_popcountll(lanes);
            }
            i0 += 4 / kPer;
            if (few || i0 >= listed) break;
          }
        }
        in_wave();
        for (int i = lane; i < n; i += 64) {
          score[k * count + i] = (double)before + ((double)x_of(keys[i]) - lse);
          word[k * count + i] = word_of(keys[i]);
        }
        in_wave();
      }
    }
    for (int i = n + lane; i < count; i += 64) score[k * count + i] = -INFINITY;
  }
  __syncthreads();
  const int all = K * count;
  if (all <= kLinear) {
    // the place of a candidate: how many are better, or as good and before it; eight lanes to a candidate
    const int eighth = (int)threadIdx.x & 7;
    for (int i = (int)threadIdx.x >> 3; i < all; i += (int)blockDim.x >> 3) {
      const double s = score[i];
      int rank = 0;
#pragma unroll 4
      for (int j = eighth; j < all; j += 8) {
        const double t = score[j];
        rank += t > s || (t == s && j < i) ? 1 : 0;
      }
      rank += __shfl_xor(rank, 1, 64);
      rank += __shfl_xor(rank, 2, 64);
      rank += __shfl_xor(rank, 4, 64);
      if (eighth != 0 || rank >= count || !(s > -INFINITY)) continue;
      const int k = i / count;
      const int64_t to = request * count + rank;
      a.out_scores[to] = (float)s;
      a.out_beams[to] = k;
      a.out_words[to] = a.ended && a.ended[request * K + k] ? a.end_word : (int64_t)word[i];
    }
  } else {
    // each row's are in order: two rows' lists at a time become one, of the best `count`; a place is found by halves in the other list
    int* from = (int*)s_join;   // [beams][count], where the loads were
    for (int i = (int)threadIdx.x; i < all; i += (int)blockDim.x) from[i] = i;
    for (int d = 1; d < K; d <<= 1) {
      constexpr int kEach = 4;   // of a thread: a wave has four rows or fewer
      __syncthreads();
      double s[kEach];
      int id[kEach], to[kEach];
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        const int i = (int)threadIdx.x + e * (int)blockDim.x, k = i / count, at = i - k * count;
        to[e] = -1;
        const bool right = (k & d) != 0;
        const int other = right ? k - d : k + d;
        if (i >= all || (k & (d - 1)) != 0 || other >= K) continue;
        s[e] = score[i];
        id[e] = from[i];
        int less = 0, more = count;   // of the other list: `less` at least go before this one, `more` at most
        while (less < more) {
          const int mid = (less + more) >> 1;
          const double t = score[other * count + mid];
          const bool before = right ? t >= s[e] : t > s[e];
          less = before ? mid + 1 : less;
          more = before ? more : mid;
        }
        if (at + less < count) to[e] = (k & ~d) * count + at + less;
      }
      __syncthreads();
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        if (to[e] < 0) continue;
        score[to[e]] = s[e];
        from[to[e]] = id[e];
      }
    }
    __syncthreads();
    for (int i = (int)threadIdx.x; i < count; i += (int)blockDim.x) {
      const double s = score[i];
      if (!(s > -INFINITY)) continue;
      const int k = from[i] / count;
      const int64_t to = request * count + i;
      a.out_scores[to] = (float)s;
      a.out_beams[to] = k;
      a.out_words[to] = a.ended && a.ended[request * K + k] ? a.end_word : (int64_t)word[from[i]];
    }
  }
  // places that are left
  if (wave == 0) {
    int there = 0;
    for (int i = lane; i < (all <= kLinear ? all : count); i += 64) there += score[i] > -INFINITY ? 1 : 0;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) there += __shfl_xor(there, d, 64);
    for (int i = there + lane; i < count; i += 64) {
      const int64_t to = request * count + i;
      a.out_scores[to] = -INFINITY;
      a.out_beams[to] = -1;
      a.out_words[to] = -1;
    }
  }
}
}  // namespace

void fx_beam_shape(FxBeamArgs& a) {
  const int words = 64 * (a.dtype == FX_DT_F32 ? 4 : 8) * kLoads;
  a.parts_a_row = (a.words + words - 1) / words;
}

hipError_t fx_launch_beam_select(const FxBeamArgs& a, hipStream_t stream, int* launched) {
  static const void* const scans[3] = {(const void*)fx_beam_scan<float>, (const void*)fx_beam_scan<_Float16>, (const void*)fx_beam_scan<__bf16>};
  static const void* const joins[2][3] = {{(const void*)fx_beam_join<float, false>, (const void*)fx_beam_join<_Float16, false>, (const void*)fx_beam_join<__bf16, false>},
                                          {(const void*)fx_beam_join<float, true>, (const void*)fx_beam_join<_Float16, true>, (const void*)fx_beam_join<__bf16, true>}};
  const int type = a.dtype == FX_DT_F32 ? 0 : a.dtype == FX_DT_F16 ? 1 : 2;
  FxBeamArgs args = a;
  void* kargs[1] = {(void*)&args};
  const int64_t units = (int64_t)a.requests * a.beams * a.parts_a_row;
  *launched = 0;
  if (a.parts_a_row > 1) {
    const hipError_t e = hipLaunchKernel(scans[type], dim3((unsigned)((units + kWaves - 1) / kWaves)), dim3(kThreads), kargs, 0, stream);
    if (e != hipSuccess) return e;
    *launched = 1;
  }
  // (64 KiB of LDS a workgroup: 32 beams of 64 candidates go in three rounds of eleven)
  const int room = 65536 - a.beams * a.count * 12, a_wave = 64 * 20 + (a.count + kMore) * 8 + kSegments * 2;
  const int rounds = (a.beams + std::min(kJoinWaves, room / a_wave) - 1) / std::min(kJoinWaves, room / a_wave), waves = (a.beams + rounds - 1) / rounds;
  const hipError_t f = hipLaunchKernel(joins[a.parts_a_row > 1 ? 0 : 1][type], dim3((unsigned)a.requests), dim3((unsigned)waves * 64), kargs, (size_t)(a.beams * a.count * 12 + waves * a_wave), stream);
  if (f == hipSuccess) ++*launched;
  return f;
}
