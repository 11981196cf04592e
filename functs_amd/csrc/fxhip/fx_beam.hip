// A beam search's selection: of each request the `count` best continuations of all its beams and words, by score + logit - log sum exp(logits).
//
// Two launches.  fx_beam_scan reads the logits once: a wave takes up to 8 192 words of a row, holds them in registers, and leaves their largest, their
// sum of exponentials and their best `count`, in order.  fx_beam_join, a workgroup a request, merges the parts of a row (a wave a row), then ranks the
// rows' candidates.
//
// What is compared within a row are its logits; between rows score + (logit - lse) in 64 bits.  Sums of exponentials: eight at a time in fp32, these in
// 64 bits, so that lse is off by some 1e-8 and rows change places only where they are as near as that.
//
// The best `count` of a wave's words: the largest of each of 256 groups of words are compared with a bound that is halved until `count` groups, and hardly
// more, have one above it; the words above it are a few more than `count`, and are ranked by counting.  Equal numbers: lower words go first, and so as
// many as there may be of them never need more than the list's 256 places (it is cut to the best `count` when it fills up).
#include <algorithm>

#include "fx_beam.h"

namespace {
constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kList = 256;   // candidates that a wave keeps: the best FX_BEAM_MAX_COUNT and two steps' of 64

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
__device__ __forceinline__ FxBeamWord word_of(uint64_t key) {
  FxBeamWord w;
  w.x = unordered((int)((unsigned)(key >> 32) ^ 0x80000000u));
  w.word = 0xffffffffu - (unsigned)key;
  return w;
}
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
#pragma unroll 4
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
// (between two passes over the words: without it the compiler keeps them as floats as well)
template <class T>
__device__ __forceinline__ void as_loaded(Load<T>& w) { asm volatile("" : "+v"(w.u[0]), "+v"(w.u[1]), "+v"(w.u[2]), "+v"(w.u[3])); }

// Terms 2^(x c - r), r the whole number next to the largest x c: product and difference are rounded once.  c is log2 e (1 + 1.3e-8), for which the sum's
// logarithm is put right.  Numbers whose x c may be infinite: by their difference to the largest.
constexpr float kC = 1.44269504088896340736f;
__device__ __forceinline__ bool far_from(float top) { return __builtin_fabsf(top) > 1e30f; }
__device__ __forceinline__ float whole_of(float top) { return __builtin_rintf(top * kC); }
__device__ __forceinline__ double lse_of(float top, double sum) {
  if (!(top > -INFINITY)) return sum == 0.0 ? -INFINITY : sum;   // (no words, or NaN)
  const double r = far_from(top) ? (double)top * (double)kC : (double)whole_of(top);
  return r * 0.69314718055994530942 + log(sum) - ((double)kC / 1.44269504088896340736 - 1.0) * (double)top;
}

// A wave: 64 * LOADS loads of 16 bytes
template <class T, int LOADS>
__global__ __launch_bounds__(kThreads, LOADS > 8 ? 3 : LOADS > 4 ? 5 : 6) void fx_beam_scan(const FxBeamArgs a) {
  constexpr int kVec = 16 / (int)sizeof(T), kGroups = 4, kPerGroup = LOADS / kGroups, kWords = 64 * kVec * LOADS;
  constexpr unsigned kNone = Load<T>::kNone;
  __shared__ uint64_t s_keys[kWaves][kList];
  __shared__ uint4 s_loads[kWaves][64];
  __shared__ int s_places[kWaves][64];
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int unit = (int)blockIdx.x * kWaves + wave, row = unit / a.chunks, chunk = unit - row * a.chunks;
  if (row >= a.requests * a.beams) return;   // (waves of a workgroup do not wait for each other)
  // beams with no continuations of their own: known ahead of the logits, which need not be read then, or with them where there is little to read
  const bool idle = (a.ended && a.ended[row]) || !(a.scores[row] > -INFINITY);
  if (LOADS > 4 && idle) return;
  const int request = row / a.beams;
  const T* x = (const T*)a.logits + (int64_t)request * a.l_request + (int64_t)(row - request * a.beams) * a.l_beam;
  const int from = chunk * kWords;

  // load l: words at_of(l) on.  Loads that would begin in a row's last words lie at its end, less the first ones, which are other lanes'
  const auto place_of = [&](int l) { return from + (l * 64 + lane) * kVec; };
  const auto at_of = [&](int l) { return min(place_of(l), a.words - kVec); };
  Load<T> v[LOADS];
  if (a.words >= kVec) {
#pragma unroll
    for (int l = 0; l < LOADS; ++l) __builtin_memcpy(v[l].u, (const char*)x + (unsigned)at_of(l) * (unsigned)sizeof(T), 16);
  } else {   // fewer words than a load
#pragma unroll
    for (int l = 0; l < LOADS; ++l) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[l].u[i] = kNone;
    }
    if (lane == 0) {
      T few[kVec];
#pragma unroll
      for (int e = 0; e < kVec; ++e) few[e] = e < a.words ? x[e] : (T)(-INFINITY);
      __builtin_memcpy(v[0].u, few, 16);
    }
  }
  if (LOADS <= 4 && idle) return;

  const int count = a.count;
  uint64_t* keys = s_keys[wave];
  uint4* loads = s_loads[wave];
  int* places = s_places[wave];
  int n = 0;                        // candidates so far
  float bound = -INFINITY;
  uint32_t last = 0xffffffffu;      // of words equal to the bound, those up to this one
  const auto cut = [&]() {          // to the best `count`, in order; what comes has to be better than the last of them
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
      const FxBeamWord worst = word_of(keys[n - 1]);
      bound = worst.x;
      last = worst.word;
    }
  };
  if (a.words >= kVec && from + kWords > a.words) {
#pragma unroll
    for (int l = 0; l < LOADS; ++l) {
      const int skip = place_of(l) - at_of(l);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (sizeof(T) == 4) v[l].u[i] = skip > i ? kNone : v[l].u[i];
        else v[l].u[i] = skip > 2 * i + 1 ? kNone : skip == 2 * i + 1 ? (v[l].u[i] & 0xffff0000u) | (kNone & 0xffffu) : v[l].u[i];
      }
    }
  }
  float best[LOADS];   // of each load
#pragma unroll
  for (int l = 0; l < LOADS; ++l) {
    float m = -INFINITY;
    as_loaded(v[l]);
#pragma unroll
    for (int e = 0; e < kVec; ++e) m = fmaxf(m, v[l][e]);   // (NaN is passed over here, and is in the sum)
    best[l] = m;
    __builtin_amdgcn_sched_barrier(0);   // (one load's words after the other: all of them as floats do not fit)
  }
  float group[kGroups], most = -INFINITY;
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    group[g] = -INFINITY;
#pragma unroll
    for (int l = 0; l < kPerGroup; ++l) group[g] = fmaxf(group[g], best[g * kPerGroup + l]);
    most = fmaxf(most, group[g]);
  }
  most = wave_max(most);

  const bool far = far_from(most);
  const float r = most > -INFINITY ? whole_of(most) : 0.0f;
  double sum = 0.0;
  if (!far) {
#pragma unroll
    for (int l = 0; l < LOADS; ++l) {
      float some = 0.0f;
      as_loaded(v[l]);
#pragma unroll
      for (int e = 0; e < kVec; ++e) some += __builtin_amdgcn_exp2f(__builtin_fmaf(v[l][e], kC, -r));
      sum += (double)some;
      __builtin_amdgcn_sched_barrier(0);
    }
  } else {
    const float least = most > -INFINITY ? most : 0.0f;
#pragma unroll
    for (int l = 0; l < LOADS; ++l) {
      float some = 0.0f;
      as_loaded(v[l]);
#pragma unroll
      for (int e = 0; e < kVec; ++e) some += __builtin_amdgcn_exp2f((v[l][e] - least) * kC);
      sum += (double)some;
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  if (most > -INFINITY) {
    // a bound with at least `count` groups at or above it (all are at or above the least), and hopefully few more
    float least = fminf(fminf(group[0], group[1]), fminf(group[2], group[3])), high = most;
    least = -wave_max(-least);
    const auto above = [&](float b) {
      int some = 0;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) some += __builtin_popcountll(__ballot(group[g] >= b));
      return some;
    };
    float low = fmaxf(least, most - 64.0f);
    if (above(low) < count) low = least;
#pragma unroll 1
    for (int i = 0; i < 12; ++i) {
      const float mid = 0.5f * low + 0.5f * high;
      if (!(mid > low)) break;
      const int some = above(mid);
      if (some >= count) low = mid;
      else high = mid;
      if (some >= count && some <= count + 6) break;
    }
    bound = fmaxf(low, -3.402823466e38f);   // (-infinity is none)
    // The loads that have a word above the bound go to LDS, 64 at most, and from there each of their words to a lane.  More than 64 (of equal words):
    // all loads take that way, read again.
    int found = 0;
#pragma unroll
    for (int l = 0; l < LOADS; ++l) {
      const uint64_t lanes = __ballot(best[l] >= bound);
      if (lanes == 0) continue;
      const int to = found + below(lanes);
      if (best[l] >= bound && to < 64) {
        loads[to] = make_uint4(v[l].u[0], v[l].u[1], v[l].u[2], v[l].u[3]);
        places[to] = a.words >= kVec ? at_of(l) : 0;
      }
      found += __builtin_popcountll(lanes);
    }
    const bool few = found <= 64;   // (rows shorter than a load have one)
#pragma unroll 1
    for (int l = 0; l < (few ? 1 : LOADS); ++l) {
      int skip = 0;
      if (!few) {
        in_wave();
        uint4 w;
        __builtin_memcpy(&w, (const char*)x + (unsigned)at_of(l) * (unsigned)sizeof(T), 16);
        loads[lane] = w;
        places[lane] = at_of(l);
        skip = from + l * 64 * kVec;   // (words before it are other lanes' or an earlier load's)
        found = 64;
      }
      in_wave();
#pragma unroll 1
      for (int i0 = 0; i0 < found; i0 += 64 / kVec) {
        if (n > kList - 64) cut();   // (no room for a word of each lane)
        const int i = i0 + lane / kVec, e = lane % kVec;
        float z = -INFINITY;
        uint32_t word = 0;
        if (i < found) {
          z = (float)((const T*)loads)[i * kVec + e];
          const int at = places[i];
          word = (uint32_t)(at + e);
          if (at + e < skip + (few ? 0 : i * kVec)) z = -INFINITY;
        }
        const bool hit = z > bound || (z == bound && word <= last);
        const uint64_t lanes = __ballot(hit);
        if (hit) keys[n + below(lanes)] = key_of(z, word);
        n += __builtin_popcountll(lanes);
      }
    }
    cut();
  }
  sum = wave_sum(sum);
  const int64_t part = (int64_t)row * a.chunks + chunk;
  if (lane == 0) {
    a.parts[part].top = most;
    a.parts[part].sum = sum;
  }
  if (lane < count) {
    FxBeamWord none;
    none.x = -INFINITY;
    none.word = 0;
    a.lists[part * count + lane] = lane < n ? word_of(keys[lane]) : none;
  }
}

// Each wave has the lists of a row in LDS: [waves][chunks * count], and there are the rows' best [beams][count]
__global__ __launch_bounds__(1024) void fx_beam_join(const FxBeamArgs a) {
  extern __shared__ uint4 s_join[];
  const int count = a.count, K = a.beams, entries = a.chunks * count;
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), waves = (int)blockDim.x >> 6;
  double* score = (double*)s_join;                    // [beams][count]
  uint32_t* word = (uint32_t*)(score + K * count);    // [beams][count]
  FxBeamWord* mine = (FxBeamWord*)(word + ((K * count + 1) & ~1)) + (size_t)wave * entries;
  const int64_t request = blockIdx.x;
  for (int k = wave; k < K; k += waves) {
    const int64_t row = request * K + k;
    // (all loads at once: what beams with no candidates of their own have there is never looked at)
    const float before = a.scores[row];
    const bool over = a.ended && a.ended[row];
    const FxBeamPart p = lane < a.chunks ? a.parts[row * a.chunks + lane] : FxBeamPart{-INFINITY, 0.0f, 0.0};
    in_wave();
    for (int i = lane; i < entries; i += 64) mine[i] = a.lists[row * entries + i];
    in_wave();
    const bool live = before > -INFINITY;
    int n = 0;
    if (over) {
      if (lane == 0 && live) {
        score[k * count] = (double)before;
        word[k * count] = 0;   // (the end word, which need not be one of the vocabulary's)
      }
      n = live ? 1 : 0;
    } else if (live) {
      const float top = wave_max(p.top);
      const double most = (double)top;
      const double part = lse_of(p.top, p.sum);
      const double sum = wave_sum(part == -INFINITY ? 0.0 : exp(part - most));   // (NaN stays)
      const double lse = log(sum) + most;
      if (top > -INFINITY && lse - lse == 0.0) {   // (a row with NaN or +infinity has none)
        int at = 0;                                 // the lane's place in the list of its part
        float x = -INFINITY;
        uint32_t w = 0;
        const auto next = [&]() {
          x = -INFINITY;
          if (lane < a.chunks && at < count) {
            const FxBeamWord e = mine[lane * count + at];
            x = e.x;
            w = e.word;
          }
        };
        next();
        for (; n < count; ++n) {
          const float m = wave_max(x);
          if (!(m > -INFINITY)) break;
          const int first = __builtin_ctzll(__ballot(x == m));   // (parts are in the order of their words)
          if (lane == first) {
            score[k * count + n] = (double)before + ((double)x - lse);
            word[k * count + n] = w;
            ++at;
            next();
          }
        }
      }
    }
    for (int i = n + lane; i < count; i += 64) score[k * count + i] = -INFINITY;
  }
  __syncthreads();
  // the place of a candidate: how many are better, or as good and before it
  const int all = K * count;
  for (int i = (int)threadIdx.x; i < all; i += (int)blockDim.x) {
    const double s = score[i];
    if (!(s > -INFINITY)) continue;
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < all; ++j) {
      const double t = score[j];
      rank += t > s || (t == s && j < i) ? 1 : 0;
    }
    if (rank >= count) continue;
    const int k = i / count;
    const int64_t to = request * count + rank;
    a.out_scores[to] = (float)s;
    a.out_beams[to] = k;
    a.out_words[to] = a.ended && a.ended[request * K + k] ? a.end_word : (int64_t)word[i];
  }
  // places that are left
  if (wave == 0) {
    int there = 0;
    for (int i = lane; i < all; i += 64) there += score[i] > -INFINITY ? 1 : 0;
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

int chunks_of(const FxBeamArgs& a, int loads) {
  const int words = 64 * (a.dtype == FX_DT_F32 ? 4 : 8) * loads;
  return (a.words + words - 1) / words;
}
}  // namespace

void fx_beam_shape(FxBeamArgs& a) {
  // few rows: shorter parts; a row has no more of them than a wave of fx_beam_join has lanes
  a.loads = chunks_of(a, 4) <= 64 && (int64_t)a.requests * a.beams * chunks_of(a, 4) <= 8192 ? 4 : chunks_of(a, 8) <= 64 ? 8 : 16;
  a.chunks = chunks_of(a, a.loads);
}

hipError_t fx_launch_beam_select(const FxBeamArgs& a, hipStream_t stream, int* launched) {
  static const void* const scans[2][3] = {{(const void*)fx_beam_scan<float, 4>, (const void*)fx_beam_scan<_Float16, 4>, (const void*)fx_beam_scan<__bf16, 4>},
                                          {(const void*)fx_beam_scan<float, 8>, (const void*)fx_beam_scan<_Float16, 8>, (const void*)fx_beam_scan<__bf16, 8>}};
  // (16: 64 parts of 16-bit rows are 2^18 words with 8)
  const void* const scan = a.loads == 16 ? (const void*)fx_beam_scan<float, 16> : scans[a.loads == 8][a.dtype == FX_DT_F32 ? 0 : a.dtype == FX_DT_F16 ? 1 : 2];
  FxBeamArgs args = a;
  void* kargs[1] = {(void*)&args};
  const int64_t units = (int64_t)a.requests * a.beams * a.chunks;
  *launched = 0;
  const hipError_t e = hipLaunchKernel(scan, dim3((unsigned)((units + kWaves - 1) / kWaves)), dim3(kThreads), kargs, 0, stream);
  if (e != hipSuccess) return e;
  *launched = 1;
  // (64 KiB of LDS a workgroup: at most 32 * 64 candidates of 12 bytes, and one row's lists of 64 * 64 words of 8)
  const size_t rows = (size_t)a.beams * a.count * 12 + 8, lists = (size_t)a.chunks * a.count * sizeof(FxBeamWord);
  const int waves = std::max(1, std::min(std::min(a.beams, 16), (int)((65536 - rows) / lists)));
  const hipError_t f = hipLaunchKernel((const void*)fx_beam_join, dim3((unsigned)a.requests), dim3((unsigned)waves * 64), kargs, rows + (size_t)waves * lists, stream);
  if (f == hipSuccess) *launched = 2;
  return f;
}
