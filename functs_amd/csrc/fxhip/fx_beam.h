// A beam search's selection: arguments of its kernels (fx_beam.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../../include/fxhip.h"

// What a wave finds in its part of a row: the largest logit, the sum of 2^(x c - r) (NaN where there is one in the part), and in a list of its own
// the best `count` (x, word), best first
struct FxBeamPart {
  float top;
  float unused;
  double sum;
};
struct FxBeamWord {
  float x;        // -infinity: none
  uint32_t word;
};
struct FxBeamArgs {
  const void* logits;                  // [requests][beams][words], a beam's words side by side
  int64_t l_request, l_beam;           // elements
  const float* scores;                 // [requests][beams]
  const uint8_t* ended;                // [requests][beams], or null
  float* out_scores;                   // [requests][count]
  int32_t* out_beams;
  int64_t* out_words;
  int64_t end_word;
  FxBeamPart* parts;                   // [requests * beams][chunks]
  FxBeamWord* lists;                   // [requests * beams][chunks][count]
  int32_t requests, beams, words, count, dtype, chunks, loads;   // loads: of 16 bytes that a lane has under way
};
void fx_beam_shape(FxBeamArgs& a);     // chunks and loads
hipError_t fx_launch_beam_select(const FxBeamArgs& a, hipStream_t stream, int* launched);
