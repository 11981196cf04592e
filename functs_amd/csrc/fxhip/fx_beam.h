// A beam search's selection: arguments of its kernels (fx_beam.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../../include/fxhip.h"

#define FX_BEAM_SEGMENTS 8   // of a wave's words: what 16 lanes have loaded in two neighbouring loads
// What a wave finds in its words: the largest logit and the sum of 2^(x c - r) (NaN where there is one)
struct FxBeamPart {
  float top;
  float unused;
  double sum;
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
  FxBeamPart* parts;                   // [requests * beams][parts_a_row]
  int32_t* tops;                       // [requests * beams][parts_a_row][FX_BEAM_SEGMENTS]: the largest of each segment, as a whole number in the order of floats
  int32_t requests, beams, words, count, dtype, parts_a_row;
};
void fx_beam_shape(FxBeamArgs& a);     // parts_a_row
hipError_t fx_launch_beam_select(const FxBeamArgs& a, hipStream_t stream, int* launched);
