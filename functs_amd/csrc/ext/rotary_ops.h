// Arguments of rotary positions, which functs::rotary and functs::kv_append share.
#pragma once
#include "op_checks.h"

namespace functs {
// positions' and frequencies' part of a descriptor, checked against a head's depth
fx_rotary_desc rotaryDesc(const char* op, const Tensor& positions, const Tensor& frequencies, double magnitude, bool interleaved, int64_t depth, c10::Device dev);
}  // namespace functs
