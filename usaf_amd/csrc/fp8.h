// What the 8-bit block-scaled kernels share (fp8.hip, fp8_gemm.hip, few.hip).
#pragma once

#include "moe_gemm.h"

namespace usaf {

constexpr int FP8_BLOCK = 128;  // values of one scale along a row; rows of one scale of a weight

}  // namespace usaf
