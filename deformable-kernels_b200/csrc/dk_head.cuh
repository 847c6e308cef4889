// The last linear layer of a classifier with its softmax cross entropy: what dk_head.cu (plans, small kernels, the general
// kernels) and the tensor-core kernels share.
#pragma once

#include <cuda_bf16.h>

#include "dk_common.cuh"

namespace dk {
namespace head {

constexpr double kLog2e = 1.4426950408889634074, kLn2 = 0.69314718055994530942;

}  // namespace head
}  // namespace dk
