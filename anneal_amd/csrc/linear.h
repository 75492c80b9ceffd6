// linear.h — linear layers with bias, activation, factor and residual (kernels in linear.hip), and their gradients (linear_grad.hip).
#pragma once
#include <hip/hip_runtime.h>

#include "../../include/anneal_hip.h"

namespace ah {

// Bytes of workspace that the calls need for d (16-byte aligned, contents of no matter).
int64_t linear_workspace(const ah_linear_desc &d);
int64_t linear_grad_workspace(const ah_linear_grad_desc &d);
// Enqueue the operators on s. Descriptors must have been checked.
hipError_t linear(const ah_linear_desc &d, hipStream_t s);
hipError_t linear_grad(const ah_linear_grad_desc &d, hipStream_t s);

}  // namespace ah
