// resnorm.h — norms after and before a block, fused with its gate and the residual sum (kernels in resnorm.hip).
#pragma once
#include <hip/hip_runtime.h>

#include "../../include/anneal_hip.h"

namespace ah {

// Enqueues the operators on s. Descriptors must have been checked.
hipError_t residual_norm(const ah_residual_norm_desc &d, hipStream_t s);
// Bytes of workspace that residual_norm_grad needs for d (16-byte aligned, contents of no matter).
int64_t residual_norm_grad_workspace(const ah_residual_norm_grad_desc &d);
hipError_t residual_norm_grad(const ah_residual_norm_grad_desc &d, hipStream_t s);

}  // namespace ah
