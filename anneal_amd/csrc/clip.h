// clip.h — the global norm of many tensors, and clipping by it (kernels in clip.hip).
#pragma once
#include <hip/hip_runtime.h>

#include "../../include/anneal_hip.h"

namespace ah {

// Bytes of workspace that clip_norm needs for d (16-byte aligned, contents of no matter).
int64_t clip_workspace(const ah_clip_desc &d);
// Enqueues the operator on s. d must have been checked.
hipError_t clip_norm(const ah_clip_desc &d, hipStream_t s);

}  // namespace ah
