// linear_ce.h — softmax cross-entropy of a linear head, its logits in pieces of rows (kernels in linear_ce.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ah {

struct LinearCe {
    int f16;         // operands X, W, bias: f16, else f32
    int g16;         // gradients: f16, else f32
    int N, D, V;
    const void *X, *W, *bias;   // [N,D], [V,D], [V] or null
    long ldx, ldw;
    const int *labels;          // [N]; outside [0, V): the row does not count
    float *loss;                // [1]
    float *rowloss, *lse;       // [N] or null
    void *dX, *dW;              // [N,D], [V,D] or null
    long lddx, lddw;
    float *dbias;               // [V] or null
    float grad_scale;
    int piece_mb;               // MiB of kept logits (of statistics, for the loss alone), at most (0: 2048)
    int mean;                   // divide loss and gradients by the number of counted rows
};

// Bytes of workspace that linear_ce needs for d (16-byte aligned, contents of no matter).
int64_t linear_ce_workspace(const LinearCe &d);
// Enqueues the operator on s. d must have been checked (shapes positive, pointers set, strides at least a row).
hipError_t linear_ce(const LinearCe &d, void *ws, hipStream_t s);

}  // namespace ah
