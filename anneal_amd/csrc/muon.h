// muon.h — orthogonalised updates: Newton-Schulz iteration and the weight step built on it (kernels in muon.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ah {

struct Muon {
    int f16;                    // G: f16, else f32
    int rows, cols, batch;
    const void *G;
    long ldg, sg;               // elements from row to row and from matrix to matrix
    int steps;
    float a, b, c, eps;
    // orthogonalise alone: O = NS(G); out16: O is f16
    void *O;
    long ldo, so;
    int out16;
    // weight step (W set): M_out = momentum M + G; U = nesterov ? G + momentum M_out : M_out;
    // W_out = (1 - lr decay) W - lr scale NS(U); W16_out = f16(W_out)
    const float *M;
    float *M_out;
    const float *W;
    float *W_out;
    void *W16_out;
    long ldw, sw;               // of M, W and their outputs
    float lr, momentum, decay, scale;
    int nesterov;
};

int64_t muon_workspace(const Muon &d);
// Enqueues the operator on s. d must have been checked.
hipError_t muon(const Muon &d, void *ws, hipStream_t s);

}  // namespace ah
