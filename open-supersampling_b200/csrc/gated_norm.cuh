// Parameters of the gated residual norm's kernels (gated_norm.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace oss {

struct GatedNorm {
    int64_t rows;
    int c;
    float inv_c, eps;
    int layer;      // 1: mean and variance, 0: mean of squares
    int gate_kind;  // 0 none, 1 one a row, 2 one an element
    int act;        // 0 none, 1 sigmoid, 2 silu
    int param_type; // 0 fp32, 1 bf16, 2 fp16
    const void *x, *h, *gate;
    int64_t x_st, h_st, g_st;  // row strides in elements
    const void *weight, *bias, *scale, *next_weight, *next_bias;
    void *y, *z;     // contiguous; z null: no second norm
    float4* stats;   // [rows] mean, 1 / deviation of h and of y; forward: may be null
    const void *dy, *dz;
    int64_t dy_st, dz_st;
    void *dx, *dh, *dgate;  // contiguous, each may be null
    float* partial;         // [5][parts][c]
    void* dparam[5];        // weight, scale, next_weight, bias, next_bias; each may be null
};

int64_t gated_norm_partial_floats(int64_t rows, int c);
cudaError_t launch_gated_norm_forward(const GatedNorm& p, int type, cudaStream_t s);
cudaError_t launch_gated_norm_backward(const GatedNorm& p, int type, cudaStream_t s);

}  // namespace oss
