// layernorm.h -- layer norm: what the C ABI (ops_train.cpp) hands to the kernels
// (layernorm.hip).
//
//   y = (s - mean) / sqrt(var + eps) * w + b,   s = x + residual
#pragma once

#include <hip/hip_runtime.h>

#include "ssla_hip.h"

namespace ssla {

struct LayerNormArgs {
    const void *x, *res, *weight, *bias;
    void* out;
    float* stats;                         // [row] mean (two floats) and scale
    long long xr, rr, orow;               // strides between rows, elements
    // backward
    const void* dout;
    void *dx, *dw, *db;
    long long dor, dxr;
    float* ws;                            // [part][2][channels] partial sums of dw and db
    int rows, channels;
    int wide;                             // weight, bias and their gradients are fp32
    float eps;
    double inv_channels;
    // how the call is cut (layer_norm_plan)
    int vec, reps;                        // channels of a piece; pieces a thread keeps (0: rows in strides)
    int lanes;                            // threads of a row (over 64: a workgroup)
    int threads, wgs;
    int parts;                            // of the rows, for the sums over them
};

void layer_norm_plan(LayerNormArgs& a, int dtype, bool backward);
hipError_t layer_norm_launch(const LayerNormArgs& a, int dtype, hipStream_t st);
hipError_t layer_norm_launch_backward(const LayerNormArgs& a, int dtype, hipStream_t st);

}  // namespace ssla
