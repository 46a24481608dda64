// linrec.h -- the gated linear recurrence: what the C ABI (ops_train.cpp) hands
// to the kernels (linrec.hip), and how work is cut into them.
//
//   h_t = sigmoid(g_t) h_{t-1} + v_t,    o_t = q_t h_t       per channel
#pragma once

#include <hip/hip_runtime.h>

#include "ssla_hip.h"

namespace ssla {

struct LinRecArgs {
    const void *g, *v, *q;
    void* out;
    long long gt, vt, qt, ot;             // strides between tokens, elements
    const int* cu;                        // first token of each sequence, or null
    const int* slots;                     // state slot of each sequence, or null
    const float* s_in;
    float* s_out;
    long long si, so;                     // floats between slots
    float* carries;                       // [tile][channels] states before a tile's first token
    // backward
    const void* dout;
    const float* ds_out;
    void *dg, *dv, *dq;
    float* ds_in;
    long long dot, dgt, dvt, dqt, dso, dsi;
    long long n_tokens;
    int n_seqs, n_slots, channels;
    int seq_len;                          // without cu
    int tiles;                            // of `tile` tokens
    int tile;
};

void linrec_plan(LinRecArgs& a, int dtype);
hipError_t linrec_launch(const LinRecArgs& a, int dtype, hipStream_t st);
hipError_t linrec_launch_backward(const LinRecArgs& a, int dtype, hipStream_t st);
hipError_t linrec_launch_step(const LinRecArgs& a, int dtype, hipStream_t st);

}  // namespace ssla
