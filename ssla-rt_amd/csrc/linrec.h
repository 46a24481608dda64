// linrec.h -- the gated linear recurrence: what the C ABI (ops_train.cpp) hands
// to the kernels (linrec.hip, linrec_step.hip), and how work is cut into them.
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
    // how the call is cut (linrec_plan)
    int vec;                              // channels of a thread
    int cols, blocks;                     // threads along the channels; workgroups along them
    int lanes, tile, tiles;               // threads along the tokens, their tokens, tiles of all tokens
    unsigned* tickets;                    // workspace: a counter for each block of channels
    unsigned long long* words;            // [place in the chain][block][cols * vec] maps and states
};

constexpr int kLinRecThreads = 256;
constexpr int kTicketStep = 32;           // counters lie 128 bytes apart

void linrec_plan(LinRecArgs& a, int dtype);
// Workspace: 0 where one tile holds all tokens.
inline size_t linrec_words(const LinRecArgs& a) {
    return a.tiles > 1 ? (size_t)a.tiles * a.blocks * a.cols * a.vec : 0;
}
inline size_t linrec_bytes(const LinRecArgs& a) {
    return a.tiles > 1 ? linrec_words(a) * 8 + (size_t)a.blocks * kTicketStep * 4 : 0;
}
hipError_t linrec_launch(const LinRecArgs& a, int dtype, hipStream_t st);
hipError_t linrec_launch_backward(const LinRecArgs& a, int dtype, hipStream_t st);
hipError_t linrec_launch_step(const LinRecArgs& a, int dtype, hipStream_t st);

#ifdef __HIPCC__
// A gate a = sigmoid(x) as one float c: the smaller of a and 1 - a, s = sigmoid(-|x|),
// to a few roundings of itself, negative where it is 1 - a (x > 0).  An open gate
// keeps the digits of what it forgets, a closed one those of what it lets through.
__device__ __forceinline__ float gate_of(float x) {
    const float e = __expf(-fabsf(x));
    return __builtin_copysignf(e * __builtin_amdgcn_rcpf(1.0f + e), -x);
}
// a h, of such a c: h - s h, or s h.
__device__ __forceinline__ float through(float c, float h) {
    return fmaf(c, h, __builtin_signbit(c) ? h : 0.0f);
}
// a (1 - a)
__device__ __forceinline__ float slope_of(float c) {
    const float s = fabsf(c);
    return fmaf(-s, s, s);
}

__device__ __forceinline__ int linrec_slot(const LinRecArgs& a, int seq) {
    if (seq < 0 || seq >= a.n_seqs) return -1;
    const int s = a.slots ? a.slots[seq] : seq;
    return s < 0 || s >= a.n_slots ? -1 : s;
}
#endif

}  // namespace ssla
