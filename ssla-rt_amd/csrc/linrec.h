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
    float* carries;                       // [token / carry][channels] states before every carry-th token
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
    unsigned per_col;                     // 2^16 / cols, rounded up: exact for a workgroup's threads
    int lanes, tile, tiles;               // threads along the tokens, their tokens, tiles of all tokens
    int carry;                            // tokens of a tile of the backward pass
    int brief;                            // a thread a channel, without tiles
    unsigned patience;                    // ticks of 10 ns that a workgroup waits for another
    int alone;                            // tiles start with the last, and publish nothing of their own
    unsigned long long* words;            // workspace: [block][kBehind + place in the chain][kChannels] maps and states
    // forward, where the last states take the first ones' place (else null): the first state of the
    // sequence that a tile's last token belongs to, and which that is (-1: it has none)
    float* firsts;                        // workspace: [tile][channels]
    int* cut;                             // workspace: [tile]
};

constexpr int kLinRecThreads = 256;
constexpr int kChannels = 64;             // most of a workgroup
constexpr int kBehind = 32;               // places before a chain's first one, never published

// Sequences of len tokens each that begin before token t.
constexpr int linrec_begun(int t, int len) { return t ? (t - 1) / len + 1 : 0; }

void linrec_plan(LinRecArgs& a, int dtype, bool backward);
inline int linrec_threads(const LinRecArgs& a) { return (a.cols * a.lanes + 63) / 64 * 64; }
// Workspace: 0 where one tile holds all tokens.
inline size_t linrec_words(const LinRecArgs& a) {
    return a.tiles > 1 ? ((size_t)a.tiles + kBehind) * a.blocks * kChannels : 0;
}
inline size_t linrec_firsts(const LinRecArgs& a) {
    return a.tiles > 1 ? (size_t)a.tiles * a.channels : 0;
}
// Of the forward pass: with firsts and cut, wherever the states are.
inline size_t linrec_bytes(const LinRecArgs& a, bool backward) {
    return linrec_words(a) * 8 + (backward || a.tiles < 2 ? 0 : (linrec_firsts(a) + a.tiles) * 4);
}
inline void linrec_bind(LinRecArgs& a, void* workspace) {
    a.words = (unsigned long long*)workspace;
    if (a.tiles < 2 || !a.s_in || a.s_in != a.s_out) return;
    a.firsts = (float*)(a.words + linrec_words(a));
    a.cut = (int*)(a.firsts + linrec_firsts(a));
}
inline size_t linrec_carries(const LinRecArgs& a) {
    return (size_t)((a.n_tokens + a.carry - 1) / a.carry) * a.channels * 4;
}
hipError_t linrec_launch(const LinRecArgs& a, int dtype, hipStream_t st);
hipError_t linrec_launch_backward(const LinRecArgs& a, int dtype, hipStream_t st);
hipError_t linrec_launch_step(const LinRecArgs& a, int dtype, hipStream_t st);

#ifdef __HIPCC__
// A gate a = sigmoid(x), rounded once from 1 - s where x > 0, and its slope a (1 - a) =
// s (1 - s), with s = sigmoid(-|x|): 1 - a would have none of a gate's digits that is
// nearly open.  s is off by some ten roundings of itself, and by up to |x| more: the
// exponential's argument is rounded, which counts where a gate is nearly shut.
struct Gate {
    float a, slope;
};
__device__ __forceinline__ Gate gate_of(float x) {
    #pragma clang fp contract(off)
    const float e = __builtin_amdgcn_exp2f(-1.44269504f * fabsf(x));
    const float s = e * __builtin_amdgcn_rcpf(1.0f + e);
    return Gate{x > 0.0f ? 1.0f - s : s, fmaf(-s, s, s)};
}

__device__ __forceinline__ int linrec_slot(const LinRecArgs& a, int seq) {
    if (seq < 0 || seq >= a.n_seqs) return -1;
    const int s = a.slots ? a.slots[seq] : seq;
    return s < 0 || s >= a.n_slots ? -1 : s;
}
#endif

}  // namespace ssla
