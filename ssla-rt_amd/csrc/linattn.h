// linattn.h -- linear attention with a decay for each head: what the C ABI
// (ops.cpp) hands to the kernels, and how work is cut into them.
//
//   S_t = exp(g_t) S_{t-1} + k_t v_t^T,     o_t = scale q_t^T S_t     (S: dk x dv)
//
// A workgroup runs one segment of one sequence for one head and one slice of
// the dv columns, chunk by chunk with the state in registers
// (linattn_kernel.h).  Sequences longer than a segment take three launches: the
// segments' own states from zero (FULL = false), the states before each
// segment (k_linattn_chain), then every segment from its state (FULL = true).
#pragma once

#include <hip/hip_runtime.h>

#include "ssla_hip.h"

namespace ssla {

constexpr int kLinAttnMaxDim = 256;      // dk, dv
constexpr int kCUs = 256;                 // compute units
constexpr float kMinLogDecay = -65536.0f;

struct LinAttnArgs {
    const void *q, *k, *v;
    void* out;
    const float* g;                       // log decay
    long long qt, qh, kt, kh, vt, vh, ot, oh, gt, gh;   // strides, elements: token, head
    const int* cu;                        // first token of each sequence, or null
    const int* slots;                     // state slot of each sequence, or null
    const float* s_in;
    float* s_out;
    long long s_stride;                   // floats between slots
    float* ws_state;                      // [state][head][dk][dv], of the segments of cut sequences
    float* ws_decay;                      // [state][head]
    long long n_tokens;
    int n_seqs, n_slots, max_len;
    int heads, rep, dk, dv, slices;       // rep: heads sharing q and k
    int seg_shift, n_segs;                // log2 of a segment's tokens; segments of the call
    int n_states, paired;                 // states of the workspace; where they lie: linattn_states
    int by_length;                        // whole sequences of unlike lengths: see linattn_by_length
    int vec;                              // buffer loads of q, k, v and stores of out, in pieces
    float scale;
};

// Where a segment lies: sequence `seq`, tokens [t0, t1) of its `len`, which
// begin at row `row`.  Segment slots of sequence s begin at
// (cu[s] >> seg_shift) + s: as many as it can need whatever the lengths, so
// the grid needs only the number of tokens and sequences.  Its state is `state` of
// the workspace, where the sequence is cut.
struct Segment {
    long long row;
    int seq, index, state, t0, t1, len;
    bool ok;
};

#ifdef __HIP_DEVICE_COMPILE__
__device__ __forceinline__ long long linattn_first(const LinAttnArgs& a, int s) {
    const long long c = a.cu[s];
    return c < 0 ? 0 : c > a.n_tokens ? a.n_tokens : c;
}

// Place in the workspace of the first state of a sequence that begins at token
// `first`: its first segment slot; or (paired) twice the whole segments' lengths of
// tokens before it.  Only sequences of n > 1 segments have states there, and the
// next one begins at least n / 2 such lengths later, so that 2 (n_tokens >> shift)
// states do, however many sequences there are: 511 sequences of a token beside one of
// 4000 (16 heads of 128, segments of 256) take 36 MB instead of 555.
__device__ __forceinline__ int linattn_states(const LinAttnArgs& a, long long first, int seq) {
    const int piece = (int)(first >> a.seg_shift);
    return a.paired ? 2 * piece : piece + seq;
}

// Whole sequences (up to 64) of unlike lengths: the longest first, and every
// second round of the compute units in the other direction, so that those
// that share a compute unit are not all long.  48 sequences of 340 to 1531 tokens
// with 16 heads of 64, lengths repeating every 8: 166 -> 121 us.
__device__ __forceinline__ int linattn_by_length(const LinAttnArgs& a, int j, int lane) {
    const int n = a.n_seqs, per = a.heads * a.slices;
    int len = 0;
    if (lane < n) len = (int)(linattn_first(a, lane + 1) - linattn_first(a, lane));
    int rank = 0;
    for (int t = 0; t < n; ++t) {
        const int other = __builtin_amdgcn_readlane(len, t);
        rank += other > len || (other == len && t < lane);
    }
    const int round = per < kCUs ? kCUs / per : 1, r = j / round, end = min(n, (r + 1) * round);
    const int want = r & 1 ? end - 1 - (j - r * round) : j;
    return __ffsll((unsigned long long)__ballot(lane < n && rank == want)) - 1;
}
#endif

__device__ __forceinline__ Segment linattn_segment(const LinAttnArgs& a, int j, int lane) {
    Segment g;
#ifdef __HIP_DEVICE_COMPILE__
    long long len;
    if (a.by_length) {
        g.seq = linattn_by_length(a, j, lane);
        g.row = linattn_first(a, g.seq);
        len = linattn_first(a, g.seq + 1) - g.row;
        g.index = g.state = 0;
    } else if (a.cu) {
        // the last sequence whose first slot is at or before j, 64 candidates a round
        int lo = 0, n = a.n_seqs;
        while (n > 1) {
            const int step = (n + 63) >> 6;
            const int s = lo + lane * step;
            const bool in = lane * step < n &&
                            (linattn_first(a, s < a.n_seqs ? s : a.n_seqs) >> a.seg_shift) + s <= j;
            const int hits = __popcll(__ballot(in));
            const int at = hits ? hits - 1 : 0;
            lo += at * step;
            n = min(step, n - at * step);
        }
        g.seq = __builtin_amdgcn_readfirstlane(lo);
        g.row = linattn_first(a, g.seq);
        len = linattn_first(a, g.seq + 1) - g.row;
        g.index = j - (int)((g.row >> a.seg_shift) + g.seq);
        g.state = linattn_states(a, g.row, g.seq) + g.index;
    } else {
        const int per = a.n_segs / a.n_seqs;
        g.seq = j / per;
        g.index = j - g.seq * per;
        g.state = j;
        len = a.max_len;
        g.row = (long long)g.seq * a.max_len;
    }
    g.len = (int)(len < 0 ? 0 : len > a.max_len ? a.max_len : len);
    const long long t0 = (long long)g.index << a.seg_shift;
    const long long t1 = t0 + (1ll << a.seg_shift);
    g.ok = g.index >= 0 && (t0 < g.len || g.index == 0);
    g.t0 = g.ok ? (int)t0 : 0;
    g.t1 = t1 < g.len ? (int)t1 : g.len;
#endif
    return g;
}

// The state slot of a sequence, or -1: its slot is no slot of the pool, and
// the sequence is passed over.
__device__ __forceinline__ int linattn_slot(const LinAttnArgs& a, int seq) {
    if (!a.slots) return seq;
    const int s = a.slots[seq];
    return s >= 0 && s < a.n_slots ? s : -1;
}

// Launchers, one object file each.  `full`: outputs and final states, else
// the segments' own states.  hipError_t of the launch.
hipError_t linattn_launch_bf16(const LinAttnArgs& a, bool full, hipStream_t st);
hipError_t linattn_launch_f16(const LinAttnArgs& a, bool full, hipStream_t st);
hipError_t linattn_launch_f32(const LinAttnArgs& a, bool full, hipStream_t st);
hipError_t linattn_launch_chain(const LinAttnArgs& a, hipStream_t st);
hipError_t linattn_launch_step(const LinAttnArgs& a, int dtype, hipStream_t st);

// Waves of a workgroup: each owns 16 columns of out, and all of a head's columns
// share one reading of q and k where eight waves' are enough; idle waves cost more
// than that (16 sequences of 2000 tokens: bf16, 16 heads of 64, four waves 104 us,
// eight 136; fp32, 4 heads of 96, six 92, eight 99, four twice 136; bf16, 16 heads of
// 128, eight 173, four twice 185).
inline int linattn_waves(int dk, int dv) { return dk > 128 || dv <= 64 ? 4 : dv <= 96 ? 6 : 8; }

// Launches a chunked kernel with `lds` bytes.  More than 64 KB of LDS has to be
// asked for; the attribute is the function's, and setting it again costs a lookup.
inline hipError_t linattn_launch(const void* f, const LinAttnArgs& a, int waves, size_t lds, hipStream_t st) {
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    LinAttnArgs args = a;
    void* pa[] = {&args};
    const long long blocks = (long long)a.n_segs * a.heads * a.slices;
    return hipLaunchKernel(f, dim3((unsigned)blocks), dim3(64 * waves), pa, lds, st);
}

}  // namespace ssla
