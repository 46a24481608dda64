// linattn_chain.hip -- the states before each segment of a cut sequence.
#include "linattn.h"

namespace ssla {
namespace {

// ws_state holds each segment's own state L_j (from zero) and decay A_j; the
// state before segment j + 1 is A_j X_j + L_j, from X_0 = the sequence's
// initial state.  Every thread runs the chain of W neighbouring state values in
// order and leaves X_j in L_j's place.  X_0 too: the next launch writes final
// states to s_out, which may be s_in, so none of its segments may read a cut
// sequence's s_in.
// Bound by the states' traffic, each read and written once: 32 segments of 16
// heads of 128 x 128, 65 MB, take 12.8 us (13.4 with W = 1).
template <int W>
__global__ __launch_bounds__(256) void k_linattn_chain(const LinAttnArgs a) {
    const int per = a.dk * a.dv, wide = (per + 256 * W - 1) / (256 * W);
    const int sh = blockIdx.x / wide, i = (blockIdx.x - sh * wide) * 256 * W + threadIdx.x * W;
    const int seq = sh / a.heads, head = sh - seq * a.heads;
    int j, n;
    if (a.cu) {
#ifdef __HIP_DEVICE_COMPILE__
        const long long first = linattn_first(a, seq);
        const long long len = linattn_first(a, seq + 1) - first;
        const int l = (int)(len < 0 ? 0 : len > a.max_len ? a.max_len : len);
        j = linattn_states(a, first, seq);
        n = (int)(((unsigned)l + (1u << a.seg_shift) - 1) >> a.seg_shift);
#endif
    } else {
        n = a.n_segs / a.n_seqs;
        j = seq * n;
    }
    const int slot = linattn_slot(a, seq);
    if (slot < 0 || n < 2 || i >= per) return;
    typedef float vec __attribute__((ext_vector_type(W)));
    vec* w = (vec*)(a.ws_state + ((long long)j * a.heads + head) * per + i);
    const float* d = a.ws_decay + (long long)j * a.heads + head;
    const long long step = (long long)a.heads * per / W;
    vec x = {};
    if (a.s_in) x = *(const vec*)(a.s_in + (long long)slot * a.s_stride + (long long)head * per + i);
    constexpr int U = 8;                       // loads in flight ahead of the chain
    for (int k0 = 0; k0 < n - 1; k0 += U) {
        vec own[U];
        float dec[U];
        #pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = min(k0 + u, n - 2);
            own[u] = w[k * step];
            dec[u] = d[(long long)k * a.heads];
        }
        #pragma unroll
        for (int u = 0; u < U; ++u)
            if (k0 + u < n - 1) {
                w[(k0 + u) * step] = x;
                x = dec[u] * x + own[u];
            }
    }
    w[(n - 1) * step] = x;
}

}  // namespace

hipError_t linattn_launch_chain(const LinAttnArgs& a, hipStream_t st) {
    const bool wide = a.dk * a.dv % 4 == 0 && a.s_stride % 4 == 0 && (size_t)a.s_in % 16 == 0;
    LinAttnArgs args = a;
    void* pa[] = {&args};
    const int per = wide ? 1024 : 256;                   // state values of a workgroup
    const long long blocks = (long long)((a.dk * a.dv + per - 1) / per) * a.n_seqs * a.heads;
    return hipLaunchKernel(wide ? (const void*)k_linattn_chain<4> : (const void*)k_linattn_chain<1>,
                           dim3((unsigned)blocks), dim3(256), pa, 0, st);
}

}  // namespace ssla
