// linattn_chain.hip -- the states before each segment of a cut sequence.
#include "linattn.h"

namespace ssla {
namespace {

// ws_state holds each segment's own state L_j (from zero) and decay A_j; the
// state before segment j + 1 is A_j X_j + L_j, from X_0 = the sequence's
// initial state.  Every thread runs the chain of one state value in order and
// leaves X_j in L_j's place.
__global__ __launch_bounds__(256) void k_linattn_chain(const LinAttnArgs a) {
    const int per = a.dk * a.dv, wide = (per + 255) / 256;
    const int sh = blockIdx.x / wide, i = (blockIdx.x - sh * wide) * 256 + threadIdx.x;
    const int seq = sh / a.heads, head = sh - seq * a.heads;
    int j, n;
    if (a.cu) {
#ifdef __HIP_DEVICE_COMPILE__
        const long long first = linattn_first(a, seq);
        const long long len = linattn_first(a, seq + 1) - first;
        const int l = (int)(len < 0 ? 0 : len > a.max_len ? a.max_len : len);
        j = (int)(first >> a.seg_shift) + seq;
        n = (int)(((unsigned)l + (1u << a.seg_shift) - 1) >> a.seg_shift);
#endif
    } else {
        n = a.n_segs / a.n_seqs;
        j = seq * n;
    }
    const int slot = linattn_slot(a, seq);
    if (slot < 0 || n < 2 || i >= per) return;
    float* w = a.ws_state + ((long long)j * a.heads + head) * per + i;
    const float* d = a.ws_decay + (long long)j * a.heads + head;
    const long long step = (long long)a.heads * per;
    float x = a.s_in ? a.s_in[(long long)slot * a.s_stride + (long long)head * per + i] : 0.0f;
    constexpr int U = 8;                       // loads in flight ahead of the chain
    for (int k0 = 0; k0 < n; k0 += U) {
        float own[U], dec[U];
        #pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool in = k0 + u < n - 1;
            own[u] = in ? w[(k0 + u) * step] : 0.0f;
            dec[u] = in ? d[(long long)(k0 + u) * a.heads] : 0.0f;
        }
        #pragma unroll
        for (int u = 0; u < U; ++u)
            if (k0 + u < n) {
                w[(k0 + u) * step] = x;
                x = fmaf(dec[u], x, own[u]);
            }
    }
}

}  // namespace

hipError_t linattn_launch_chain(const LinAttnArgs& a, hipStream_t st) {
    LinAttnArgs args = a;
    void* pa[] = {&args};
    const long long blocks = (long long)((a.dk * a.dv + 255) / 256) * a.n_seqs * a.heads;
    return hipLaunchKernel((const void*)k_linattn_chain, dim3((unsigned)blocks), dim3(256), pa, 0, st);
}

}  // namespace ssla
