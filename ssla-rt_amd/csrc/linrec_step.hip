// linrec_step.hip -- the gated linear recurrence for one token of every sequence.
//
// Each state is read and written once, with a few operations a value: bound by
// memory (8000 sequences of 2048 bf16 channels: 38.4 us, 6.0 TB/s, states and all once),
// and by its launch where there are few (one sequence: 1.9 us in a graph).  A thread owns 16 bytes
// of a row's values (what is left over at a row's end goes by single values).
#include "linrec.h"

namespace ssla {
namespace {

constexpr int NT = kLinRecThreads;

template <class T, int V>
__global__ __launch_bounds__(NT) void k_linrec_step(const LinRecArgs a) {
    const int per = (a.channels + V - 1) / V;                // pieces of a row
    const long long id = (long long)blockIdx.x * NT + threadIdx.x;
    const int seq = (int)(id / per), c = (int)(id - (long long)seq * per) * V;
    const int slot = linrec_slot(a, seq);
    if (slot < 0) return;
    const T* g = (const T*)a.g + seq * a.gt + c;
    const T* v = (const T*)a.v + seq * a.vt + c;
    const T* q = a.q ? (const T*)a.q + seq * a.qt + c : nullptr;
    T* out = (T*)a.out + seq * a.ot + c;
    const float* from = a.s_in + slot * a.si + c;
    float* to = a.s_out + slot * a.so + c;
    if (c + V <= a.channels) {
        T pg[V], pv[V], pq[V];
        float h[V];
        __builtin_memcpy(h, from, sizeof(h));
        __builtin_memcpy(pg, g, sizeof(pg));
        __builtin_memcpy(pv, v, sizeof(pv));
        if (q) __builtin_memcpy(pq, q, sizeof(pq));
        #pragma unroll
        for (int i = 0; i < V; ++i) {
            h[i] = fmaf(gate_of((float)pg[i]).a, h[i], (float)pv[i]);
            pv[i] = (T)(q ? (float)pq[i] * h[i] : h[i]);
        }
        __builtin_memcpy(to, h, sizeof(h));
        __builtin_memcpy(out, pv, sizeof(pv));
    } else {
        for (int i = 0; i < a.channels - c; ++i) {
            const float h = fmaf(gate_of((float)g[i]).a, from[i], (float)v[i]);
            to[i] = h;
            out[i] = (T)(q ? (float)q[i] * h : h);
        }
    }
}

template <class T>
hipError_t launch(const LinRecArgs& a, hipStream_t st) {
    constexpr int V = 16 / sizeof(T);
    // One value a thread as long as the card holds all of them at once, 2048 a compute unit (us, so
    // and with 16 bytes: 1 x 2048 bf16 2.05 and 2.32, 32 x 2048 2.18 and 2.53, 128 x 2048 2.59 and
    // 2.73, 19200 x 96 fp32 7.99 and 6.35).
    const bool wide = (long long)a.n_seqs * a.channels > 256 * 2048;
    const long long n = (long long)a.n_seqs * ((a.channels + (wide ? V : 1) - 1) / (wide ? V : 1));
    LinRecArgs args = a;
    void* pa[] = {&args};
    return hipLaunchKernel(wide ? (const void*)k_linrec_step<T, V> : (const void*)k_linrec_step<T, 1>,
                           dim3((unsigned)((n + NT - 1) / NT)), dim3(NT), pa, 0, st);
}

}  // namespace

hipError_t linrec_launch_step(const LinRecArgs& a, int dtype, hipStream_t st) {
    if (dtype == SSLA_F32) return launch<float>(a, st);
    if (dtype == SSLA_BF16) return launch<__bf16>(a, st);
    return launch<_Float16>(a, st);
}

}  // namespace ssla
