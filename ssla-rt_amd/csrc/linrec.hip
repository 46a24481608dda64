// linrec.hip -- the gated linear recurrence, its gradients, and its single
// tokens.  One thread a channel of a sequence, token by token.
#include "linrec.h"

namespace ssla {
namespace {

constexpr int NT = 256;
constexpr int TILE = 64;

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

struct Range {
    long long t0, t1;
};
__device__ __forceinline__ Range range_of(const LinRecArgs& a, int seq) {
    if (!a.cu) return Range{(long long)seq * a.seq_len, (long long)(seq + 1) * a.seq_len};
    const long long lo = max(a.cu[seq], 0), hi = max(a.cu[seq + 1], 0);
    return Range{min(lo, a.n_tokens), min(hi, a.n_tokens)};
}
__device__ __forceinline__ int slot_of(const LinRecArgs& a, int seq) {
    const int s = a.slots ? a.slots[seq] : seq;
    return s < 0 || ((a.slots || a.s_in || a.s_out) && s >= a.n_slots) ? -1 : s;
}

template <class T>
__global__ __launch_bounds__(NT) void k_linrec(const LinRecArgs a) {
    const long long id = (long long)blockIdx.x * NT + threadIdx.x;
    const int seq = (int)(id / a.channels), c = (int)(id - (long long)seq * a.channels);
    if (seq >= a.n_seqs) return;
    const int slot = slot_of(a, seq);
    if (slot < 0) return;
    const Range r = range_of(a, seq);
    float h = a.s_in ? a.s_in[slot * a.si + c] : 0.0f;
    for (long long t = r.t0; t < r.t1; ++t) {
        if (a.carries && t % TILE == 0 && t > r.t0) a.carries[t / TILE * a.channels + c] = h;
        h = through(gate_of((float)((const T*)a.g)[t * a.gt + c]), h) + (float)((const T*)a.v)[t * a.vt + c];
        ((T*)a.out)[t * a.ot + c] = (T)(a.q ? (float)((const T*)a.q)[t * a.qt + c] * h : h);
    }
    if (a.s_out) a.s_out[slot * a.so + c] = h;
}

template <class T>
__global__ __launch_bounds__(NT) void k_linrec_zero(T* p, long long stride, long long rows, int channels) {
    const long long id = (long long)blockIdx.x * NT + threadIdx.x;
    const long long row = id / channels;
    if (row < rows) p[row * stride + id - row * channels] = (T)0.0f;
}

template <class T>
__global__ __launch_bounds__(NT) void k_linrec_backward(const LinRecArgs a) {
    const long long id = (long long)blockIdx.x * NT + threadIdx.x;
    const int seq = (int)(id / a.channels), c = (int)(id - (long long)seq * a.channels);
    if (seq >= a.n_seqs) return;
    const Range r = range_of(a, seq);
    float m = a.ds_out ? a.ds_out[seq * a.dso + c] : 0.0f;
    long long t1 = r.t1;
    while (t1 > r.t0) {
        long long t0 = (t1 - 1) / TILE * TILE;
        float h;
        if (t0 > r.t0) {
            h = a.carries[t0 / TILE * a.channels + c];
        } else {
            t0 = r.t0;
            h = a.s_in ? a.s_in[seq * a.si + c] : 0.0f;
        }
        float hs[TILE];
        for (long long t = t0; t < t1; ++t) {
            hs[t - t0] = h;
            h = through(gate_of((float)((const T*)a.g)[t * a.gt + c]), h) + (float)((const T*)a.v)[t * a.vt + c];
        }
        for (long long t = t1 - 1; t >= t0; --t) {
            const float s = gate_of((float)((const T*)a.g)[t * a.gt + c]);
            const float v = (float)((const T*)a.v)[t * a.vt + c];
            const float d = a.dout ? (float)((const T*)a.dout)[t * a.dot + c] : 0.0f;
            const float dh = (a.q ? (float)((const T*)a.q)[t * a.qt + c] * d : d) + m;
            if (a.dq) ((T*)a.dq)[t * a.dqt + c] = (T)(d * (through(s, hs[t - t0]) + v));
            if (a.dv) ((T*)a.dv)[t * a.dvt + c] = (T)dh;
            if (a.dg) ((T*)a.dg)[t * a.dgt + c] = (T)(dh * hs[t - t0] * slope_of(s));
            m = through(s, dh);
        }
        t1 = t0;
    }
    if (a.ds_in) a.ds_in[seq * a.dsi + c] = m;
}

template <class T>
__global__ __launch_bounds__(NT) void k_linrec_step(const LinRecArgs a) {
    const long long id = (long long)blockIdx.x * NT + threadIdx.x;
    const int seq = (int)(id / a.channels), c = (int)(id - (long long)seq * a.channels);
    if (seq >= a.n_seqs) return;
    const int slot = slot_of(a, seq);
    if (slot < 0) return;
    const float h = through(gate_of((float)((const T*)a.g)[seq * a.gt + c]), a.s_in[slot * a.si + c]) +
                    (float)((const T*)a.v)[seq * a.vt + c];
    ((T*)a.out)[seq * a.ot + c] = (T)(a.q ? (float)((const T*)a.q)[seq * a.qt + c] * h : h);
    a.s_out[slot * a.so + c] = h;
}

unsigned blocks_of(long long n) { return (unsigned)((n + NT - 1) / NT); }

template <class T>
hipError_t launch(const LinRecArgs& a, hipStream_t st) {
    k_linrec<T><<<blocks_of((long long)a.n_seqs * a.channels), NT, 0, st>>>(a);
    return hipGetLastError();
}

template <class T>
hipError_t launch_backward(const LinRecArgs& a, hipStream_t st) {
    void* const out[3] = {a.dg, a.dv, a.dq};
    const long long stride[3] = {a.dgt, a.dvt, a.dqt};
    for (int i = 0; i < 3; ++i)
        if (out[i] && a.n_tokens)
            k_linrec_zero<T><<<blocks_of(a.n_tokens * a.channels), NT, 0, st>>>((T*)out[i], stride[i], a.n_tokens,
                                                                                a.channels);
    if (a.n_seqs) k_linrec_backward<T><<<blocks_of((long long)a.n_seqs * a.channels), NT, 0, st>>>(a);
    return hipGetLastError();
}

template <class T>
hipError_t launch_step(const LinRecArgs& a, hipStream_t st) {
    k_linrec_step<T><<<blocks_of((long long)a.n_seqs * a.channels), NT, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace

void linrec_plan(LinRecArgs& a, int dtype) {
    a.tile = TILE;
    a.tiles = (int)((a.n_tokens + TILE - 1) / TILE);
}

hipError_t linrec_launch(const LinRecArgs& a, int dtype, hipStream_t st) {
    return dtype == SSLA_F32 ? launch<float>(a, st) : dtype == SSLA_BF16 ? launch<__bf16>(a, st) : launch<_Float16>(a, st);
}
hipError_t linrec_launch_backward(const LinRecArgs& a, int dtype, hipStream_t st) {
    return dtype == SSLA_F32    ? launch_backward<float>(a, st)
           : dtype == SSLA_BF16 ? launch_backward<__bf16>(a, st)
                                : launch_backward<_Float16>(a, st);
}
hipError_t linrec_launch_step(const LinRecArgs& a, int dtype, hipStream_t st) {
    return dtype == SSLA_F32    ? launch_step<float>(a, st)
           : dtype == SSLA_BF16 ? launch_step<__bf16>(a, st)
                                : launch_step<_Float16>(a, st);
}

}  // namespace ssla
