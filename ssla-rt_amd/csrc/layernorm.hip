// layernorm.hip -- layer norm and its gradients: a workgroup a row, a thread a
// channel of some rows for the sums over them.
#include "layernorm.h"

#include "norm.h"

namespace ssla {
namespace {

constexpr int NT = 256;

struct Stat {
    float hi, lo, scale;
};

template <class T>
__device__ __forceinline__ float sum_at(const LayerNormArgs& a, long long row, int c) {
    const float x = (float)((const T*)a.x)[row * a.xr + c];
    return a.res ? x + (float)((const T*)a.res)[row * a.rr + c] : x;
}
template <class T>
__device__ __forceinline__ float param(const void* p, int c, int wide, float none) {
    return !p ? none : wide ? ((const float*)p)[c] : (float)((const T*)p)[c];
}
__device__ __forceinline__ float normed(float x, const Stat& f) {
    return fmaf(fmaf(x, kDown, -f.hi), f.scale, -f.lo * f.scale);
}

template <class F>
__device__ __forceinline__ F block_sum(F s, F* waves) {
    s = lanes_sum(s, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = s;
    __syncthreads();
    return waves[0] + waves[1] + waves[2] + waves[3];
}

template <class T>
__global__ __launch_bounds__(NT) void k_ln(const LayerNormArgs a) {
    __shared__ double waves[NT / 64];
    const long long row = blockIdx.x;
    double s = 0.0;
    for (int c = threadIdx.x; c < a.channels; c += NT) s += (double)sum_at<T>(a, row, c);
    const double mean = block_sum(s, waves) / a.channels;
    double q = 0.0;
    for (int c = threadIdx.x; c < a.channels; c += NT) {
        const double d = (double)sum_at<T>(a, row, c) - mean;
        q = fma(d, d, q);
    }
    q = block_sum(q, waves) / a.channels;
    const Norm n = norm_of(mean, q, a.eps);
    const Stat f = {n.hi, n.lo, n.scale};
    if (a.stats && threadIdx.x == 0) ((Stat*)a.stats)[row] = f;
    for (int c = threadIdx.x; c < a.channels; c += NT)
        ((T*)a.out)[row * a.orow + c] =
            (T)fmaf(normed(sum_at<T>(a, row, c), f), param<T>(a.weight, c, a.wide, 1.0f), param<T>(a.bias, c, a.wide, 0.0f));
}

template <class T>
__global__ __launch_bounds__(NT) void k_ln_backward(const LayerNormArgs a) {
    __shared__ float waves[NT / 64];
    const long long row = blockIdx.x;
    const Stat f = ((const Stat*)a.stats)[row];
    float s = 0.0f, q = 0.0f;
    for (int c = threadIdx.x; c < a.channels; c += NT) {
        const float u = (float)((const T*)a.dout)[row * a.dor + c] * param<T>(a.weight, c, a.wide, 1.0f);
        s += u;
        q = fmaf(u, normed(sum_at<T>(a, row, c), f), q);
    }
    s = block_sum(s, waves) / a.channels;
    q = block_sum(q, waves) / a.channels;
    const float r = f.scale * kDown;
    for (int c = threadIdx.x; c < a.channels; c += NT) {
        const float u = (float)((const T*)a.dout)[row * a.dor + c] * param<T>(a.weight, c, a.wide, 1.0f);
        ((T*)a.dx)[row * a.dxr + c] = (T)(r * (u - s - normed(sum_at<T>(a, row, c), f) * q));
    }
}

// Sums over a part's rows, a thread a channel.
template <class T>
__global__ __launch_bounds__(NT) void k_ln_columns(const LayerNormArgs a) {
    const int c = blockIdx.x * NT + threadIdx.x, part = blockIdx.y;
    if (c >= a.channels) return;
    const int r0 = (int)((long long)a.rows * part / a.parts), r1 = (int)((long long)a.rows * (part + 1) / a.parts);
    float w = 0.0f, b = 0.0f;
    for (long long row = r0; row < r1; ++row) {
        const float d = (float)((const T*)a.dout)[row * a.dor + c];
        w = fmaf(d, normed(sum_at<T>(a, row, c), ((const Stat*)a.stats)[row]), w);
        b += d;
    }
    float* ws = a.ws + (long long)part * 2 * a.channels;
    ws[c] = w;
    ws[a.channels + c] = b;
}

template <class T>
__global__ __launch_bounds__(NT) void k_ln_join(const LayerNormArgs a) {
    const int c = blockIdx.x * NT + threadIdx.x;
    if (c >= a.channels) return;
    double w = 0.0, b = 0.0;
    for (int p = 0; p < a.parts; ++p) {
        w += (double)a.ws[(long long)p * 2 * a.channels + c];
        b += (double)a.ws[((long long)p * 2 + 1) * a.channels + c];
    }
    if (a.dw) a.wide ? (void)(((float*)a.dw)[c] = (float)w) : (void)(((T*)a.dw)[c] = (T)(float)w);
    if (a.db) a.wide ? (void)(((float*)a.db)[c] = (float)b) : (void)(((T*)a.db)[c] = (T)(float)b);
}

template <class T>
hipError_t launch_backward(const LayerNormArgs& a, hipStream_t st) {
    if (a.dx && a.rows) k_ln_backward<T><<<a.rows, NT, 0, st>>>(a);
    if (a.dw || a.db) {
        const unsigned blocks = (a.channels + NT - 1) / NT;
        if (a.rows) k_ln_columns<T><<<dim3(blocks, a.parts), NT, 0, st>>>(a);
        k_ln_join<T><<<blocks, NT, 0, st>>>(a);
    }
    return hipGetLastError();
}

}  // namespace

void layer_norm_plan(LayerNormArgs& a, int dtype, bool sums) {
    a.parts = sums && a.rows ? (a.rows < 256 ? (a.rows + 15) / 16 : 256) : 0;
}

hipError_t layer_norm_launch(const LayerNormArgs& a, int dtype, hipStream_t st) {
    if (dtype == SSLA_F32) k_ln<float><<<a.rows, NT, 0, st>>>(a);
    else if (dtype == SSLA_BF16) k_ln<__bf16><<<a.rows, NT, 0, st>>>(a);
    else k_ln<_Float16><<<a.rows, NT, 0, st>>>(a);
    return hipGetLastError();
}
hipError_t layer_norm_launch_backward(const LayerNormArgs& a, int dtype, hipStream_t st) {
    return dtype == SSLA_F32    ? launch_backward<float>(a, st)
           : dtype == SSLA_BF16 ? launch_backward<__bf16>(a, st)
                                : launch_backward<_Float16>(a, st);
}

}  // namespace ssla
