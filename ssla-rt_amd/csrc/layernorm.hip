// layernorm.hip -- layer norm and its gradients.
//
//   y = xh w + b,   xh = (s - mean) r,   r = 1 / sqrt(var + eps),   s = x + residual
//   u = w dy,   ds = r (u - mean(u) - xh mean(u xh)),   dw = sum dy xh,   db = sum dy
//
// Bound by memory: every tensor is read and written once.  A row is kept in registers
// by some lanes of a wave, in 16-byte pieces a lane, and nothing but shuffles joins
// them; a longer one by a workgroup, joined through LDS; one that no workgroup
// holds is read in strides, again for each use (k_ln, k_ln_backward, k_ln_columns).
// The mean is taken first, then squared differences from it, both in 64 bits (norm.h);
// it is kept as two floats, with the scale, for the backward pass.
//
// The sums over rows: a workgroup goes through rows a stride apart, each thread's
// channels stay the same, and so their sums stay in its registers; the
// workgroup's are joined in LDS and left in the workspace, and k_ln_join adds them up.
// Every order is fixed.
#include "layernorm.h"

#include "norm.h"

namespace ssla {
namespace {

constexpr int NT = 256;

struct Stat {
    float hi, lo, scale;
};

template <class T, int V>
struct Piece {
    T v[V];
};

// What the compiler has made of 16-bit values ends here: it would otherwise keep all of
// them as floats from one use to the next, and from row to row.
template <class T, int V, int K>
__device__ __forceinline__ void opaque(Piece<T, V> (&p)[K]) {
    if constexpr (sizeof(T) == 2 && V % 2 == 0) {
        #pragma unroll
        for (int k = 0; k < K; ++k) {
            unsigned x[V / 2];
            __builtin_memcpy(x, &p[k], sizeof(x));
            #pragma unroll
            for (unsigned& w : x) asm("" : "+v"(w));
            __builtin_memcpy(&p[k], x, sizeof(x));
        }
    }
}

__device__ __forceinline__ float normed(float x, const Stat& f) {
    return fmaf(fmaf(x, kDown, -f.hi), f.scale, -f.lo * f.scale);
}

// ---- rows in registers -----------------------------------------------------------
// Where a thread works: l-th of a row's lanes, its pieces l, l + lanes, ...  The last
// piece of a row whose channels are no whole pieces is the row's last V channels;
// those that the piece before has too are `over`.
template <int V, int K, bool TAIL>
struct Columns {
    int l, c[K], over[K];
    bool on[K];

    __device__ __forceinline__ Columns(const LayerNormArgs& a) {
        l = threadIdx.x & (a.lanes - 1);
        if (a.lanes > 64) l = threadIdx.x;
        #pragma unroll
        for (int k = 0; k < K; ++k) {
            const int at = (l + k * a.lanes) * V;
            on[k] = at < a.channels;
            c[k] = TAIL ? max(min(at, a.channels - V), 0) : at;
            over[k] = TAIL ? at - c[k] : 0;
        }
    }
    // Whether value i of piece k is the thread's own.
    __device__ __forceinline__ bool own(int k, int i) const { return on[k] && (!TAIL || i >= over[k]); }

    template <class T>
    __device__ __forceinline__ void load(Piece<T, V> (&x)[K], const void* base, long long at) const {
        #pragma unroll
        for (int k = 0; k < K; ++k)
            if (on[k]) __builtin_memcpy(&x[k], (const T*)base + at + c[k], sizeof(x[k]));
    }
    template <class T>
    __device__ __forceinline__ void store(void* base, long long at, const Piece<T, V>& x, int k) const {
        T* to = (T*)base + at + c[k];
        if (!TAIL || over[k] == 0) {
            __builtin_memcpy(to, &x, sizeof(x));
        } else {
            #pragma unroll
            for (int i = 1; i < V; ++i)
                if (i >= over[k]) to[i] = x.v[i];
        }
    }
    // weight or bias
    template <class W>
    __device__ __forceinline__ void params(Piece<W, V> (&w)[K], const void* p, float none) const {
        #pragma unroll
        for (int k = 0; k < K; ++k) {
            #pragma unroll
            for (int i = 0; i < V; ++i) w[k].v[i] = (W)none;
            if (p && on[k]) __builtin_memcpy(&w[k], (const W*)p + c[k], sizeof(w[k]));
        }
    }
};

// Sum over a row's threads, in each of them.  Two buffers in turn need one barrier.
template <bool WHOLE, class F>
__device__ __forceinline__ F row_sum(F s, int lanes, F* waves) {
    s = lanes_sum(s, WHOLE ? 64 : lanes);
    if (WHOLE) {
        const int n = blockDim.x >> 6;
        if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = s;
        __syncthreads();
        s = waves[0];
        for (int i = 1; i < n; ++i) s += waves[i];
    }
    return s;
}

// Row of a thread's group at step i, and how many there are at a time.
__device__ __forceinline__ int rows_at_once(const LayerNormArgs& a, bool whole) {
    return whole ? 1 : blockDim.x / a.lanes;
}

template <class T, class W, int V, int K, bool WHOLE, bool TAIL>
__global__ __launch_bounds__(512) void k_ln_rows(const LayerNormArgs a) {
    __shared__ double sums[2][2][8];
    const Columns<V, K, TAIL> col(a);
    const int per = rows_at_once(a, WHOLE);
    Piece<W, V> w[K], b[K];
    col.params(w, a.weight, 1.0f);
    col.params(b, a.bias, 0.0f);
    const long long step = (long long)gridDim.x * per;
    int turn = 0;
    for (long long row = (long long)blockIdx.x * per + (WHOLE ? 0 : threadIdx.x / a.lanes); row < a.rows;
         row += step, turn ^= 1) {
        Piece<T, V> x[K], res[K];
        col.load(x, a.x, row * a.xr);
        if (a.res) col.load(res, a.res, row * a.rr);
        auto at = [&](int k, int i) { return a.res ? (float)x[k].v[i] + (float)res[k].v[i] : (float)x[k].v[i]; };
        double sum = 0.0;
        #pragma unroll
        for (int k = 0; k < K; ++k)
            #pragma unroll
            for (int i = 0; i < V; ++i) sum += col.own(k, i) ? (double)at(k, i) : 0.0;
        opaque(x), opaque(res);
        const double mean = row_sum<WHOLE>(sum, a.lanes, sums[turn][0]) * a.inv_channels;
        double sq = 0.0;
        #pragma unroll
        for (int k = 0; k < K; ++k)
            #pragma unroll
            for (int i = 0; i < V; ++i) {
                const double d = (double)at(k, i) - mean;
                sq = col.own(k, i) ? fma(d, d, sq) : sq;
            }
        opaque(x), opaque(res), opaque(w), opaque(b);
        sq = row_sum<WHOLE>(sq, a.lanes, sums[turn][1]);
        const Norm n = norm_of(mean, sq * a.inv_channels, a.eps);
        const Stat f = {n.hi, n.lo, n.scale};
        if (a.stats && col.l == 0) ((Stat*)a.stats)[row] = f;
        #pragma unroll
        for (int k = 0; k < K; ++k) {
            if (!col.on[k]) continue;
            Piece<T, V> y;
            #pragma unroll
            for (int i = 0; i < V; ++i) y.v[i] = (T)fmaf(normed(at(k, i), f), (float)w[k].v[i], (float)b[k].v[i]);
            col.store(a.out, row * a.orow, y, k);
        }
    }
}

template <class T, class W, int V, int K, bool WHOLE, bool TAIL>
__global__ __launch_bounds__(512) void k_ln_rows_backward(const LayerNormArgs a) {
    extern __shared__ float joined[];                        // [groups of lanes][2][lanes * K * V], by halves
    __shared__ float sums[2][2][8];
    const Columns<V, K, TAIL> col(a);
    const int per = rows_at_once(a, WHOLE), group = WHOLE ? 0 : threadIdx.x / a.lanes;
    const float inv = (float)a.inv_channels;
    Piece<W, V> w[K];
    col.params(w, a.weight, 1.0f);
    float dw[K][V], db[K][V];
    #pragma unroll
    for (int k = 0; k < K; ++k)
        #pragma unroll
        for (int i = 0; i < V; ++i) dw[k][i] = db[k][i] = 0.0f;
    const long long step = (long long)gridDim.x * per;
    int turn = 0;
    for (long long row = (long long)blockIdx.x * per + group; row < a.rows; row += step, turn ^= 1) {
        Piece<T, V> x[K], res[K], dy[K];
        col.load(x, a.x, row * a.xr);
        if (a.res) col.load(res, a.res, row * a.rr);
        col.load(dy, a.dout, row * a.dor);
        const Stat f = ((const Stat*)a.stats)[row];
        auto at = [&](int k, int i) { return a.res ? (float)x[k].v[i] + (float)res[k].v[i] : (float)x[k].v[i]; };
        float c1 = 0.0f, c2 = 0.0f;
        #pragma unroll
        for (int k = 0; k < K; ++k)
            #pragma unroll
            for (int i = 0; i < V; ++i) {
                const float xh = normed(at(k, i), f), g = (float)dy[k].v[i], u = g * (float)w[k].v[i];
                if (col.own(k, i)) {
                    dw[k][i] = fmaf(g, xh, dw[k][i]);
                    db[k][i] += g;
                    c1 += u;
                    c2 = fmaf(u, xh, c2);
                }
            }
        opaque(x), opaque(res), opaque(dy), opaque(w);
        if (!a.dx) continue;
        c1 = lanes_sum(c1, WHOLE ? 64 : a.lanes);
        c2 = lanes_sum(c2, WHOLE ? 64 : a.lanes);
        if (WHOLE) {
            const int n = blockDim.x >> 6;
            if ((threadIdx.x & 63) == 0) {
                sums[turn][0][threadIdx.x >> 6] = c1;
                sums[turn][1][threadIdx.x >> 6] = c2;
            }
            __syncthreads();
            c1 = sums[turn][0][0], c2 = sums[turn][1][0];
            for (int i = 1; i < n; ++i) c1 += sums[turn][0][i], c2 += sums[turn][1][i];
        }
        c1 *= inv, c2 *= inv;
        const float r = f.scale * kDown;
        #pragma unroll
        for (int k = 0; k < K; ++k) {
            if (!col.on[k]) continue;
            Piece<T, V> y;
            #pragma unroll
            for (int i = 0; i < V; ++i)
                y.v[i] = (T)(r * (fmaf((float)dy[k].v[i], (float)w[k].v[i], -c1) - normed(at(k, i), f) * c2));
            col.store(a.dx, row * a.dxr, y, k);
        }
    }
    if (!a.parts) return;
    // the workgroup's sums: of its rows' lanes, one half of the groups onto the other
    float* ws = a.ws + (long long)blockIdx.x * 2 * a.channels;
    if (!WHOLE) {
        const int width = a.lanes * K * V;
        for (int n = per / 2; n > 0; n /= 2) {
            float* to = joined + (group - n) * 2 * width;
            if (group >= n && group < 2 * n) {
                #pragma unroll
                for (int k = 0; k < K; ++k)
                    #pragma unroll
                    for (int i = 0; i < V; ++i) {
                        to[(k * V + i) * a.lanes + col.l] = dw[k][i];
                        to[width + (k * V + i) * a.lanes + col.l] = db[k][i];
                    }
            }
            __syncthreads();
            if (group < n) {
                const float* from = joined + group * 2 * width;
                #pragma unroll
                for (int k = 0; k < K; ++k)
                    #pragma unroll
                    for (int i = 0; i < V; ++i) {
                        dw[k][i] += from[(k * V + i) * a.lanes + col.l];
                        db[k][i] += from[width + (k * V + i) * a.lanes + col.l];
                    }
            }
            __syncthreads();
        }
        if (group) return;
    }
    #pragma unroll
    for (int k = 0; k < K; ++k)
        #pragma unroll
        for (int i = 0; i < V; ++i)
            if (col.own(k, i)) {
                ws[col.c[k] + i] = dw[k][i];
                ws[a.channels + col.c[k] + i] = db[k][i];
            }
}

// Adds up the parts: sixteen neighbouring sums a workgroup, sixty-four parts at a time.
template <class T>
__global__ __launch_bounds__(1024) void k_ln_join(const LayerNormArgs a) {
    __shared__ double part[64][17];
    const int x = threadIdx.x & 15, y = threadIdx.x >> 4;
    const long long at = (long long)blockIdx.x * 16 + x, n = 2ll * a.channels;
    double s = 0.0;
    if (at < n)
        for (int p = y; p < a.parts; p += 64) s += (double)a.ws[p * n + at];
    part[y][x] = s;
    __syncthreads();
    for (int m = 32; m > 0; m /= 2) {
        if (y < m) part[y][x] += part[y + m][x];
        __syncthreads();
    }
    if (y || at >= n) return;
    void* to = at < a.channels ? a.dw : a.db;
    const long long c = at < a.channels ? at : at - a.channels;
    if (!to) return;
    if (a.wide) ((float*)to)[c] = (float)part[0][x];
    else ((T*)to)[c] = (T)(float)part[0][x];
}

// ---- rows in strides --------------------------------------------------------------
template <class T>
__device__ __forceinline__ float sum_at(const LayerNormArgs& a, long long row, int c) {
    const float x = (float)((const T*)a.x)[row * a.xr + c];
    return a.res ? x + (float)((const T*)a.res)[row * a.rr + c] : x;
}
template <class T>
__device__ __forceinline__ float param(const void* p, int c, int wide, float none) {
    return !p ? none : wide ? ((const float*)p)[c] : (float)((const T*)p)[c];
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
    const double mean = block_sum(s, waves) * a.inv_channels;
    double q = 0.0;
    for (int c = threadIdx.x; c < a.channels; c += NT) {
        const double d = (double)sum_at<T>(a, row, c) - mean;
        q = fma(d, d, q);
    }
    q = block_sum(q, waves) * a.inv_channels;
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
    s = block_sum(s, waves) * (float)a.inv_channels;
    q = block_sum(q, waves) * (float)a.inv_channels;
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

template <class T, class W, int V, int K, bool WHOLE>
const void* kernel(const LayerNormArgs& a, bool backward) {
    if (V > 1 && a.channels % V)
        return backward ? (const void*)k_ln_rows_backward<T, W, V, K, WHOLE, (V > 1)>
                        : (const void*)k_ln_rows<T, W, V, K, WHOLE, (V > 1)>;
    return backward ? (const void*)k_ln_rows_backward<T, W, V, K, WHOLE, false>
                    : (const void*)k_ln_rows<T, W, V, K, WHOLE, false>;
}
template <class T, class W>
const void* kernel(const LayerNormArgs& a, bool backward) {
    constexpr int V = 16 / sizeof(T);
    if (a.vec == 1) return kernel<T, W, 1, 1, false>(a, backward);
    if (a.lanes > 64) return kernel<T, W, V, 4, true>(a, backward);
    return a.reps == 1   ? kernel<T, W, V, 1, false>(a, backward)
           : a.reps == 2 ? kernel<T, W, V, 2, false>(a, backward)
           : a.reps == 3 ? kernel<T, W, V, 3, false>(a, backward)
                         : kernel<T, W, V, 4, false>(a, backward);
}
template <class T>
const void* kernel(const LayerNormArgs& a, bool backward) {
    return a.wide ? kernel<T, float>(a, backward) : kernel<T, T>(a, backward);
}

template <class T>
hipError_t launch(const LayerNormArgs& a, hipStream_t st) {
    LayerNormArgs args = a;
    void* pa[] = {&args};
    return hipLaunchKernel(a.reps ? kernel<T>(a, false) : (const void*)k_ln<T>, dim3(a.wgs), dim3(a.threads), pa, 0, st);
}

template <class T>
hipError_t launch_backward(const LayerNormArgs& a, hipStream_t st) {
    LayerNormArgs args = a;
    void* pa[] = {&args};
    hipError_t e = hipSuccess;
    if (a.rows && a.reps) {
        const size_t lds = a.parts && a.lanes <= 64 ? (size_t)(a.threads / 2) * a.reps * a.vec * 2 * 4 : 0;
        if (lds > 65536) {
            e = hipFuncSetAttribute(kernel<T>(a, true), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
            if (e != hipSuccess) return e;
        }
        e = hipLaunchKernel(kernel<T>(a, true), dim3(a.wgs), dim3(a.threads), pa, lds, st);
    } else if (a.rows) {
        if (a.dx) e = hipLaunchKernel((const void*)k_ln_backward<T>, dim3(a.wgs), dim3(NT), pa, 0, st);
        if (e == hipSuccess && a.parts)
            e = hipLaunchKernel((const void*)k_ln_columns<T>, dim3((a.channels + NT - 1) / NT, a.parts), dim3(NT), pa, 0, st);
    }
    if (e == hipSuccess && (a.dw || a.db))
        e = hipLaunchKernel((const void*)k_ln_join<T>, dim3((unsigned)((2ll * a.channels + 15) / 16)), dim3(1024), pa, 0, st);
    return e;
}

}  // namespace

void layer_norm_plan(LayerNormArgs& a, int dtype, bool backward) {
    const bool sums = backward && (a.dw || a.db);
    a.inv_channels = 1.0 / a.channels;
    a.vec = dtype == SSLA_F32 ? 4 : 8;
    if (a.channels < a.vec) a.vec = 1;
    const int pieces = (a.channels - 1) / a.vec + 1;
    a.parts = 0;
    a.threads = backward && pieces > 128 ? 512 : NT;
    if (pieces <= 256) {
        // as few lanes as hold a row in four pieces each, or in three where that fills them
        int lanes = 1;
        while (lanes * 4 < pieces) lanes *= 2;
        a.lanes = lanes;
        a.reps = (pieces + lanes - 1) / lanes;
        if (a.vec == 1) a.lanes = 8, a.reps = 1;
    } else if (pieces <= 2048) {
        a.threads = (pieces + 255) / 256 * 64;
        a.lanes = a.threads;
        a.reps = 4;
    } else {
        a.threads = NT, a.lanes = NT, a.reps = 0;
        a.wgs = a.rows;
        if (sums) a.parts = a.rows < 256 ? (a.rows + 15) / 16 : 256;
        return;
    }
    const int per = a.lanes > 64 ? 1 : a.threads / a.lanes;
    const long long all = ((long long)a.rows + per - 1) / per, most = backward ? 256 * 1024 / a.threads / 2 : 2048 * 256 / a.threads;
    a.wgs = (int)(all < most ? all : most);
    if (sums) a.parts = a.wgs;
}

hipError_t layer_norm_launch(const LayerNormArgs& a, int dtype, hipStream_t st) {
    if (dtype == SSLA_F32) return launch<float>(a, st);
    if (dtype == SSLA_BF16) return launch<__bf16>(a, st);
    return launch<_Float16>(a, st);
}
hipError_t layer_norm_launch_backward(const LayerNormArgs& a, int dtype, hipStream_t st) {
    if (dtype == SSLA_F32) return launch_backward<float>(a, st);
    if (dtype == SSLA_BF16) return launch_backward<__bf16>(a, st);
    return launch_backward<_Float16>(a, st);
}

}  // namespace ssla
