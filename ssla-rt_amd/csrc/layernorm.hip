// layernorm.hip -- layer norm and its gradients.
//
//   y = xh w + b,   xh = (s - mean) r,   r = 1 / sqrt(var + eps),   s = x + residual
//   u = w dy,   ds = r (u - mean(u) - xh mean(u xh)),   dw = sum dy xh,   db = sum dy
//
// Bound by memory: every tensor is read and written once.  A row is kept in registers
// by some lanes of a wave, in 16-byte pieces a lane, and nothing but shuffles joins
// them; a longer one by a workgroup, joined through LDS; one that no workgroup
// holds is read in strides, again for each use (k_ln, k_ln_backward, k_ln_columns; 20000 bf16
// values 0.9 TB/s each way).
// The mean is taken first, in 64 bits, then squared differences from it, in 64 bits
// too, or for 16-bit types in 32 where those hold them (below); mean and scale are kept as
// three floats (norm.h) for the backward pass.
//
// Measured with 100 MB a tensor: fp32 rows of 96 to 2048 channels, forward 5.2 to 5.8 TB/s,
// backward 4.9 to 5.1; bf16 rows of 256 to 4096 4.6 to 5.1 and 4.2 to 4.8, of 8192 4.9 and 3.8
// (its workgroups have barriers in every row, and more sums to leave), of 4104, which take
// workgroups of three waves a row, 4.0 and 2.5, of 4099, which no line holds either, 3.2 and 2.1.
//
// The sums over rows: a workgroup goes through rows a stride apart, each thread's
// channels stay the same, and so their sums stay in its registers; the
// workgroup's are joined in LDS and left in the workspace, and k_ln_join adds them up.
// Every order is fixed.
#include "layernorm.h"

#include "norm.h"
#include "piece.h"

namespace ssla {
namespace {

constexpr int NT = 256;

struct Stat {
    float hi, lo, scale;
};

__device__ __forceinline__ float normed(float x, const Stat& f) {
    return fmaf(fmaf(x, kDown, -f.hi), f.scale, -f.lo * f.scale);
}

// ---- rows in registers -----------------------------------------------------------
// Where a thread works: l-th of a row's lanes, its pieces l, l + lanes, ...  The last
// piece of a row whose channels are no whole pieces is the row's last V channels;
// those that the piece before has too are `over`.  A piece that is not there is the
// first one again, with a weight of zero in every sum.
template <int V, int K, bool TAIL>
struct Columns {
    int group, l, c[K], over[K];                             // row of those at once; thread of the row
    bool on[K];

    __device__ __forceinline__ Columns(const LayerNormArgs& a) {
        group = threadIdx.x / a.lanes;
        l = threadIdx.x - group * a.lanes;
        #pragma unroll
        for (int k = 0; k < K; ++k) {
            const int at = (l + k * a.lanes) * V;
            on[k] = at < a.channels;
            c[k] = !on[k] ? 0 : TAIL ? min(at, a.channels - V) : at;
            over[k] = TAIL && on[k] ? at - c[k] : 0;
        }
    }
    // Whether value i of piece k is the thread's own, where piece k is there.
    __device__ __forceinline__ bool own(int k, int i) const { return !TAIL || i >= over[k]; }

    template <class T>
    __device__ __forceinline__ void load(Piece<T, V> (&x)[K], const void* base, long long at) const {
        #pragma unroll
        for (int k = 0; k < K; ++k) x[k].load((const T*)base + at + c[k]);
    }
    template <class T>
    __device__ __forceinline__ void store(void* base, long long at, const Piece<T, V>& x, int k) const {
        if (!on[k]) return;
        T* to = (T*)base + at + c[k];
        if (!TAIL || over[k] == 0) x.store(to);
        else x.store_from(to, over[k]);
    }
    // weight or bias
    template <class W>
    __device__ __forceinline__ void params(Piece<W, V> (&w)[K], const void* p, float none) const {
        float x[V];
        #pragma unroll
        for (int i = 0; i < V; ++i) x[i] = none;
        #pragma unroll
        for (int k = 0; k < K; ++k) {
            if (p) w[k].load((const W*)p + c[k]);
            else w[k].set(x);
        }
    }
};
template <class T, int V, int K>
__device__ __forceinline__ void opaque(Piece<T, V> (&x)[K]) {
    #pragma unroll
    for (int k = 0; k < K; ++k) x[k].opaque();
}

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

template <bool WHOLE>
__device__ __forceinline__ void row_sums(float& s, float& q, int lanes, float* waves, int group = 0) {
    s = lanes_sum(s, WHOLE ? 64 : lanes);
    q = lanes_sum(q, WHOLE ? 64 : lanes);
    if (WHOLE) {
        const int n = lanes >> 6, first = group * n;
        if ((threadIdx.x & 63) == 0) {
            waves[threadIdx.x >> 6] = s;
            waves[8 + (threadIdx.x >> 6)] = q;
        }
        __syncthreads();
        s = waves[first], q = waves[8 + first];
        for (int i = 1; i < n; ++i) s += waves[first + i], q += waves[8 + first + i];
    }
}

// Pieces one after another: the scheduler otherwise makes floats of all of them first.
__device__ __forceinline__ void in_turn() { __builtin_amdgcn_sched_barrier(0); }

template <class T, class W, int V, int K, bool WHOLE, bool TAIL>
__global__ __launch_bounds__(512) void k_ln_rows(const LayerNormArgs a) {
    __shared__ double sums[2][2][8];
    const Columns<V, K, TAIL> col(a);
    const int per = blockDim.x / a.lanes;
    Piece<W, V> w[K], b[K];
    col.params(w, a.weight, 1.0f);
    col.params(b, a.bias, 0.0f);
    const long long step = (long long)gridDim.x * per;
    int turn = 0;
    for (long long row = (long long)blockIdx.x * per + col.group; row < a.rows;
         row += step, turn ^= 1) {
        Piece<T, V> x[K], res[K];
        col.load(x, a.x, row * a.xr);
        if (a.res) col.load(res, a.res, row * a.rr);
        auto at = [&](int k, int i) { return a.res ? x[k].at(i) + res[k].at(i) : x[k].at(i); };
        double sum = 0.0;
        #pragma unroll
        for (int k = 0; k < K; ++k) {
            double one = 0.0;
            #pragma unroll
            for (int i = 0; i < V; ++i) one += col.own(k, i) ? (double)at(k, i) : 0.0;
            sum += col.on[k] ? one : 0.0;
        }
        opaque(x), opaque(res);
        const double mean = row_sum<WHOLE>(sum, a.lanes, sums[turn][0]) * a.inv_channels;
        // squares in 64 bits
        auto squares = [&] {
            double sq = 0.0;
            #pragma unroll
            for (int k = 0; k < K; ++k) {
                double one = 0.0;
                #pragma unroll
                for (int i = 0; i < V; ++i) {
                    const double d = (double)at(k, i) - mean;
                    one = col.own(k, i) ? fma(d, d, one) : one;
                }
                sq += col.on[k] ? one : 0.0;
            }
            opaque(x), opaque(res);
            return row_sum<WHOLE>(sq, a.lanes, sums[turn][1]) * a.inv_channels;
        };
        double var;
        if constexpr (sizeof(T) == 4) {
            var = squares();
        } else {
            // In 32 bits (6139 x 8192 bf16: 39.9 us, in 64 bits 44.0; 196602 x 256 44.0 and 47.0):
            // of differences from the mean's float, whose own mean is what that leaves of the
            // mean.  Each is rounded by 2^-24 of itself at most, which the variance keeps, but for
            // squares below 2^-126, of which a row's 2^14 at most lose 2^-112: 2^-32 of a sum of
            // 2^-80, and nothing beside an eps of 2^-60.
            const float m = (float)mean;
            float sq = 0.0f;
            #pragma unroll
            for (int k = 0; k < K; ++k) {
                float one = 0.0f;
                #pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float d = col.own(k, i) ? at(k, i) - m : 0.0f;
                    one = fmaf(d, d, one);
                }
                sq += col.on[k] ? one : 0.0f;
            }
            opaque(x), opaque(res);
            sq = row_sum<WHOLE>(sq, a.lanes, (float*)sums[turn][1]);
            // a row whose squares are too large or too small, or that is not finite; all of a
            // row's lanes agree
            if (sq < __builtin_inff() && (sq >= 0x1p-80f || a.eps >= 0x1p-60f)) {
                const double rest = mean - (double)m;
                var = fma(-rest, rest, (double)sq * a.inv_channels);
                var = var < 0.0 ? 0.0 : var;
            } else {
                if (WHOLE) __syncthreads();
                var = squares();
            }
        }
        const Norm n = norm_of(mean, var, a.eps);
        opaque(w), opaque(b);
        const Stat f = {n.hi, n.lo, n.scale};
        if (a.stats && col.l == 0) ((Stat*)a.stats)[row] = f;
        #pragma unroll
        for (int k = 0; k < K; ++k) {
            float o[V];
            #pragma unroll
            for (int i = 0; i < V; ++i) o[i] = fmaf(normed(at(k, i), f), w[k].at(i), b[k].at(i));
            Piece<T, V> y;
            y.set(o);
            col.store(a.out, row * a.orow, y, k);
        }
    }
}

template <class T, class W, int V, int K, bool WHOLE, bool TAIL>
__global__ __launch_bounds__(512) void k_ln_rows_backward(const LayerNormArgs a) {
    extern __shared__ float joined[];                        // [half of the threads][2 K V + 1]
    __shared__ float sums[2][16];
    const Columns<V, K, TAIL> col(a);
    const int per = blockDim.x / a.lanes, group = col.group;
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
    for (long long at_row = (long long)blockIdx.x * per; at_row < a.rows; at_row += step, turn ^= 1) {
        // all rows of a workgroup go through its barriers; one behind the last is that
        // again, with gradients of zero
        const bool there = at_row + group < a.rows;
        const long long row = there ? at_row + group : a.rows - 1;
        Piece<T, V> x[K], res[K], dy[K];
        col.load(x, a.x, row * a.xr);
        if (a.res) col.load(res, a.res, row * a.rr);
        col.load(dy, a.dout, row * a.dor);
        const Stat f = ((const Stat*)a.stats)[row];
        auto at = [&](int k, int i) { return a.res ? x[k].at(i) + res[k].at(i) : x[k].at(i); };
        float c1 = 0.0f, c2 = 0.0f;
        #pragma unroll
        for (int k = 0; k < K; ++k) {
            if (!col.on[k] || !there) dy[k].zero();
            #pragma unroll
            for (int i = 0; i < V; ++i) {
                const float xh = normed(at(k, i), f), g = col.own(k, i) ? dy[k].at(i) : 0.0f, u = g * w[k].at(i);
                dw[k][i] = fmaf(g, xh, dw[k][i]);
                db[k][i] += g;
                c1 += u;
                c2 = fmaf(u, xh, c2);
            }
            in_turn();
        }
        opaque(x), opaque(res), opaque(dy), opaque(w);
        if (a.dx) {
            row_sums<WHOLE>(c1, c2, a.lanes, sums[turn], group);
            c1 *= inv, c2 *= inv;
            const float r = f.scale * kDown;
            #pragma unroll
            for (int k = 0; k < K; ++k) {
                float o[V];
                #pragma unroll
                for (int i = 0; i < V; ++i) o[i] = r * (fmaf(dy[k].at(i), w[k].at(i), -c1) - normed(at(k, i), f) * c2);
                Piece<T, V> y;
                y.set(o);
                if (there) col.store(a.dx, row * a.dxr, y, k);
                in_turn();
            }
        }
    }
    if (!a.parts) return;
    // the workgroup's sums: of its rows' lanes, one half of the groups onto the other
    float* ws = a.ws + (long long)blockIdx.x * 2 * a.channels;
    constexpr int kOwn = 2 * K * V + 1;
    for (int n = (per + 1) / 2, m = per; m > 1; m = n, n = (n + 1) / 2) {        // m groups onto n
        if (group >= n && group < m) {
            float* to = joined + ((group - n) * a.lanes + col.l) * kOwn;
            #pragma unroll
            for (int k = 0; k < K; ++k)
                #pragma unroll
                for (int i = 0; i < V; ++i) to[k * V + i] = dw[k][i], to[K * V + k * V + i] = db[k][i];
        }
        __syncthreads();
        if (group < m - n) {
            const float* from = joined + (group * a.lanes + col.l) * kOwn;
            #pragma unroll
            for (int k = 0; k < K; ++k)
                #pragma unroll
                for (int i = 0; i < V; ++i) dw[k][i] += from[k * V + i], db[k][i] += from[K * V + k * V + i];
        }
        __syncthreads();
    }
    if (group) return;
    #pragma unroll
    for (int k = 0; k < K; ++k)
        #pragma unroll
        for (int i = 0; i < V; ++i)
            if (col.on[k] && col.own(k, i)) {
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
    if (a.lanes > 64)
        return a.reps == 3 ? kernel<T, W, V, 3, true>(a, backward) : kernel<T, W, V, 4, true>(a, backward);
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
        const size_t lds = a.parts ? (size_t)((a.threads / a.lanes) / 2 * a.lanes) * (2 * a.reps * a.vec + 1) * 4 : 0;
        if (lds > 65536) {
            e = hipFuncSetAttribute(kernel<T>(a, true), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
            if (e != hipSuccess) return e;
        }
        e = hipLaunchKernel(kernel<T>(a, true), dim3(a.wgs), dim3(a.threads), pa, lds, st);
    } else if (a.rows) {
        if (a.dx) e = hipLaunchKernel((const void*)k_ln_backward<T>, dim3(a.wgs), dim3(NT), pa, 0, st);
        if (e == hipSuccess && a.parts)
            e = hipLaunchKernel((const void*)k_ln_columns<T>, dim3((a.channels - 1) / NT + 1, a.parts), dim3(NT), pa, 0, st);
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
    // Lanes of a wave, up to four pieces each: more pieces a lane are more bytes in flight
    // for the registers that a row costs besides (us, so and with two where a wave has the lanes:
    // 262143 x 96 fp32 forward 34.9 and 47.4, 49147 x 1024 bf16 backward 65 and 73).  A row of more
    // than a wave's 256 pieces goes to a workgroup (6139 x 8192 bf16: forward 39.9, backward 83; in
    // strides 177 and 246), up to the 2048 that one of 512 threads holds.
    if (a.vec == 1) {
        a.lanes = 8;
    } else if (pieces <= 256) {
        a.lanes = 1;
        while (a.lanes * 4 < pieces) a.lanes *= 2;
    } else if (pieces <= 2048) {
        a.lanes = (pieces + 255) / 256 * 64;
    } else {
        a.threads = NT, a.lanes = NT, a.reps = 0;
        a.wgs = a.rows;
        if (sums) a.parts = a.rows < 256 ? (a.rows + 15) / 16 : 256;
        return;
    }
    a.reps = (pieces + a.lanes - 1) / a.lanes;
    // Forward: 256 threads, eight workgroups a compute unit.  Backward one of 512 threads (or two
    // of 256), so that few of them leave sums in the workspace (us, 512 and 256: 24570 x 2048 bf16
    // 63.6 and 67.4, 6139 x 8192 83 and 90; 196602 x 256 68.6 and 66.0).
    const int most = !backward ? NT : pieces > 128 ? 512 : NT;
    a.threads = a.lanes > most || (!backward && a.lanes > 64) ? a.lanes : most / a.lanes * a.lanes;
    const int per = a.threads / a.lanes;
    const long long all = ((long long)a.rows + per - 1) / per, cap = (backward ? 256ll * 512 : 2048ll * NT) / a.threads;
    a.wgs = (int)(all < cap ? all : cap);
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
