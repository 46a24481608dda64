// groupnorm.hip -- group norm with an activation over channels-last data.
//
// Bound by memory: x is read once (or twice), out written once, some ten
// operations a value.  A workgroup owns whole groups (`gb` neighbouring ones,
// up to 256 pieces of 16 bytes of a row) and rows of one item.  A thread keeps
// to one piece of the row, so that its channels, weights and groups are fixed,
// and steps over rows; neighbouring threads read neighbouring pieces.
//   lanes      a group is small (a token's head): some lanes of a wave hold it,
//              and nothing but shuffles joins them; or a workgroup holds it
//              (k_group_lanes)
//   one pass   the item's rows fit in the workgroup's registers: x is read once
//   two passes k_group<kStats> leaves each part's sums in the workspace,
//              k_group<kApply> adds them up and reads x again (from the 256 MB
//              cache where x fits it)
// Moments are sums of x and x^2 in 64 bits: squares of finite values do not
// overflow, the variance's difference loses little (with a mean 10^6 standard
// deviations from zero 10^12 of 10^16), the order of summation does not show, and
// the conversions hide behind the loads.  k_group_lanes has a group's values in
// registers and takes the mean first, then squared differences from it, in 64
// bits too.  The mean is subtracted as two floats (norm_of).
// 16 items of 19200 rows of 96 fp32 channels (118 MB in, 118 out) take 74 us out of
// memory, 20 + 39 with x in the cache: three passes at 4.7 to 6 TB/s.  8191 tokens
// of 2048 bf16 channels in 16 groups with a gate (101 MB): 25 us, 4.0 TB/s.
#include "groupnorm.h"

#include <cmath>

#include "drain_common.h"
#include "norm.h"

namespace ssla {
namespace {

using ssla::lanes_sum;
using ssla::norm_of;

enum Mode { kOnePass, kStats, kApply };

struct Sums {
    double s, q;
};

template <class T, int V>
struct alignas(sizeof(T) * V) Piece {
    T v[V];
};

__device__ __forceinline__ float activate(float x, int act) {
    switch (act) {
        case SSLA_ACT_SILU: return x * sigmoid_fast(x);
        case SSLA_ACT_SIGMOID: return sigmoid_fast(x);
        case SSLA_ACT_RELU: return x < 0.0f ? 0.0f : x;      // a NaN stays
        default: return x;
    }
}

__device__ __forceinline__ Norm norm_of(Sums s, double inv_count, float eps) {
    const double mean = s.s * inv_count, var = fma(-mean, mean, s.q * inv_count);
    return norm_of(mean, var < 0.0 ? 0.0 : var, eps);        // a NaN stays
}

__device__ __forceinline__ Sums lanes_sum(Sums a, int w) {
    return Sums{lanes_sum(a.s, w), lanes_sum(a.q, w)};
}

// NT: most threads of a workgroup.
template <class T, int V, int R, int NT, Mode MODE>
__global__ __launch_bounds__(NT) void k_group(const GroupNormArgs a) {
    extern __shared__ __align__(16) char smem[];
    typedef Piece<T, V> P;
    const int nt = blockDim.x, tid = threadIdx.x;
    const int cg = a.channels / a.groups;
    const int nparts = MODE == kOnePass ? 1 : a.parts;
    const int ib = blockIdx.x / nparts, part = blockIdx.x - ib * nparts;
    const int item = ib / a.blocks, block = ib - item * a.blocks;
    const int g0 = block * a.gb, ng = min(a.gb, a.groups - g0);
    // columns [c0, c1) in pieces p0 .. p0 + np - 1 (the outer ones may reach over)
    const int c0 = g0 * cg, c1 = c0 + ng * cg;
    const int p0 = c0 / V, np = (c1 - 1) / V + 1 - p0;
    const int cols = min(np, nt), lanes = nt / cols;         // threads along a row, rows at a time
    const int py = tid / cols, px = tid - py * cols;
    const bool on = py < lanes;
    const int r0 = (int)((long long)a.rows * part / nparts), r1 = (int)((long long)a.rows * (part + 1) / nparts);
    const bool whole = cg % V == 0;                          // a piece lies in one group

    const T* x = (const T*)a.x + item * a.xn;
    const T* gate = a.gate ? (const T*)a.gate + item * a.gn : nullptr;
    T* out = (T*)a.out + item * a.on;

    // LDS: the groups' sums, then their mean and 1 / sqrt(var + eps); behind them
    // every thread's sums (one a piece, or one a channel), then the channels' table
    Sums* total = (Sums*)smem;
    Norm* norm = (Norm*)smem;
    static_assert(sizeof(Norm) == sizeof(Sums));
    Sums* own = total + a.gb;
    float* table = (float*)own;                              // hi, scale, bias of a stretch's channels
    const int width = cols * V;
    const int per = whole ? 1 : V;
    int w = 1;                                               // lanes that add up a group
    while (w < 64 && 2 * w * ng <= nt) w *= 2;

    // weight and bias of a channel of a stretch; each thread's first one is read ahead
    auto weight_of = [&](int ch) {
        const int c = p0 * V + ch;
        return a.weight && c >= c0 && c < c1 ? (float)((const T*)a.weight)[c] : 1.0f;
    };
    auto bias_of = [&](int ch) {
        const int c = p0 * V + ch;
        return a.bias && c >= c0 && c < c1 ? (float)((const T*)a.bias)[c] : 0.0f;
    };
    float w0 = 1.0f, b0 = 0.0f;
    if (MODE != kStats) w0 = weight_of(tid), b0 = bias_of(tid);

    // what the last step needs first is out before the sums: the gate's pieces of
    // the first rows, and x's where this pass has no sums of its own
    P keep[R], pgate[R];
    if (MODE != kStats && on) {
        #pragma unroll
        for (int k = 0; k < R; ++k) {
            const int row = r0 + py + k * lanes;
            if (row < r1) {
                if (gate) pgate[k] = *(const P*)(gate + row * a.gr + (long long)(p0 + px) * V);
                if (MODE == kApply) keep[k] = *(const P*)(x + row * a.xr + (long long)(p0 + px) * V);
            }
        }
    }
    if (MODE != kApply) {
        for (int g = tid; g < ng; g += nt) total[g] = Sums{0.0, 0.0};
        for (int pc = 0; pc < np; pc += cols) {              // once, where a row's pieces fit
            const int p = p0 + pc + px;
            const bool in = on && pc + px < np;
            Sums acc[V];
            #pragma unroll
            for (int i = 0; i < V; ++i) acc[i] = Sums{0.0, 0.0};
            if (in) {
                for (int row = r0 + py; row < r1; row += R * lanes) {      // one pass: once
                    #pragma unroll
                    for (int k = 0; k < R; ++k)
                        if (row + k * lanes < r1)
                            keep[k] = *(const P*)(x + (long long)(row + k * lanes) * a.xr + (long long)p * V);
                    #pragma unroll
                    for (int k = 0; k < R; ++k)
                        if (row + k * lanes < r1) {
                            #pragma unroll
                            for (int i = 0; i < V; ++i) {
                                const double v = (double)(float)keep[k].v[i];
                                acc[i].s += v;
                                acc[i].q = fma(v, v, acc[i].q);
                            }
                        }
                    if (MODE == kOnePass) break;
                }
            }
            __syncthreads();                                 // `total` is set, `own` free
            if (on) {
                if (whole) {
                    #pragma unroll
                    for (int i = 1; i < V; ++i) {
                        acc[0].s += acc[i].s;
                        acc[0].q += acc[i].q;
                    }
                    own[tid] = acc[0];
                } else {
                    #pragma unroll
                    for (int i = 0; i < V; ++i) own[tid * V + i] = acc[i];
                }
            }
            __syncthreads();
            // a group's entries: its units (pieces or channels) of this stretch, of every row lane
            const int unit = whole ? cg / V : cg;
            const int lo = whole ? p0 + pc : (p0 + pc) * V, wide = min(cols, np - pc) * per;
            for (int g = tid / w; g < ng; g += nt / w) {
                const int first = (g0 + g) * unit;
                const int u0 = max(0, first - lo), u1 = min(wide, first + unit - lo), n = max(0, u1 - u0);
                Sums s = {0.0, 0.0};
                if (n) {
                    int y = tid % w / n, u = tid % w - y * n;      // entry (row lane y, unit u)
                    const int dy = w / n, du = w - dy * n;
                    for (; y < lanes; y += dy, u += du) {
                        if (u >= n) {
                            u -= n;
                            if (++y >= lanes) break;
                        }
                        const Sums t = own[y * cols * per + u0 + u];
                        s.s += t.s;
                        s.q += t.q;
                    }
                }
                s = lanes_sum(s, w);
                if (tid % w == 0) {
                    total[g].s += s.s;
                    total[g].q += s.q;
                }
            }
        }
        __syncthreads();
    }
    if (MODE == kStats) {
        Sums* ws = (Sums*)a.ws + ((long long)item * nparts + part) * a.groups + g0;
        for (int g = tid; g < ng; g += nt) ws[g] = total[g];
        return;
    }

    // ---- means and scales -----------------------------------------------------
    for (int g = tid / w; g < ng; g += nt / w) {
        Sums s = {0.0, 0.0};
        if (MODE == kApply) {
            const Sums* ws = (const Sums*)a.ws + (long long)item * nparts * a.groups + g0 + g;
            for (int i = tid % w; i < nparts; i += 4 * w) {
                Sums t[4];
                #pragma unroll
                for (int u = 0; u < 4; ++u)
                    t[u] = i + u * w < nparts ? ws[(long long)(i + u * w) * a.groups] : Sums{0.0, 0.0};
                #pragma unroll
                for (int u = 0; u < 4; ++u) {
                    s.s += t[u].s;
                    s.q += t[u].q;
                }
            }
            s = lanes_sum(s, w);
        } else {
            s = total[g];
        }
        // in `total`'s place: one group's lanes read it above and write it here
        if (tid % w == 0) norm[g] = norm_of(s, a.inv_count, a.eps);
    }
    __syncthreads();

    for (int pc = 0; pc < np; pc += cols) {
        if (pc) __syncthreads();                             // the last stretch's readers are done
        for (int ch = tid; ch < width; ch += nt) {
            const int at = pc * V + ch, c = p0 * V + at;
            const bool mine = c >= c0 && c < c1, ahead = at == tid;
            const Norm f = norm[mine ? (c - c0) / cg : 0];
            const float scale = f.scale * (ahead ? w0 : weight_of(at));
            table[ch] = f.hi;
            table[width + ch] = scale;
            table[2 * width + ch] = fmaf(-f.lo, scale, ahead ? b0 : bias_of(at));
        }
        __syncthreads();
        const int p = p0 + pc + px;
        if (!on || pc + px >= np) continue;
        float hi[V], scale[V], bias[V];
        #pragma unroll
        for (int i = 0; i < V; ++i) {
            hi[i] = table[px * V + i];
            scale[i] = table[width + px * V + i];
            bias[i] = table[2 * width + px * V + i];
        }
        const bool inside = p * V >= c0 && p * V + V <= c1;
        auto finish = [&](int row, const P& in, const P& pg) {
            P y;
            #pragma unroll
            for (int i = 0; i < V; ++i) {
                const float v = fmaf(fmaf((float)in.v[i], kDown, -hi[i]), scale[i], bias[i]);
                y.v[i] = (T)(gate ? v * activate((float)pg.v[i], a.act) : activate(v, a.act));
            }
            T* o = out + (long long)row * a.orow + (long long)p * V;
            if (inside) {
                *(P*)o = y;
            } else {
                #pragma unroll
                for (int i = 0; i < V; ++i)
                    if (p * V + i >= c0 && p * V + i < c1) o[i] = y.v[i];
            }
        };
        for (int row = r0 + py; row < r1; row += R * lanes) {              // one pass: once
            if (MODE == kApply && (pc || row != r0 + py)) {
                #pragma unroll
                for (int k = 0; k < R; ++k)
                    if (row + k * lanes < r1) {
                        keep[k] = *(const P*)(x + (long long)(row + k * lanes) * a.xr + (long long)p * V);
                        if (gate)
                            pgate[k] = *(const P*)(gate + (long long)(row + k * lanes) * a.gr + (long long)p * V);
                    }
            }
            #pragma unroll
            for (int k = 0; k < R; ++k)
                if (row + k * lanes < r1) finish(row + k * lanes, keep[k], pgate[k]);
            if (MODE == kOnePass) break;
        }
    }
}

// What the compiler has made of p's values ends here.  It would otherwise keep all of
// them in 64 bits from one use to the next: 220 registers instead of 146 for four pieces of
// eight values, and 1100 us instead of 784 for 4096 items of 64 rows of 2048 bf16
// channels in 16 groups.
template <class P>
__device__ __forceinline__ void opaque(P& p) {
    constexpr int N = sizeof(P) / 4;
    if constexpr (N == 0) {
        unsigned x = __builtin_bit_cast(unsigned short, p);
        asm("" : "+v"(x));
        p = __builtin_bit_cast(P, (unsigned short)x);
    } else {
        unsigned x[N];
        __builtin_memcpy(x, &p, sizeof(P));
        #pragma unroll
        for (int i = 0; i < N; ++i) asm("" : "+v"(x[i]));
        __builtin_memcpy(&p, x, sizeof(P));
    }
}

// Pieces a thread of a 1024-thread workgroup keeps: what 128 registers hold.
template <int V> constexpr int kWideReps = V == 8 ? 2 : 4;

// ---- small groups --------------------------------------------------------------
// `w` threads hold a group of one item, R pieces each: some lanes of a wave, with
// neighbouring lanes' groups neighbours, or (WHOLE) a workgroup.  The mean first, then the sum of squared differences from it.
template <int NT, bool WHOLE>
__device__ __forceinline__ double group_sum(double s, int w, double* waves) {
    s = lanes_sum(s, WHOLE ? 64 : w);
    if (WHOLE) {
        if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = s;
        __syncthreads();
        s = waves[0];
        #pragma unroll
        for (int i = 1; i < NT / 64; ++i) s += waves[i];
    }
    return s;
}

template <class T, int V, int R, int NT, bool WHOLE>
__global__ __launch_bounds__(NT) void k_group_lanes(const GroupNormArgs a) {
    typedef Piece<T, V> P;
    __shared__ double sums[NT / 64], squares[NT / 64];
    const int w = WHOLE ? NT : a.reps;                       // threads of a group
    const int l = threadIdx.x & (w - 1);
    const long long ig = (long long)blockIdx.x * (NT / w) + threadIdx.x / w;
    const long long item = ig / a.groups;
    const int group = (int)(ig - item * a.groups);
    const bool on = item < a.n;
    const int cg = a.channels / a.groups, pr = cg / V;       // pieces of a row of the group
    const int pieces = pr * a.rows;
    const T* x = (const T*)a.x + item * a.xn + (long long)group * cg;
    const T* gate = a.gate ? (const T*)a.gate + item * a.gn + (long long)group * cg : nullptr;
    T* out = (T*)a.out + item * a.on + (long long)group * cg;

    P px[R], pg[R], pw[R], pb[R];
    #pragma unroll
    for (int k = 0; k < R; ++k) {
        const int i = l + k * w;
        #pragma unroll
        for (int j = 0; j < V; ++j) px[k].v[j] = pg[k].v[j] = pb[k].v[j] = (T)0.0f, pw[k].v[j] = (T)1.0f;
        if (on && i < pieces) {
            const int row = i / pr, p = (i - row * pr) * V;
            px[k] = *(const P*)(x + row * a.xr + p);
            if (gate) pg[k] = *(const P*)(gate + row * a.gr + p);
            if (k && w % pr == 0) {                          // a thread's pieces have the same channels
                pw[k] = pw[0];
                pb[k] = pb[0];
            } else {
                if (a.weight) pw[k] = *(const P*)((const T*)a.weight + (long long)group * cg + p);
                if (a.bias) pb[k] = *(const P*)((const T*)a.bias + (long long)group * cg + p);
            }
        }
    }
    double s = 0.0;
    #pragma unroll
    for (int k = 0; k < R; ++k)
        #pragma unroll
        for (int j = 0; j < V; ++j) s += (double)(float)px[k].v[j];
    #pragma unroll
    for (int k = 0; k < R; ++k) opaque(px[k]);
    s = group_sum<NT, WHOLE>(s, w, sums);
    const double mean = s * a.inv_count;
    double q = 0.0;
    #pragma unroll
    for (int k = 0; k < R; ++k)
        if (l + k * w < pieces) {
            #pragma unroll
            for (int j = 0; j < V; ++j) {
                const double d = (double)(float)px[k].v[j] - mean;
                q = fma(d, d, q);
            }
        }
    q = group_sum<NT, WHOLE>(q, w, squares);
    #pragma unroll
    for (int k = 0; k < R; ++k) opaque(px[k]);
    const Norm f = norm_of(mean, q * a.inv_count, a.eps);
    const float low = -f.lo * f.scale;
    #pragma unroll
    for (int k = 0; k < R; ++k) {
        const int i = l + k * w;
        if (on && i < pieces) {
            const int row = i / pr, p = (i - row * pr) * V;
            P y;
            #pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = fmaf(fmaf((float)px[k].v[j], kDown, -f.hi), f.scale, low);
                const float v = fmaf(d, (float)pw[k].v[j], (float)pb[k].v[j]);
                y.v[j] = (T)(gate ? v * activate((float)pg[k].v[j], a.act) : activate(v, a.act));
            }
            *(P*)(out + row * a.orow + p) = y;
        }
    }
}

// LDS of a workgroup of k_group: the groups' sums, and the larger of the threads'
// sums (of every channel, where groups do not begin with pieces) and the table.
size_t group_norm_lds(const GroupNormArgs& a, int threads, long long np) {
    const size_t sums = (size_t)threads * (a.channels / a.groups % a.vec ? a.vec : 1) * sizeof(Sums);
    const size_t table = (size_t)(np < threads ? np : threads) * a.vec * 3 * sizeof(float);
    return sizeof(Sums) * (size_t)a.gb + (sums > table ? sums : table);
}

template <class T, int V>
hipError_t launch(const GroupNormArgs& a, hipStream_t st) {
    if (a.kind == kGroupLanes) {
        GroupNormArgs args = a;
        void* pa[] = {&args};
        const int nt = a.reps > 256 ? 1024 : 256;
        const long long per = nt / a.reps, wgs = ((long long)a.n * a.groups + per - 1) / per;
        const void* f = a.reps > 256  ? (const void*)k_group_lanes<T, V, kWideReps<V>, 1024, true>
                        : a.reps > 64 ? a.threads > 1 ? (const void*)k_group_lanes<T, V, 4, 256, true>
                                                      : (const void*)k_group_lanes<T, V, 1, 256, true>
                        : a.threads == 1 ? (const void*)k_group_lanes<T, V, 1, 256, false>
                        : a.threads == 2 ? (const void*)k_group_lanes<T, V, 2, 256, false>
                                         : (const void*)k_group_lanes<T, V, 4, 256, false>;
        return hipLaunchKernel(f, dim3((unsigned)wgs), dim3(nt), pa, 0, st);
    }
    GroupNormArgs args = a;
    void* pa[] = {&args};
    const size_t lds = group_norm_lds(a, a.threads, a.np);
    const long long wgs = (long long)a.n * a.blocks;
    if (a.kind == kGroupOnePass) {
        const void* f = a.threads > 256 ? (const void*)k_group<T, V, kWideReps<V>, 1024, kOnePass>
                        : a.reps > 1    ? (const void*)k_group<T, V, 4, 256, kOnePass>
                                        : (const void*)k_group<T, V, 1, 256, kOnePass>;
        if (lds > 65536) {
            const hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
            if (e != hipSuccess) return e;
        }
        return hipLaunchKernel(f, dim3((unsigned)wgs), dim3(a.threads), pa, lds, st);
    }
    const dim3 grid((unsigned)(wgs * a.parts));
    const void* f = (const void*)k_group<T, V, 4, 256, kStats>;
    const hipError_t e = hipLaunchKernel(f, grid, dim3(a.threads), pa, lds, st);
    if (e != hipSuccess) return e;
    return hipLaunchKernel((const void*)k_group<T, V, 4, 256, kApply>, grid, dim3(a.threads), pa, lds, st);
}

template <class T>
hipError_t launch_vec(const GroupNormArgs& a, hipStream_t st) {
    if (a.vec == 1) return launch<T, 1>(a, st);
    if (a.vec == 2) return launch<T, 2>(a, st);
    if (a.vec == 4) return launch<T, 4>(a, st);
    return launch<T, 16 / sizeof(T)>(a, st);
}

}  // namespace

void group_norm_plan(GroupNormArgs& a, int dtype) {
    const int e = dtype == SSLA_F32 ? 4 : 2;
    // pieces: 16 bytes, or what the addresses, strides and rows are multiples of
    unsigned long long bits = (unsigned long long)a.channels | a.orow | a.xr | 16 / e;
    if (a.n > 1) bits |= (unsigned long long)(a.xn | a.on);
    if (a.gate) bits |= (unsigned long long)(a.gr | (a.n > 1 ? a.gn : 0));
    bits = bits * e | (unsigned long long)(size_t)a.x | (size_t)a.out | (size_t)a.gate | (size_t)a.weight |
           (size_t)a.bias;
    a.vec = (int)((bits & -bits) / e);
    const int cg = a.channels / a.groups;
    const double count = (double)cg * a.rows;
    a.inv_count = 1.0 / count;
    a.parts = 0;
    // lanes of a wave, one to four pieces each, hold a group: as few pieces as
    // 64 lanes allow (a token's groups of 128 bf16 channels: 16 lanes, one piece)
    int v = a.vec;
    while (cg % v) v /= 2;
    const long long pieces = (long long)a.rows * (cg / v);
    // A workgroup for each larger group, while what its rows' 128-byte lines hold
    // besides, which the groups beside it read again, is small: one item of 320 rows
    // of 48 fp32 channels in 8 groups takes 4.3 us instead of 10.0 by whole rows, 64
    // of them (17 MB besides) 9.2 instead of 10.7, 128 14 instead of 11; 4096 rows of
    // 96 channels in 24 groups (11 MB) 9.8 instead of 10.6, two such items 13.1
    // instead of 10.9.  Groups of whole lines: 256 tokens of 16384 fp32 channels in 8
    // groups 10.8 instead of 65, 64 items of 64 rows of 2048 bf16 channels in 16
    // groups 16.8 instead of 22.6.  The number of items is not looked at: 4096 such items,
    // 2 GB, take 784 us, 684 by whole rows.
    // A piece a thread, or up to four (two) of 256 (1024) threads; more than 512
    // groups keep to 256 threads (256 tokens of 65536 bf16 channels in 16 groups: 31
    // us, with 1024 threads 60).
    const long long rows = (long long)a.n * a.groups * a.rows, width = (long long)cg * e;
    const bool few = rows * ((width + 127) / 128 * 128 - width) <= 8 << 20;
    for (int r = 1; r <= (few ? 1 : 4); r *= 2)
        if (pieces <= 64 * r) {
            int w = 1;
            while (w * r < pieces) w *= 2;
            a.kind = kGroupLanes;
            a.vec = v;
            a.reps = w;
            a.threads = r;
            a.gb = a.blocks = 1;
            return;
        }
    if (few && pieces <= 1024 * (v == 8 ? 2 : 4)) {
        a.kind = kGroupLanes;
        a.vec = v;
        a.threads = pieces <= 256 ? 1 : 4;
        a.reps = pieces <= 256 || (pieces <= 1024 && (long long)a.n * a.groups > 512) ? 256 : 1024;
        a.gb = a.blocks = 1;
        return;
    }
    const int row = a.channels / a.vec;
    a.blocks = (row + 255) / 256;
    a.gb = (a.groups + a.blocks - 1) / a.blocks;
    a.blocks = (a.groups + a.gb - 1) / a.gb;
    // pieces of a workgroup's row; one more where its first channel is not a piece's
    const long long np = ((long long)a.gb * cg + a.vec - 1) / a.vec + (cg % a.vec && a.blocks > 1 ? 1 : 0);
    a.np = (int)np;
    a.kind = kGroupOnePass;
    for (int nt = 256; nt <= 1024; nt *= 4) {
        if (np > nt || group_norm_lds(a, nt, np) > 144 * 1024) continue;
        const long long reps = (a.rows + nt / np - 1) / (nt / np);
        if (reps > (nt == 1024 && a.vec == 8 ? kWideReps<8> : 4)) continue;
        a.threads = nt;
        a.reps = (int)reps;
        return;
    }
    a.kind = kGroupTwoPass;
    a.threads = 256;
    a.reps = 4;
    const long long lanes = np > 256 ? 1 : 256 / np;
    long long parts = 2048 / ((long long)a.n * a.blocks);
    const long long most = (a.rows + 4 * lanes - 1) / (4 * lanes);   // four rows a thread at least
    // Beyond 128 parts, as many as cost a workgroup of the second launch no more sums to
    // read than values, while that is 1024 workgroups in all: 40000 rows of 512 bf16
    // channels in 32 groups take 106 us in 128 parts, 63 in the 282 of this rule, 51 in
    // 512, 84 in 1024, two such items 108, 74, 75, 152; one of 19200 rows of 96 fp32
    // channels in 8 groups 16.9, 13.6 (240), 14.0, 14.0.
    const long long even = (long long)sqrt((double)a.rows * (double)cg * e / sizeof(Sums));
    const long long share = 1024 / ((long long)a.n * a.blocks), few_sums = even < share ? even : share;
    const long long cap = few_sums > 128 ? few_sums : 128;
    parts = parts < 1 ? 1 : parts > cap ? cap : parts;
    a.parts = (int)(parts > most ? most : parts);
}

hipError_t group_norm_launch(const GroupNormArgs& a, int dtype, hipStream_t st) {
    if (dtype == SSLA_F32) return launch_vec<float>(a, st);
    if (dtype == SSLA_BF16) return launch_vec<__bf16>(a, st);
    return launch_vec<_Float16>(a, st);
}

}  // namespace ssla
