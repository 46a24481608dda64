// groupnorm.hip -- group norm with an activation over channels-last data.
//
// Bound by memory: x is read once (or twice), out written once, some ten
// operations a value.  A workgroup owns whole groups (`gb` neighbouring ones,
// up to 256 pieces of 16 bytes of a row) and rows of one item.  A thread keeps
// to one piece of the row, so that its channels, weights and groups are fixed,
// and steps over rows; neighbouring threads read neighbouring pieces.
//   one pass   the item's rows fit in the workgroup's registers: x is read once
//   two passes k_group<kStats> leaves each part's sums in the workspace,
//              k_group<kApply> adds them up and reads x again (from the 256 MB
//              cache where x fits it)
// Moments are sums of x and x^2 in 64 bits: the variance's difference then
// loses nothing that an fp32 input holds (a mean 10^6 standard deviations from
// zero costs 10^12 of 10^16), the order of summation does not show, and the
// matrix-free vector units add 64-bit values as fast as 32-bit ones.
#include "groupnorm.h"

#include "drain_common.h"

namespace ssla {
namespace {

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

// Sum over the w lanes (a power of two up to 64) that share a group.
__device__ __forceinline__ Sums lanes_sum(Sums a, int w) {
    for (int o = w >> 1; o; o >>= 1) {
        a.s += __shfl_xor(a.s, o);
        a.q += __shfl_xor(a.q, o);
    }
    return a;
}

template <class T, int V, int R, Mode MODE>
__global__ __launch_bounds__(R > 4 ? 1024 : 256) void k_group(const GroupNormArgs a) {
    extern __shared__ __align__(16) char smem[];
    typedef Piece<T, V> P;
    const int nt = blockDim.x, tid = threadIdx.x;
    const int cg = a.channels / a.groups;
    const int nparts = MODE == kOnePass ? 1 : a.parts;
    const int ib = blockIdx.x / nparts, part = blockIdx.x - ib * nparts;
    const int item = ib / a.blocks, block = ib - item * a.blocks;
    const int g0 = block * a.gb, ng = min(a.gb, a.groups - g0);
    // columns [c0, c1) in pieces p0 .. p0 + np - 1 (the outer ones may reach over)
    const long long c0 = (long long)g0 * cg, c1 = c0 + (long long)ng * cg;
    const int p0 = (int)(c0 / V), np = (int)((c1 + V - 1) / V) - p0;
    const int cols = min(np, nt), lanes = nt / cols;         // threads along a row, rows at a time
    const int py = tid / cols, px = tid - py * cols;
    const bool on = py < lanes;
    const int r0 = (int)((long long)a.rows * part / nparts), r1 = (int)((long long)a.rows * (part + 1) / nparts);
    const bool whole = cg % V == 0;                          // a piece lies in one group

    const T* x = (const T*)a.x + item * a.xn;
    const T* gate = a.gate ? (const T*)a.gate + item * a.gn : nullptr;
    T* out = (T*)a.out + item * a.on;

    // LDS: mean and 1 / sqrt(var + eps) of the groups (their sums while stats
    // run), then every thread's sums (one a piece, or one a channel)
    Sums* total = (Sums*)smem;
    float2* norm = (float2*)smem;
    Sums* own = total + a.gb;
    const int per = whole ? 1 : V;
    int w = 1;                                               // lanes that add up a group
    while (w < 64 && 2 * w * ng <= nt) w *= 2;

    P keep[R];
    if (MODE != kApply) {
        for (int g = tid; g < ng; g += nt) total[g] = Sums{0.0, 0.0};
        for (int pc = 0; pc < np; pc += cols) {              // once, where a row's pieces fit
            const int p = p0 + pc + px;
            const bool in = on && pc + px < np;
            Sums acc[V];
            #pragma unroll
            for (int i = 0; i < V; ++i) acc[i] = Sums{0.0, 0.0};
            if (MODE == kOnePass) {
                #pragma unroll
                for (int k = 0; k < R; ++k) {
                    const int row = py + k * lanes;
                    if (in && row < r1) keep[k] = *(const P*)(x + row * a.xr + (long long)p * V);
                }
                #pragma unroll
                for (int k = 0; k < R; ++k)
                    if (in && py + k * lanes < r1) {
                        #pragma unroll
                        for (int i = 0; i < V; ++i) {
                            const double v = (double)(float)keep[k].v[i];
                            acc[i].s += v;
                            acc[i].q = fma(v, v, acc[i].q);
                        }
                    }
            } else if (in) {
                for (int row = r0 + py; row < r1; row += R * lanes) {
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
                    own[py * cols + px] = acc[0];
                } else {
                    #pragma unroll
                    for (int i = 0; i < V; ++i) own[(py * cols + px) * V + i] = acc[i];
                }
            }
            __syncthreads();
            // a group's entries: its units (pieces or channels) of this stretch, of every row lane
            const int unit = whole ? cg / V : cg;
            const int lo = whole ? p0 + pc : (p0 + pc) * V, width = min(cols, np - pc) * per;
            for (int g = tid / w; g < ng; g += nt / w) {
                const long long first = (long long)(g0 + g) * unit;
                const int u0 = (int)max(0ll, first - lo), u1 = (int)min((long long)width, first + unit - lo);
                const int n = max(0, u1 - u0);
                Sums s = {0.0, 0.0};
                for (int i = tid % w; i < n * lanes; i += w) {
                    const int y = i / n, u = i - y * n;
                    const Sums t = own[y * cols * per + u0 + u];
                    s.s += t.s;
                    s.q += t.q;
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
    const double count = (double)cg * a.rows;
    for (int g = tid / w; g < ng; g += nt / w) {
        Sums s = {0.0, 0.0};
        if (MODE == kApply) {
            const Sums* ws = (const Sums*)a.ws + (long long)item * nparts * a.groups + g0 + g;
            for (int i = tid % w; i < nparts; i += w) {
                const Sums t = ws[(long long)i * a.groups];
                s.s += t.s;
                s.q += t.q;
            }
            s = lanes_sum(s, w);
        } else {
            s = total[g];
        }
        const double mean = s.s / count;
        double var = s.q / count - mean * mean;
        var = var < 0.0 ? 0.0 : var;                         // a NaN stays
        // in `total`'s place: one group's lanes read it above and write it here
        if (tid % w == 0) {
            if (MODE == kOnePass) {
                float2* f = (float2*)&total[g];
                *f = float2{(float)mean, (float)(1.0 / sqrt(var + (double)a.eps))};
            } else {
                norm[2 * g] = float2{(float)mean, (float)(1.0 / sqrt(var + (double)a.eps))};
            }
        }
    }
    __syncthreads();

    for (int pc = 0; pc < np; pc += cols) {
        const int p = p0 + pc + px;
        if (!on || pc + px >= np) continue;
        float mean[V], rstd[V], wt[V], bs[V];
        bool inside = true;
        #pragma unroll
        for (int i = 0; i < V; ++i) {
            const long long c = (long long)p * V + i;
            const bool mine = c >= c0 && c < c1;
            inside &= mine;
            const float2 f = norm[mine ? 2 * (int)((c - c0) / cg) : 0];
            mean[i] = f.x;
            rstd[i] = f.y;
            wt[i] = a.weight && mine ? (float)((const T*)a.weight)[c] : 1.0f;
            bs[i] = a.bias && mine ? (float)((const T*)a.bias)[c] : 0.0f;
        }
        auto finish = [&](int row, const P& px_, const P& pg) {
            P y;
            #pragma unroll
            for (int i = 0; i < V; ++i) {
                float v = fmaf(((float)px_.v[i] - mean[i]) * rstd[i], wt[i], bs[i]);
                v = gate ? v * activate((float)pg.v[i], a.act) : activate(v, a.act);
                y.v[i] = (T)v;
            }
            T* o = out + (long long)row * a.orow + (long long)p * V;
            if (inside) {
                *(P*)o = y;
            } else {
                #pragma unroll
                for (int i = 0; i < V; ++i) {
                    const long long c = (long long)p * V + i;
                    if (c >= c0 && c < c1) o[i] = y.v[i];
                }
            }
        };
        if (MODE == kOnePass) {
            #pragma unroll
            for (int k = 0; k < R; ++k) {
                const int row = py + k * lanes;
                if (row < r1) {
                    P pg{};
                    if (gate) pg = *(const P*)(gate + row * a.gr + (long long)p * V);
                    finish(row, keep[k], pg);
                }
            }
        } else {
            for (int row = r0 + py; row < r1; row += R * lanes) {
                P pg[R];
                #pragma unroll
                for (int k = 0; k < R; ++k)
                    if (row + k * lanes < r1) {
                        keep[k] = *(const P*)(x + (long long)(row + k * lanes) * a.xr + (long long)p * V);
                        if (gate)
                            pg[k] = *(const P*)(gate + (long long)(row + k * lanes) * a.gr + (long long)p * V);
                    }
                #pragma unroll
                for (int k = 0; k < R; ++k)
                    if (row + k * lanes < r1) finish(row + k * lanes, keep[k], pg[k]);
            }
        }
    }
}

template <class T, int V>
hipError_t launch(const GroupNormArgs& a, hipStream_t st) {
    GroupNormArgs args = a;
    void* pa[] = {&args};
    const int per = a.channels / a.groups % V ? V : 1;
    const unsigned lds = (unsigned)(sizeof(Sums) * ((size_t)a.gb + (size_t)a.threads * per));
    const long long wgs = (long long)a.n * a.blocks;
    if (!a.parts) {
        const void* f = a.threads > 256 ? (const void*)k_group<T, V, 16, kOnePass>
                        : a.reps > 1    ? (const void*)k_group<T, V, 4, kOnePass>
                                        : (const void*)k_group<T, V, 1, kOnePass>;
        return hipLaunchKernel(f, dim3((unsigned)wgs), dim3(a.threads), pa, lds, st);
    }
    const dim3 grid((unsigned)(wgs * a.parts));
    const hipError_t e = hipLaunchKernel((const void*)k_group<T, V, 4, kStats>, grid, dim3(a.threads), pa, lds, st);
    if (e != hipSuccess) return e;
    return hipLaunchKernel((const void*)k_group<T, V, 4, kApply>, grid, dim3(a.threads), pa, lds, st);
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
    unsigned long long bits = (unsigned long long)a.channels | a.xr | a.xn | a.orow | a.on | 16 / e;
    if (a.gate) bits |= (unsigned long long)(a.gr | a.gn);
    bits = bits * e | (unsigned long long)(size_t)a.x | (size_t)a.out | (size_t)a.gate;
    a.vec = (int)((bits & -bits) / e);
    const int cg = a.channels / a.groups;
    const int pieces = a.channels / a.vec;
    a.blocks = (pieces + 255) / 256;
    a.gb = (a.groups + a.blocks - 1) / a.blocks;
    a.blocks = (a.groups + a.gb - 1) / a.gb;
    // pieces of a workgroup's row; one more where its first channel is not a piece's
    const long long np = ((long long)a.gb * cg + a.vec - 1) / a.vec + (cg % a.vec && a.blocks > 1 ? 1 : 0);
    a.parts = 0;
    const bool wide = cg % a.vec == 0;      // 1024 threads' sums of every channel would not fit the LDS
    for (int nt = 64; nt <= (wide ? 1024 : 256); nt *= 4) {
        if (np > nt) continue;
        const long long reps = (a.rows + nt / np - 1) / (nt / np);
        if (reps > (nt == 64 ? 1 : nt == 256 ? 4 : 16)) continue;
        a.threads = nt;
        a.reps = (int)reps;
        return;
    }
    a.threads = 256;
    a.reps = 4;
    const long long lanes = np > 256 ? 1 : 256 / np;
    long long parts = 2048 / ((long long)a.n * a.blocks);
    const long long most = (a.rows + 4 * lanes - 1) / (4 * lanes);   // four rows a thread at least
    parts = parts < 1 ? 1 : parts > 128 ? 128 : parts;
    a.parts = (int)(parts > most ? most : parts);
}

hipError_t group_norm_launch(const GroupNormArgs& a, int dtype, hipStream_t st) {
    if (dtype == SSLA_F32) return launch_vec<float>(a, st);
    if (dtype == SSLA_BF16) return launch_vec<__bf16>(a, st);
    return launch_vec<_Float16>(a, st);
}

}  // namespace ssla
