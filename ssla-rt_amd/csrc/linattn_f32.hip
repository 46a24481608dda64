// linattn_f32.hip -- chunked linear attention over fp32 tokens on the
// 16 x 16 x 4 fp32 matrix instruction, the chain of segment states and the
// form for single tokens.
//
// The chunked kernel is the one of linattn16.h without the splits: everything
// transposed, the state S[d][e] in D registers (row 4 g + r, column m of lane
// 16 g + m), where register r is the A operand of the step that contracts
// d = 4 g + r over the lane groups g; Q, K and P are read in the same order
// (one float4 a lane, four steps).  Chunks of 32 tokens: what a chunk costs
// beside the products with the state grows with its length, and nothing has
// to be converted per chunk, as the 16-bit kernel's state has.
#include "linattn.h"

namespace ssla {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));

constexpr int C = 32;            // tokens of a chunk
constexpr int PAD = 4;           // floats behind a row in LDS: four rows apart, 16 banks apart

__device__ __forceinline__ f4 mma(float a, float b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

template <int DK, int NW>
struct Lds {
    static constexpr int DV = 32 * NW;
    static constexpr int QS = DK + PAD, VS = DV + PAD, PS = C + PAD;
    float q[C * QS];
    float k[C * QS];
    float v[C * VS];
    float p[C * PS];
    float bhi[C], blo[C], eb[C], w[C];
    int bad[DV];                 // first token whose v is not finite, per column
    int any_bad;
};

__device__ __forceinline__ bool not_finite(float x) {
    return (__builtin_bit_cast(unsigned, x) & 0x7f800000u) == 0x7f800000u;
}

template <int DK, int NW, bool FULL>
__global__ __launch_bounds__(64 * NW, 1) void k_linattn32(const LinAttnArgs a) {
    typedef Lds<DK, NW> L;
    constexpr int NT = 64 * NW, DT = DK / 16;
    constexpr int QC = DK / 4, QP = (C * QC + NT - 1) / NT;     // 16-byte pieces: a row, a thread
    constexpr int VC = L::DV / 4, VP = C * VC / NT;
    static_assert(C * QC % NT == 0 && C * VC % NT == 0, "whole pieces a thread");
    extern __shared__ __align__(16) char smem[];
    L& lds = *reinterpret_cast<L*>(smem);

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int m = lane & 15, g = lane >> 4;
    const int per = a.heads * a.slices;
    const int j_seg = blockIdx.x / per, hs = blockIdx.x - j_seg * per;
    const int head = hs / a.slices, slice = hs - head * a.slices;
    const Segment sg = linattn_segment(a, j_seg, lane);
    if (!sg.ok) return;
    const bool last = sg.t1 >= sg.len;
    if (!FULL && last) return;                 // nothing follows this segment
    const int slot = linattn_slot(a, sg.seq);
    if (slot < 0) return;
    const int e0 = slice * L::DV + wave * 32;  // the wave's first column

    const float* qb = (const float*)a.q + (long long)(head / a.rep) * a.qh;
    const float* kb = (const float*)a.k + (long long)(head / a.rep) * a.kh;
    const float* vb = (const float*)a.v + (long long)head * a.vh + slice * L::DV;
    const float* gb = a.g + (long long)head * a.gh;
    const int dvs = a.dv - slice * L::DV;      // columns of v from the slice's first

    f4 S[DT][2];
    const long long hstate = (long long)head * a.dk * a.dv;
    {
        const float* src = nullptr;
        if (FULL) {
            if (sg.index > 0) src = a.ws_state + (long long)j_seg * a.heads * a.dk * a.dv + hstate;
            else if (a.s_in) src = a.s_in + (long long)slot * a.s_stride + hstate;
        }
        #pragma unroll
        for (int dt = 0; dt < DT; ++dt)
            #pragma unroll
            for (int et = 0; et < 2; ++et)
                #pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int d = 16 * dt + 4 * g + r, e = e0 + 16 * et + m;
                    S[dt][et][r] = src && d < a.dk && e < a.dv ? src[(long long)d * a.dv + e] : 0.0f;
                }
    }

    f4 rq[FULL ? QP : 1], rk[QP], rv[VP];
    float rg = 0.0f;
    auto piece = [&](const float* base, long long stride, int idx, int cols, int per_row, int n) -> f4 {
        const int row = idx / per_row, c = (idx - row * per_row) * 4;
        f4 x = {0.0f, 0.0f, 0.0f, 0.0f};
        if (row < n && c < cols) {
            const float* p = base + row * stride + c;
            if (a.vec_in) {
                x = *(const f4*)p;
            } else {
                #pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (c + i < cols) x[i] = p[i];
            }
        }
        return x;
    };
    auto load = [&](int t) {
        const int n = sg.t1 - t;
        const long long row = sg.row + t;
        #pragma unroll
        for (int p = 0; p < QP; ++p) {
            rk[p] = piece(kb + row * a.kt, a.kt, tid + p * NT, a.dk, QC, n);
            if (FULL) rq[p] = piece(qb + row * a.qt, a.qt, tid + p * NT, a.dk, QC, n);
        }
        #pragma unroll
        for (int p = 0; p < VP; ++p) rv[p] = piece(vb + row * a.vt, a.vt, tid + p * NT, dvs, VC, n);
        rg = lane < C && lane < n ? gb[(row + lane) * a.gt] : 0.0f;
    };

    if (FULL) {     // the tile of P above the diagonal is never written again
        for (int i = tid; i < C * L::PS; i += NT) lds.p[i] = 0.0f;
    }
    float decay = 1.0f;
    if (sg.t0 < sg.t1) load(sg.t0);
    for (int t = sg.t0; t < sg.t1; t += C) {
        const int n = min(C, sg.t1 - t);
        __syncthreads();                       // the last chunk's readers are done
        if (tid == 0) lds.any_bad = 0;
        if (tid < L::DV) lds.bad[tid] = C;
        if (wave == 0) {
            double b = rg < kMinLogDecay ? kMinLogDecay : rg;
            #pragma unroll
            for (int o = 1; o < C; o <<= 1) {
                const double u = __shfl_up(b, o);
                if (lane >= o) b += u;
            }
            const double end = __shfl(b, C - 1);
            const float hi = (float)b;
            if (lane < C) {
                lds.bhi[lane] = hi;
                lds.blo[lane] = (float)(b - (double)hi);
                lds.eb[lane] = __expf(hi);
                lds.w[lane] = __expf((float)(end - b));
            }
        }
        __syncthreads();
        #pragma unroll
        for (int p = 0; p < QP; ++p) {
            const int idx = tid + p * NT, row = idx / QC, c = (idx - row * QC) * 4;
            *(f4*)&lds.k[row * L::QS + c] = rk[p];
            if (FULL) *(f4*)&lds.q[row * L::QS + c] = rq[p];
        }
        #pragma unroll
        for (int p = 0; p < VP; ++p) {
            const int idx = tid + p * NT, row = idx / VC, c = (idx - row * VC) * 4;
            f4 x = rv[p];
            // see linattn16.h: infinities and NaN of v act through `bad`
            #pragma unroll
            for (int i = 0; i < 4; ++i)
                if (not_finite(x[i])) {
                    lds.any_bad = 1;
                    atomicMin(&lds.bad[c + i], row);
                    x[i] = 0.0f;
                }
            *(f4*)&lds.v[row * L::VS + c] = x;
        }
        __syncthreads();
        if (t + C < sg.t1) load(t + C);

        // v of the wave's columns: column m, token 16 jt + 4 g + r
        float vf[2][2][4];
        #pragma unroll
        for (int et = 0; et < 2; ++et)
            #pragma unroll
            for (int jt = 0; jt < 2; ++jt)
                #pragma unroll
                for (int r = 0; r < 4; ++r)
                    vf[et][jt][r] = lds.v[(16 * jt + 4 * g + r) * L::VS + wave * 32 + 16 * et + m];

        if (FULL) {
            f4 O[2][2];
            // ---- P^T = K Q^T: three tiles on and below the diagonal ---------
            for (int u = wave; u < 3; u += NW) {
                const int it = u >= 1 ? 1 : 0, jt = u - it;
                f4 acc[2] = {};
                #pragma unroll
                for (int s = 0; s < DT; ++s) {
                    const f4 ka = *(const f4*)&lds.k[(16 * jt + m) * L::QS + 16 * s + 4 * g];
                    const f4 qa = *(const f4*)&lds.q[(16 * it + m) * L::QS + 16 * s + 4 * g];
                    #pragma unroll
                    for (int r = 0; r < 4; ++r) acc[r & 1] = mma(ka[r], qa[r], acc[r & 1]);
                }
                const int i = 16 * it + m, j = 16 * jt + 4 * g;
                const f4 jh = *(const f4*)&lds.bhi[j], jl = *(const f4*)&lds.blo[j];
                const float ih = lds.bhi[i], il = lds.blo[i];
                f4 p;
                #pragma unroll
                for (int r = 0; r < 4; ++r)
                    p[r] = j + r <= i ? (acc[0][r] + acc[1][r]) * __expf((ih - jh[r]) + (il - jl[r])) : 0.0f;
                *(f4*)&lds.p[i * L::PS + j] = p;
            }
            // ---- O^T = S^T Q^T ------------------------------------------------
            #pragma unroll
            for (int et = 0; et < 2; ++et)
                #pragma unroll
                for (int it = 0; it < 2; ++it) O[et][it] = f4{0.0f, 0.0f, 0.0f, 0.0f};
            #pragma unroll
            for (int s = 0; s < DT; ++s) {
                f4 qf[2];
                #pragma unroll
                for (int it = 0; it < 2; ++it)
                    qf[it] = *(const f4*)&lds.q[(16 * it + m) * L::QS + 16 * s + 4 * g];
                #pragma unroll
                for (int r = 0; r < 4; ++r)
                    #pragma unroll
                    for (int et = 0; et < 2; ++et)
                        #pragma unroll
                        for (int it = 0; it < 2; ++it) O[et][it] = mma(S[s][et][r], qf[it][r], O[et][it]);
            }
            #pragma unroll
            for (int it = 0; it < 2; ++it) {
                const float eb = lds.eb[16 * it + m];
                #pragma unroll
                for (int et = 0; et < 2; ++et) O[et][it] *= eb;
            }
            __syncthreads();                   // P is whole
            // ---- O^T += V^T P^T -------------------------------------------------
            #pragma unroll
            for (int jt = 0; jt < 2; ++jt)
                #pragma unroll
                for (int it = jt; it < 2; ++it) {
                    const f4 p = *(const f4*)&lds.p[(16 * it + m) * L::PS + 16 * jt + 4 * g];
                    #pragma unroll
                    for (int r = 0; r < 4; ++r)
                        #pragma unroll
                        for (int et = 0; et < 2; ++et) O[et][it] = mma(vf[et][jt][r], p[r], O[et][it]);
                }
            if (lds.any_bad) {
                #pragma unroll
                for (int et = 0; et < 2; ++et)
                    #pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int first = lds.bad[wave * 32 + 16 * et + 4 * g + r];
                        #pragma unroll
                        for (int it = 0; it < 2; ++it)
                            if (16 * it + m >= first) O[et][it][r] = __builtin_nanf("");
                    }
            }
            #pragma unroll
            for (int it = 0; it < 2; ++it) {
                const int i = 16 * it + m;
                if (i < n) {
                    float* p = (float*)a.out + (sg.row + t + i) * a.ot + (long long)head * a.oh;
                    #pragma unroll
                    for (int et = 0; et < 2; ++et) {
                        const int e = e0 + 16 * et + 4 * g;
                        const f4 y = a.scale * O[et][it];
                        if (a.vec_out) {
                            if (e < a.dv) *(f4*)(p + e) = y;
                        } else {
                            #pragma unroll
                            for (int r = 0; r < 4; ++r)
                                if (e + r < a.dv) p[e + r] = y[r];
                        }
                    }
                }
            }
        }

        // ---- S = exp(b_32) S + K^T (w v) ----------------------------------------
        const float eC = lds.eb[C - 1];
        decay *= eC;
        if (!FULL || !last || t + C < sg.t1 || a.s_out) {
            #pragma unroll
            for (int dt = 0; dt < DT; ++dt)
                #pragma unroll
                for (int et = 0; et < 2; ++et) S[dt][et] *= eC;
            #pragma unroll
            for (int jt = 0; jt < 2; ++jt) {
                const f4 w = *(const f4*)&lds.w[16 * jt + 4 * g];
                #pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float x0 = vf[0][jt][r] * w[r], x1 = vf[1][jt][r] * w[r];
                    #pragma unroll
                    for (int dt = 0; dt < DT; ++dt) {
                        const float kf = lds.k[(16 * jt + 4 * g + r) * L::QS + 16 * dt + m];
                        S[dt][0] = mma(kf, x0, S[dt][0]);
                        S[dt][1] = mma(kf, x1, S[dt][1]);
                    }
                }
            }
            if (lds.any_bad) {
                #pragma unroll
                for (int et = 0; et < 2; ++et)
                    if (lds.bad[wave * 32 + 16 * et + m] < C) {
                        #pragma unroll
                        for (int dt = 0; dt < DT; ++dt)
                            #pragma unroll
                            for (int r = 0; r < 4; ++r) S[dt][et][r] = __builtin_nanf("");
                    }
            }
        }
    }

    float* dst = nullptr;
    if (!FULL) {
        const long long at = (long long)j_seg * a.heads + head;
        dst = a.ws_state + (long long)j_seg * a.heads * a.dk * a.dv + hstate;
        if (slice == 0 && tid == 0) a.ws_decay[at] = decay;
    } else if (last && a.s_out) {
        dst = a.s_out + (long long)slot * a.s_stride + hstate;
    }
    if (dst) {
        #pragma unroll
        for (int dt = 0; dt < DT; ++dt)
            #pragma unroll
            for (int et = 0; et < 2; ++et)
                #pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int d = 16 * dt + 4 * g + r, e = e0 + 16 * et + m;
                    if (d < a.dk && e < a.dv) dst[(long long)d * a.dv + e] = S[dt][et][r];
                }
    }
}

// ---- the states before each segment ----------------------------------------
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
        n = (l + (1 << a.seg_shift) - 1) >> a.seg_shift;
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

// ---- one token a sequence -------------------------------------------------------
// Reads and writes each state once, 8 bytes a state value and nothing to win
// from arithmetic: bound by memory.  A workgroup owns one head of one sequence
// and 64 columns of its state; a wave takes every fourth row.
template <class T>
__global__ __launch_bounds__(256) void k_linattn_step(const LinAttnArgs a) {
    __shared__ float part[4][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wide = (a.dv + 63) / 64, sh = blockIdx.x / wide;
    const int seq = sh / a.heads, head = sh - seq * a.heads;
    const int slot = linattn_slot(a, seq);
    if (slot < 0) return;
    const int e = (blockIdx.x - sh * wide) * 64 + lane;
    const bool in = e < a.dv;
    const T* q = (const T*)a.q + seq * a.qt + (long long)(head / a.rep) * a.qh;
    const T* k = (const T*)a.k + seq * a.kt + (long long)(head / a.rep) * a.kh;
    const float v = in ? (float)((const T*)a.v)[seq * a.vt + (long long)head * a.vh + e] : 0.0f;
    const float dec = expf(a.g[seq * a.gt + (long long)head * a.gh]);
    const long long at = (long long)slot * a.s_stride + (long long)head * a.dk * a.dv + e;
    float o = 0.0f;
    for (int d = wave; d < a.dk; d += 4)
        if (in) {
            const float s = fmaf((float)k[d], v, dec * a.s_in[at + (long long)d * a.dv]);
            a.s_out[at + (long long)d * a.dv] = s;
            o = fmaf((float)q[d], s, o);
        }
    part[wave][lane] = o;
    __syncthreads();
    if (wave == 0 && in) {
        o = (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]);
        ((T*)a.out)[seq * a.ot + (long long)head * a.oh + e] = (T)(a.scale * o);
    }
}

template <int DK, int NW, bool FULL>
hipError_t launch_one(const LinAttnArgs& a, hipStream_t st) {
    const size_t bytes = sizeof(Lds<DK, NW>);
    const void* f = (const void*)k_linattn32<DK, NW, FULL>;
    hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e != hipSuccess) return e;
    LinAttnArgs args = a;
    void* pa[] = {&args};
    const long long blocks = (long long)a.n_segs * a.heads * a.slices;
    return hipLaunchKernel(f, dim3((unsigned)blocks), dim3(64 * NW), pa, bytes, st);
}

template <int DK>
hipError_t launch_dk(const LinAttnArgs& a, bool full, hipStream_t st) {
    if (linattn_waves(a.dv) == 4)
        return full ? launch_one<DK, 4, true>(a, st) : launch_one<DK, 4, false>(a, st);
    return full ? launch_one<DK, 2, true>(a, st) : launch_one<DK, 2, false>(a, st);
}

}  // namespace

hipError_t linattn_launch_f32(const LinAttnArgs& a, bool full, hipStream_t st) {
    if (a.dk <= 32) return launch_dk<32>(a, full, st);
    if (a.dk <= 64) return launch_dk<64>(a, full, st);
    if (a.dk <= 96) return launch_dk<96>(a, full, st);
    if (a.dk <= 128) return launch_dk<128>(a, full, st);
    return launch_dk<256>(a, full, st);
}

hipError_t linattn_launch_chain(const LinAttnArgs& a, hipStream_t st) {
    LinAttnArgs args = a;
    void* pa[] = {&args};
    const long long blocks = (long long)((a.dk * a.dv + 255) / 256) * a.n_seqs * a.heads;
    return hipLaunchKernel((const void*)k_linattn_chain, dim3((unsigned)blocks), dim3(256), pa, 0, st);
}

hipError_t linattn_launch_step(const LinAttnArgs& a, int dtype, hipStream_t st) {
    LinAttnArgs args = a;
    void* pa[] = {&args};
    const void* f = dtype == SSLA_F32   ? (const void*)k_linattn_step<float>
                    : dtype == SSLA_BF16 ? (const void*)k_linattn_step<__bf16>
                                         : (const void*)k_linattn_step<_Float16>;
    const long long blocks = (long long)((a.dv + 63) / 64) * a.n_seqs * a.heads;
    return hipLaunchKernel(f, dim3((unsigned)blocks), dim3(256), pa, 0, st);
}

}  // namespace ssla
