// linattn16.h -- chunked linear attention for bf16 and fp16 tokens on the
// 16 x 16 x 32 matrix instructions.
//
// Over a chunk of 64 tokens, b_i = g_1 + ... + g_i and S the state before it:
//   P_ij = (q_i . k_j) exp(b_i - b_j)  for j <= i, else 0
//   o_i  = scale (exp(b_i) q_i^T S + sum_j P_ij v_j)
//   S'   = exp(b_64) S + sum_j k_j (exp(b_64 - b_j) v_j)^T
// Everything is computed transposed, so that what one product leaves in the
// D registers (row 4 g + r, column m of lane 16 g + m) is the next one's A or
// B operand as it lies (column or row m, eight values of the contraction a
// lane): the state is S[d][e] with d along the registers, which is the A
// operand of O^T = S^T Q^T once its d order (4 g + r of two 16-row tiles) is
// used for Q as well.
//
// Precision: operands of a product with fp32 origin are split into bf16 terms
// whose sum is the value: P and the copy of S that multiplies Q in two terms
// (2^-17, well below the output's 2^-9), exp(b_64 - b_j) v_j in three (2^-25),
// because these products make up the fp32 state.  fp16 inputs are the sum of
// two bf16 terms exactly; q.k runs on the fp16 instruction as it is.
// The exponents' sums are held as two floats (hi + lo of a 64-bit sum), since
// b_i - b_j is small where b is large.
//
// Each wave owns 32 columns of v, the state and the output; the 64 x 64
// products P are dealt over the waves and shared through LDS.
#pragma once

#include "linattn.h"

namespace ssla {
namespace la16 {

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f8 __attribute__((ext_vector_type(8)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));

constexpr int C = 64;            // tokens of a chunk
constexpr int PAD = 16;          // elements behind a row in LDS: rows 8 banks apart

__device__ __forceinline__ f4 mma(bf8 a, bf8 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f4 mma(h8 a, h8 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ bf8 round8(f8 x) { return __builtin_convertvector(x, bf8); }
__device__ __forceinline__ f8 wide8(bf8 x) { return __builtin_convertvector(x, f8); }
__device__ __forceinline__ bf4 round4(f4 x) { return __builtin_convertvector(x, bf4); }
__device__ __forceinline__ f4 wide4(bf4 x) { return __builtin_convertvector(x, f4); }

__device__ __forceinline__ f8 join(f4 a, f4 b) {
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

template <class T> struct Half;      // 16-bit type of the tokens
template <> struct Half<__bf16> {
    typedef bf8 V;
    static constexpr int TERMS = 1;
    static constexpr unsigned EXP = 0x7f807f80u, ONE = 0x00800080u;   // exponent bits, their lowest
};
template <> struct Half<_Float16> {
    typedef h8 V;
    static constexpr int TERMS = 2;
    static constexpr unsigned EXP = 0x7c007c00u, ONE = 0x04000400u;
};

// x as TERMS bf16 terms
__device__ __forceinline__ void terms(bf8 x, bf8* t) { t[0] = x; }
__device__ __forceinline__ void terms(h8 x, bf8* t) {
    const f8 f = __builtin_convertvector(x, f8);
    t[0] = round8(f);
    t[1] = round8(f - wide8(t[0]));
}

// Four rows of a column-major operand: lane m of each group of 16 gets column
// m of rows 0..3 of the 4 x 16 block whose 8-byte pieces the group's lanes
// address (lane n: row n / 4, columns 4 (n % 4) ..).
__device__ __forceinline__ s4 tr4(const void* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s4*)(__attribute__((address_space(3))) void*)p);
}

template <class T, int DK, int NW>
struct Lds {
    static constexpr int DV = 32 * NW;
    static constexpr int QS = DK + PAD, VS = DV + PAD, PS = C + PAD;
    T q[C * QS];
    T k[C * QS];
    T v[C * VS];
    __bf16 p[2][C * PS];
    float bhi[C], blo[C], eb[C], w[C];
    int bad[DV];                 // first token whose v is not finite, per column
    int any_bad;
};

template <class T, int DK, int NW, bool FULL>
__global__ __launch_bounds__(64 * NW, 1) void k_linattn16(const LinAttnArgs a) {
    typedef typename Half<T>::V V8;
    typedef Lds<T, DK, NW> L;
    constexpr int NT = 64 * NW, TERMS = Half<T>::TERMS;
    constexpr int DT = DK / 16, KS = DK / 32;              // tiles, steps along d
    constexpr int QC = DK / 8, QP = C * QC / NT;           // 16-byte pieces: a row, a thread
    constexpr int VC = L::DV / 8, VP = C * VC / NT;
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

    const T* qb = (const T*)a.q + (long long)(head / a.rep) * a.qh;
    const T* kb = (const T*)a.k + (long long)(head / a.rep) * a.kh;
    const T* vb = (const T*)a.v + (long long)head * a.vh + slice * L::DV;
    const float* gb = a.g + (long long)head * a.gh;
    const int dvs = a.dv - slice * L::DV;      // columns of v from the slice's first

    // ---- state ---------------------------------------------------------
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

    // ---- a chunk's rows, from memory into registers ---------------------------
    u4 rq[FULL ? QP : 1], rk[QP], rv[VP];
    float rg = 0.0f;
    auto piece = [&](const T* base, long long stride, int idx, int cols, int per_row, int n) -> u4 {
        const int row = idx / per_row, c = (idx - row * per_row) * 8;
        u4 x = {0u, 0u, 0u, 0u};
        if (row < n && c < cols) {
            const T* p = base + row * stride + c;
            if (a.vec_in) {
                x = *(const u4*)p;
            } else {
                unsigned short* xs = (unsigned short*)&x;
                #pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (c + i < cols) xs[i] = ((const unsigned short*)p)[i];
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
        rg = lane < n ? gb[(row + lane) * a.gt] : 0.0f;
    };

    if (FULL) {     // the tiles of P above the diagonal are never written again
        for (int i = tid; i < C * L::PS; i += NT) lds.p[0][i] = lds.p[1][i] = (__bf16)0.0f;
    }
    float decay = 1.0f;                        // of the whole segment (exp of the sum of g)
    if (sg.t0 < sg.t1) load(sg.t0);
    for (int t = sg.t0; t < sg.t1; t += C) {
        const int n = min(C, sg.t1 - t);
        __syncthreads();                       // the last chunk's readers are done
        if (tid == 0) lds.any_bad = 0;
        if (tid < L::DV) lds.bad[tid] = C;
        if (wave == 0) {
            double b = rg < kMinLogDecay ? kMinLogDecay : rg;
            #pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const double u = __shfl_up(b, o);
                if (lane >= o) b += u;
            }
            const double end = __shfl(b, 63);
            const float hi = (float)b;
            lds.bhi[lane] = hi;
            lds.blo[lane] = (float)(b - (double)hi);
            lds.eb[lane] = __expf(hi);
            lds.w[lane] = __expf((float)(end - b));
        }
        __syncthreads();
        #pragma unroll
        for (int p = 0; p < QP; ++p) {
            const int idx = tid + p * NT, row = idx / QC, c = (idx - row * QC) * 8;
            *(u4*)&lds.k[row * L::QS + c] = rk[p];
            if (FULL) *(u4*)&lds.q[row * L::QS + c] = rq[p];
        }
        #pragma unroll
        for (int p = 0; p < VP; ++p) {
            const int idx = tid + p * NT, row = idx / VC, c = (idx - row * VC) * 8;
            u4 x = rv[p];
            // An infinity or NaN of v must not reach the rows before it through
            // their zeros of P: it is taken out here, and its column set to NaN
            // from its token on.
            unsigned bits = 0;
            #pragma unroll
            for (int i = 0; i < 4; ++i) bits |= ((x[i] & Half<T>::EXP) + Half<T>::ONE) & 0x80008000u;
            if (bits) {
                lds.any_bad = 1;
                #pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const unsigned h = (x[i >> 1] >> (16 * (i & 1))) & 0xffffu;
                    if ((h & (Half<T>::EXP & 0xffffu)) == (Half<T>::EXP & 0xffffu)) {
                        atomicMin(&lds.bad[c + i], row);
                        x[i >> 1] &= ~(0xffffu << (16 * (i & 1)));
                    }
                }
            }
            *(u4*)&lds.v[row * L::VS + c] = x;
        }
        __syncthreads();
        if (t + C < sg.t1) load(t + C);

        // v^T of the wave's columns: column m, tokens 32 s + 8 g ..
        V8 vf[2][2];
        #pragma unroll
        for (int et = 0; et < 2; ++et)
            #pragma unroll
            for (int s = 0; s < 2; ++s) {
                const T* p = &lds.v[(32 * s + 8 * g + (m >> 2)) * L::VS + wave * 32 + 16 * et + 4 * (m & 3)];
                const s4 x = tr4(p), y = tr4(p + 4 * L::VS);
                vf[et][s] = __builtin_bit_cast(V8, (s8)__builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
            }

        f4 O[2][4];
        if (FULL) {
            // ---- P^T = K Q^T: ten tiles on and below the diagonal ----------
            for (int u = wave; u < 10; u += NW) {
                const int it = u >= 6 ? 3 : u >= 3 ? 2 : u >= 1 ? 1 : 0;
                const int jt = u - it * (it + 1) / 2;
                f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
                #pragma unroll
                for (int s = 0; s < KS; ++s) {
                    const V8 ka = *(const V8*)&lds.k[(16 * jt + m) * L::QS + 32 * s + 8 * g];
                    const V8 qa = *(const V8*)&lds.q[(16 * it + m) * L::QS + 32 * s + 8 * g];
                    acc = mma(ka, qa, acc);
                }
                const int i = 16 * it + m, j = 16 * jt + 4 * g;
                const f4 jh = *(const f4*)&lds.bhi[j], jl = *(const f4*)&lds.blo[j];
                const float ih = lds.bhi[i], il = lds.blo[i];
                f4 p;
                #pragma unroll
                for (int r = 0; r < 4; ++r)
                    p[r] = j + r <= i ? acc[r] * __expf((ih - jh[r]) + (il - jl[r])) : 0.0f;
                const bf4 hi = round4(p);
                *(bf4*)&lds.p[0][i * L::PS + j] = hi;
                *(bf4*)&lds.p[1][i * L::PS + j] = round4(p - wide4(hi));
            }
            // ---- O^T = S^T Q^T ------------------------------------------------
            #pragma unroll
            for (int et = 0; et < 2; ++et)
                #pragma unroll
                for (int it = 0; it < 4; ++it) O[et][it] = f4{0.0f, 0.0f, 0.0f, 0.0f};
            #pragma unroll
            for (int s = 0; s < KS; ++s) {
                bf8 sh[2], sl[2];
                #pragma unroll
                for (int et = 0; et < 2; ++et) {
                    const f8 x = join(S[2 * s][et], S[2 * s + 1][et]);
                    sh[et] = round8(x);
                    sl[et] = round8(x - wide8(sh[et]));
                }
                #pragma unroll
                for (int it = 0; it < 4; ++it) {
                    const T* p = &lds.q[(16 * it + m) * L::QS + 32 * s + 4 * g];
                    const s4 x = *(const s4*)p, y = *(const s4*)(p + 16);
                    bf8 qf[TERMS];
                    terms(__builtin_bit_cast(V8, (s8)__builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7)), qf);
                    #pragma unroll
                    for (int et = 0; et < 2; ++et) {
                        O[et][it] = mma(sh[et], qf[0], O[et][it]);
                        O[et][it] = mma(sl[et], qf[0], O[et][it]);
                        if (TERMS == 2) O[et][it] = mma(sh[et], qf[TERMS - 1], O[et][it]);
                    }
                }
            }
            #pragma unroll
            for (int it = 0; it < 4; ++it) {
                const float eb = lds.eb[16 * it + m];
                #pragma unroll
                for (int et = 0; et < 2; ++et) O[et][it] *= eb;
            }
            __syncthreads();                   // P is whole
            // ---- O^T += V^T P^T -------------------------------------------------
            #pragma unroll
            for (int s = 0; s < 2; ++s) {
                bf8 vt[2][TERMS];
                terms(vf[0][s], vt[0]);
                terms(vf[1][s], vt[1]);
                #pragma unroll
                for (int it = 2 * s; it < 4; ++it) {
                    const bf8 ph = *(const bf8*)&lds.p[0][(16 * it + m) * L::PS + 32 * s + 8 * g];
                    const bf8 pl = *(const bf8*)&lds.p[1][(16 * it + m) * L::PS + 32 * s + 8 * g];
                    #pragma unroll
                    for (int et = 0; et < 2; ++et) {
                        O[et][it] = mma(vt[et][0], ph, O[et][it]);
                        O[et][it] = mma(vt[et][0], pl, O[et][it]);
                        if (TERMS == 2) O[et][it] = mma(vt[et][TERMS - 1], ph, O[et][it]);
                    }
                }
            }
            if (lds.any_bad) {
                #pragma unroll
                for (int et = 0; et < 2; ++et)
                    #pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int first = lds.bad[wave * 32 + 16 * et + 4 * g + r];
                        #pragma unroll
                        for (int it = 0; it < 4; ++it)
                            if (16 * it + m >= first) O[et][it][r] = __builtin_nanf("");
                    }
            }
            #pragma unroll
            for (int it = 0; it < 4; ++it) {
                const int i = 16 * it + m;
                if (i < n) {
                    T* p = (T*)a.out + (sg.row + t + i) * a.ot + (long long)head * a.oh;
                    #pragma unroll
                    for (int et = 0; et < 2; ++et) {
                        const int e = e0 + 16 * et + 4 * g;
                        T y[4];
                        #pragma unroll
                        for (int r = 0; r < 4; ++r) y[r] = (T)(a.scale * O[et][it][r]);
                        if (a.vec_out) {
                            if (e < a.dv) *(u2*)(p + e) = *(const u2*)y;
                        } else {
                            #pragma unroll
                            for (int r = 0; r < 4; ++r)
                                if (e + r < a.dv) p[e + r] = y[r];
                        }
                    }
                }
            }
        }

        // ---- S = exp(b_64) S + K^T (w v): for the next chunk, or as an answer ----
        const float eC = lds.eb[C - 1];
        decay *= eC;
        if (!FULL || !last || t + C < sg.t1 || a.s_out) {
            #pragma unroll
            for (int dt = 0; dt < DT; ++dt)
                #pragma unroll
                for (int et = 0; et < 2; ++et) S[dt][et] *= eC;
            #pragma unroll
            for (int s = 0; s < 2; ++s) {
                const f8 w = join(*(const f4*)&lds.w[32 * s + 8 * g], *(const f4*)&lds.w[32 * s + 8 * g + 4]);
                bf8 x0[2], x1[2], x2[2];
                #pragma unroll
                for (int et = 0; et < 2; ++et) {
                    f8 x = __builtin_convertvector(vf[et][s], f8) * w;
                    x0[et] = round8(x);
                    x -= wide8(x0[et]);
                    x1[et] = round8(x);
                    x -= wide8(x1[et]);
                    x2[et] = round8(x);
                }
                #pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    const T* p = &lds.k[(32 * s + 8 * g + (m >> 2)) * L::QS + 16 * dt + 4 * (m & 3)];
                    const s4 x = tr4(p), y = tr4(p + 4 * L::QS);
                    bf8 kf[TERMS];
                    terms(__builtin_bit_cast(V8, (s8)__builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7)), kf);
                    #pragma unroll
                    for (int et = 0; et < 2; ++et) {
                        S[dt][et] = mma(kf[0], x0[et], S[dt][et]);
                        S[dt][et] = mma(kf[0], x1[et], S[dt][et]);
                        S[dt][et] = mma(kf[0], x2[et], S[dt][et]);
                        if (TERMS == 2) {
                            S[dt][et] = mma(kf[TERMS - 1], x0[et], S[dt][et]);
                            S[dt][et] = mma(kf[TERMS - 1], x1[et], S[dt][et]);
                        }
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

template <class T, int DK, int NW, bool FULL>
hipError_t launch_one(const LinAttnArgs& a, hipStream_t st) {
    const size_t bytes = sizeof(Lds<T, DK, NW>);
    const void* f = (const void*)k_linattn16<T, DK, NW, FULL>;
    // more than 64 KB of LDS has to be asked for once; the attribute is the
    // function's, not the call's, and setting it again costs a lookup
    hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e != hipSuccess) return e;
    LinAttnArgs args = a;
    void* pa[] = {&args};
    const long long blocks = (long long)a.n_segs * a.heads * a.slices;
    return hipLaunchKernel(f, dim3((unsigned)blocks), dim3(64 * NW), pa, bytes, st);
}

template <class T, int DK>
hipError_t launch_dk(const LinAttnArgs& a, bool full, hipStream_t st) {
    if (linattn_waves(a.dv) == 4)
        return full ? launch_one<T, DK, 4, true>(a, st) : launch_one<T, DK, 4, false>(a, st);
    return full ? launch_one<T, DK, 2, true>(a, st) : launch_one<T, DK, 2, false>(a, st);
}

template <class T>
hipError_t launch(const LinAttnArgs& a, bool full, hipStream_t st) {
    if (a.dk <= 32) return launch_dk<T, 32>(a, full, st);
    if (a.dk <= 64) return launch_dk<T, 64>(a, full, st);
    if (a.dk <= 96) return launch_dk<T, 96>(a, full, st);
    if (a.dk <= 128) return launch_dk<T, 128>(a, full, st);
    return launch_dk<T, 256>(a, full, st);
}

}  // namespace la16
}  // namespace ssla
