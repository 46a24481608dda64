// linattn_kernel.h -- chunked linear attention on the 16 x 16 x 32 bf16 matrix
// instruction, for bf16, fp16 and fp32 tokens.
//
// Over a chunk of C tokens, b_i = g_1 + ... + g_i and S the state before it:
//   P_ij = (q_i . k_j) exp(b_i - b_j)  for j <= i, else 0
//   o_i  = scale (exp(b_i) q_i^T S + sum_j P_ij v_j)
//   S'   = exp(b_C) S + sum_j k_j (exp(b_C - b_j) v_j)^T
// Everything is computed transposed, so that what one product leaves in the
// D registers (row 4 g + r, column m of lane 16 g + m) is the next one's A or
// B operand as it lies (column or row m, eight values of the contraction a
// lane): the state is S[d][e] with d along the registers, which is the A
// operand of O^T = S^T Q^T, a lane's eight values of a step being rows 4 g + r
// of two tiles.  Which d those rows are is free: with eight neighbouring ones
// (state_row), q and k are read as they lie.  The order of a contraction over
// tokens is free too: P's columns are put into the registers' order on their way
// to LDS (operand_at), and tokens are taken in it from k and v.
//
// Precision: an operand is the sum of bf16 terms, each eight bits of what the
// ones before leave: a bf16 token value is one term, an fp16
// value two, both exactly; an fp32 value, and P and S there, three.  For bf16
// tokens P has three too: with two its rounding (2^-18) was most of what set the
// outputs apart from an fp32 computation's, 9.9e-5 against 3.9e-5 of them over 8192
// tokens of 16 heads of 128 (the third costs 1 to 2%).  P of fp16 tokens has two
// (4.7e-5; a third costs 3.6%, and the error against 64 bits, 2.074e-4, would fall
// by a four thousandth of it), and so has, for both, the copy of S that multiplies
// q, 2^-18 of each value (a third changes the bf16 outputs by 2e-6 and costs 7%).
// exp(b_C - b_j) v_j has three, since these products make up the fp32 state.
// Products of terms whose orders add up to more than the last kept one's are
// left out.  fp32 tokens take 6 bf16 products of 16 cycles where the fp32
// instruction takes 256 cycles for the same block.
//
// Each wave owns 16 columns of v, the state and the output; the C x C products
// P are dealt over the waves and shared through LDS.
//
// 16 sequences of 8192 tokens, 16 heads of 128 in bf16 (2.1 GB, one workgroup a
// compute unit) take 0.64 ms, 3.4 TB/s, a call among others whose inputs come from
// memory (0.61 to 0.69 by card).  The loads and stores alone take 0.46 (a large copy's
// rate: 0.42), the arithmetic alone 0.55, or 0.48 for each such batch where two
// workgroups share a compute unit (then 0.59 in all).  A wave and chunk issues some
// 250 vector instructions (mostly the splits into terms), 48 products, 44 LDS and 87
// scalar ones; the vector units are busy for 47% of the time, the matrix cores for
// 30%, LDS for 31%: what is left is the waits of a chunk's phases for one another.  P one chunk ahead with one barrier fewer (two chunks in LDS)
// changed nothing.
#pragma once

#include <cstddef>

#include "linattn_chunk.h"

namespace ssla {
namespace chunk {

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef unsigned short us2 __attribute__((ext_vector_type(2)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f4 mma(bf8 a, bf8 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Two values rounded to bf16, packed; x keeps what is left of them.
__device__ __forceinline__ unsigned split2(float& x, float& y) {
    const unsigned h = __builtin_bit_cast(unsigned, __builtin_convertvector(f2{x, y}, bf2));
    x -= __builtin_bit_cast(float, h << 16);
    y -= __builtin_bit_cast(float, h & 0xffff0000u);
    return h;
}
__device__ __forceinline__ unsigned round2(float x, float y) {
    return __builtin_bit_cast(unsigned, __builtin_convertvector(f2{x, y}, bf2));
}
// The same, cut off instead of rounded.
__device__ __forceinline__ unsigned cut2(float& x, float& y) {
    const unsigned a = __builtin_bit_cast(unsigned, x), b = __builtin_bit_cast(unsigned, y);
    x -= __builtin_bit_cast(float, a & 0xffff0000u);
    y -= __builtin_bit_cast(float, b & 0xffff0000u);
    return (a >> 16) | (b & 0xffff0000u);
}
// Term n of N.  The first of three is cut off: rounded, the largest fp32 values would
// become infinities, and with two terms behind it the half step does not matter
// (2^-26 is left instead of 2^-27).
template <int N>
__device__ __forceinline__ unsigned term(int n, float& x, float& y) {
    return n + 1 == N ? round2(x, y) : N == 3 && n == 0 ? cut2(x, y) : split2(x, y);
}
// x as N bf16 terms.
template <int N>
__device__ __forceinline__ void split(f8 x, bf8 (&t)[N]) {
    #pragma unroll
    for (int n = 0; n < N; ++n) {
        u4 h;
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            float a = x[2 * i], b = x[2 * i + 1];
            h[i] = term<N>(n, a, b);
            x[2 * i] = a;
            x[2 * i + 1] = b;
        }
        t[n] = __builtin_bit_cast(bf8, h);
    }
}
template <int N>
__device__ __forceinline__ void split(f4 x, u2 (&t)[N]) {
    #pragma unroll
    for (int n = 0; n < N; ++n)
        #pragma unroll
        for (int i = 0; i < 2; ++i) {
            float a = x[2 * i], b = x[2 * i + 1];
            t[n][i] = term<N>(n, a, b);
            x[2 * i] = a;
            x[2 * i + 1] = b;
        }
}

__device__ __forceinline__ f8 join(f4 a, f4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }
__device__ __forceinline__ s8 join(s4 a, s4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

// Four rows of a column-major operand: lane m of each group of 16 gets column
// m of rows 0..3 of the 4 x 16 block whose 8-byte pieces the group's lanes
// address (lane n: row n / 4, columns 4 (n % 4) ..).
__device__ __forceinline__ s4 tr4(const void* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s4*)(__attribute__((address_space(3))) void*)p);
}

// Place of index i of a contraction in an operand's row: a lane's eight values of
// a step, 32 s + 4 g .. and 32 s + 16 + 4 g .., lie together at 32 s + 8 g.
__device__ __forceinline__ int operand_at(int i) { return (i & ~31) | (i & 12) << 1 | (i & 16) >> 2 | (i & 3); }

// Elements behind a row of bf16 in LDS (a multiple of 32): rows then begin an odd
// multiple of 32 bytes apart modulo 64, at which 16 rows' 16-byte pieces are read
// in 5.5 cycles a wave (9.4 at other steps; 8-byte pieces, straight or
// transposed, take 7.5 to 8 at any).
constexpr int kPad = 16;

// Token types: terms of a value; how v lies in LDS, comes from there and is
// searched for infinities and NaN.
template <class T> struct Token;
template <class T> struct Token16 {
    typedef T V8 __attribute__((ext_vector_type(8)));
    template <int W> static constexpr int stride() { return W + kPad; }
    // column m of the wave's 16 columns at `col`, tokens 4 g .. and 16 + 4 g ..
    template <int VS> static __device__ __forceinline__ V8 column(const T* v, int col, int m, int g) {
        const T* p = &v[(4 * g + (m >> 2)) * VS + col + 4 * (m & 3)];
        return __builtin_bit_cast(V8, join(tr4(p), tr4(p + 16 * VS)));
    }
    static __device__ __forceinline__ f8 wide(V8 x) { return __builtin_convertvector(x, f8); }
};
template <> struct Token<__bf16> : Token16<__bf16> {
    static constexpr int TERMS = 1;
    static constexpr unsigned EXP = 0x7f807f80u;           // exponent bits of two values
    static __device__ __forceinline__ void terms(V8 x, bf8 (&t)[1]) { t[0] = x; }
};
template <> struct Token<_Float16> : Token16<_Float16> {
    static constexpr int TERMS = 2;
    static constexpr unsigned EXP = 0x7c007c00u;
    static __device__ __forceinline__ void terms(V8 x, bf8 (&t)[2]) { split(wide(x), t); }
};
template <> struct Token<float> {
    typedef f8 V8;
    static constexpr int TERMS = 3;
    template <int W> static constexpr int stride() { return W + 4; }     // four rows 16 banks apart
    template <int VS> static __device__ __forceinline__ f8 column(const float* v, int col, int m, int g) {
        f8 x;
        #pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = v[((i >> 2) * 16 + 4 * g + (i & 3)) * VS + col + m];
        return x;
    }
    static __device__ __forceinline__ f8 wide(f8 x) { return x; }
    static __device__ __forceinline__ void terms(f8 x, bf8 (&t)[3]) { split(x, t); }
};

// Whether any of a lane's values is an infinity or NaN.
template <class T, class V8>
__device__ __forceinline__ bool odd_values(V8 v) {
    if constexpr (sizeof(T) == 2) {
        const u4 w = __builtin_bit_cast(u4, v);
        us2 most = {0, 0};                     // largest exponents of two interleaved sets
        #pragma unroll
        for (int i = 0; i < 4; ++i)
            most = __builtin_elementwise_max(most, __builtin_bit_cast(us2, w[i] & Token<T>::EXP));
        const unsigned short ex = (unsigned short)Token<T>::EXP;
        return most[0] == ex || most[1] == ex;
    } else {
        unsigned most = 0;
        #pragma unroll
        for (int i = 0; i < 8; ++i) most = max(most, __builtin_bit_cast(unsigned, (float)v[i]) & 0x7f800000u);
        return most == 0x7f800000u;
    }
}
__device__ __forceinline__ bool not_finite(float x) {
    return (__builtin_bit_cast(unsigned, x) & 0x7f800000u) == 0x7f800000u;
}

// A piece's four values at `x`, `part` of it, as terms.
template <class T>
__device__ __forceinline__ void piece_terms(u4 x, int part, u2 (&t)[Token<T>::TERMS]) {
    if constexpr (sizeof(T) == 4) {
        split(__builtin_bit_cast(f4, x), t);
    } else if constexpr (Token<T>::TERMS == 2) {
        const u2 y = {x[2 * part], x[2 * part + 1]};
        split(__builtin_convertvector(__builtin_bit_cast(h4, y), f4), t);
    } else {
        t[0] = u2{x[2 * part], x[2 * part + 1]};
    }
}

// Tokens of a chunk, one step of the contractions over tokens.  Chunks of 64 halve
// the conversions of the state and the barriers, but take twice the registers and
// LDS: with half the waves on a compute unit they were slower (fp32, 16 x 2000
// tokens of 4 heads of 96: 72 against 61 us; bf16, 8192 tokens of 16 heads of 128:
// 53 against 45) but where there is one workgroup a compute unit anyway (16 x 8192:
// 3% faster).
constexpr int C = 32;

template <class T, int DK, int NW>
struct Lds {
    static constexpr int TERMS = Token<T>::TERMS;
    static constexpr int PT = TERMS == 2 ? 2 : 3, ST = TERMS == 3 ? 3 : 2;       // terms of P; of S's copy
    static constexpr int DV = 16 * NW;
    static constexpr int QS = DK + kPad, PS = C + kPad, VS = Token<T>::template stride<DV>();
    __bf16 q[TERMS][C * QS];
    __bf16 k[TERMS][C * QS];
    T v[C * VS];
    __bf16 p[PT][C * PS];        // rows i, columns j in operand order
    Decays<C> b[2];              // of this chunk and the next
};
// Decays are read four at a time in either of the two.
static_assert(sizeof(Decays<C>) % 16 == 0 && alignof(Decays<C>) % 16 == 0 && offsetof(Decays<C>, hi) % 16 == 0 &&
              offsetof(Decays<C>, lo) % 16 == 0 && offsetof(Decays<C>, w) % 16 == 0);

template <class T, int DK, int NW, bool FULL, bool VEC>
__global__ __launch_bounds__(64 * NW, waves_per_simd(DK, Token<T>::TERMS)) void k_linattn(const LinAttnArgs a) {
    typedef Token<T> Tk;
    typedef typename Tk::V8 V8;
    typedef Lds<T, DK, NW> L;
    constexpr int NT = 64 * NW, TERMS = L::TERMS, PT = L::PT, ST = L::ST;
    constexpr int DT = DK / 16, KS = DK / 32;              // tiles, steps along d
    constexpr int IT = C / 16;                             // tiles along tokens
    constexpr int P_ORDER = PT - 1, S_ORDER = ST - 1;      // highest orders of terms' products kept
    extern __shared__ __align__(16) char smem[];
    L& lds = *reinterpret_cast<L*>(smem);

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int m = lane & 15, g = lane >> 4;
    Place<T, NW> pl;
    if (!pl.find(a, FULL, wave, lane)) return;
    const Segment& sg = pl.sg;
    const int dvs = a.dv - pl.slice * L::DV;               // columns of v from the slice's first

    f4 S[DT];
    read_state(S, pl, a, FULL, m, g);

    Rows<T, DK, C, NT, VEC> rq, rk;
    Rows<T, L::DV, C, NT, VEC> rv;
    float rg = 0.0f;
    rk.init(a.kt, a.dk, tid);
    rv.init(a.vt, dvs, tid);
    if (FULL) rq.init(a.qt, a.dk, tid);
    auto load = [&](int t) {
        const int n = min(C, sg.t1 - t);
        const long long row = sg.row + t;
        rk.load(pl.k + row * a.kt, a.kt, a.dk, n, tid);
        rv.load(pl.v + row * a.vt, a.vt, dvs, n, tid);
        if (FULL) rq.load(pl.q + row * a.qt, a.qt, a.dk, n, tid);
        if (wave == NW - 1) rg = lane < n ? pl.g[(row + lane) * a.gt] : 0.0f;
    };

    if (FULL) {     // the tiles of P above the diagonal are never written again
        for (int i = tid; i < PT * C * L::PS; i += NT) (&lds.p[0][0])[i] = (__bf16)0.0f;
    }
    float decay = 1.0f;                        // of the whole segment (exp of the sum of g)
    if (sg.t0 < sg.t1) {
        load(sg.t0);
        if (wave == NW - 1) lds.b[0].set(rg, a.scale, lane);
    }
    int buf = 0;
    for (int t = sg.t0; t < sg.t1; t += C, buf ^= 1) {
        const int n = min(C, sg.t1 - t);
        __syncthreads();                       // the last chunk's readers are done
        rk.settle(a.dk, tid);
        rv.settle(dvs, tid);
        if (FULL) rq.settle(a.dk, tid);
        #pragma unroll
        for (int p = 0; p < rk.N; ++p) {
            const int row = rk.row(p, tid);
            if (!rk.STEPS && row >= C) continue;
            #pragma unroll
            for (int part = 0; part < rk.E / 4; ++part) {
                const int c = rk.col(p, tid) + 4 * part;
                u2 x[TERMS];
                piece_terms<T>(rk.x[p], part, x);
                #pragma unroll
                for (int i = 0; i < TERMS; ++i) *(u2*)&lds.k[i][row * L::QS + c] = x[i];
                if (FULL) {
                    piece_terms<T>(rq.x[p], part, x);
                    #pragma unroll
                    for (int i = 0; i < TERMS; ++i) *(u2*)&lds.q[i][row * L::QS + c] = x[i];
                }
            }
        }
        #pragma unroll
        for (int p = 0; p < rv.N; ++p) *(u4*)&lds.v[rv.row(p, tid) * L::VS + rv.col(p, tid)] = rv.x[p];
        __syncthreads();
        if (t + C < sg.t1) load(t + C);

        f4 O[IT];
        if (FULL) {
            // ---- P^T = K Q^T: the three tiles on and below the diagonal -------
            if (wave < 3) {
                const int it = wave >= 1 ? 1 : 0, jt = wave - it;
                f4 acc[2] = {};                // two chains: a product waits for the one before it
                constexpr int KH = TERMS > 1 ? 1 : KS > 4 ? 4 : KS;              // steps in flight
                #pragma unroll
                for (int s0 = 0; s0 < KS; s0 += KH) {
                    bf8 ka[KH][TERMS], qa[KH][TERMS];
                    #pragma unroll
                    for (int s = 0; s < KH; ++s)
                        #pragma unroll
                        for (int i = 0; i < TERMS; ++i) {
                            ka[s][i] = *(const bf8*)&lds.k[i][(16 * jt + m) * L::QS + 32 * (s0 + s) + 8 * g];
                            qa[s][i] = *(const bf8*)&lds.q[i][(16 * it + m) * L::QS + 32 * (s0 + s) + 8 * g];
                        }
                    loads_stay_above();
                    #pragma unroll
                    for (int s = 0; s < KH; ++s)
                        #pragma unroll
                        for (int i = 0; i < TERMS; ++i)
                            #pragma unroll
                            for (int j = 0; j < TERMS; ++j)
                                if (i + j <= P_ORDER) {
                                    f4& c = acc[TERMS == 1 ? s & 1 : j & 1];
                                    c = mma(ka[s][i], qa[s][j], c);
                                }
                }
                acc[0] += acc[1];
                const int i = 16 * it + m, j = 16 * jt + 4 * g;
                const f4 jh = *(const f4*)&lds.b[buf].hi[j], jl = *(const f4*)&lds.b[buf].lo[j];
                const float ih = lds.b[buf].hi[i], il = lds.b[buf].lo[i];
                f4 p;
                #pragma unroll
                for (int r = 0; r < 4; ++r) p[r] = acc[0][r] * (a.scale * exp2_((ih - jh[r]) + (il - jl[r])));
                if (it == jt)
                    #pragma unroll
                    for (int r = 0; r < 4; ++r) p[r] = j + r <= i ? p[r] : 0.0f;
                u2 x[PT];
                split(p, x);
                #pragma unroll
                for (int h = 0; h < PT; ++h) *(u2*)&lds.p[h][i * L::PS + operand_at(j)] = x[h];
            }
            // ---- O^T = S^T Q^T ------------------------------------------------
            #pragma unroll
            for (int it = 0; it < IT; ++it) O[it] = f4{0.0f, 0.0f, 0.0f, 0.0f};
            #pragma unroll
            for (int s = 0; s < KS; ++s) {
                bf8 qa[IT][TERMS];
                #pragma unroll
                for (int it = 0; it < IT; ++it)
                    #pragma unroll
                    for (int i = 0; i < TERMS; ++i)
                        qa[it][i] = *(const bf8*)&lds.q[i][(16 * it + m) * L::QS + 32 * s + 8 * g];
                loads_stay_above();
                bf8 sa[ST];
                split(join(S[2 * s], S[2 * s + 1]), sa);
                #pragma unroll
                for (int h = 0; h < ST; ++h)
                    #pragma unroll
                    for (int i = 0; i < TERMS; ++i)
                        if (h + i <= S_ORDER)
                            #pragma unroll
                            for (int it = 0; it < IT; ++it) O[it] = mma(sa[h], qa[it][i], O[it]);
            }
            #pragma unroll
            for (int it = 0; it < IT; ++it) O[it] *= lds.b[buf].eb[16 * it + m];
        }
        // v^T of the wave's columns
        V8 vf = Tk::template column<L::VS>(lds.v, 16 * wave, m, g);
        if (FULL) __syncthreads();             // P is whole
        // An infinity or NaN of v must not reach the rows before it through their
        // zeros of P: it is taken out here, and its column set to NaN from its
        // token on.
        const bool any_bad = __any(odd_values<T>(vf));
        int bad = C;                           // the column's first such token
        if (any_bad) {
            rare();
            #pragma unroll
            for (int i = 7; i >= 0; --i)
                if (not_finite((float)vf[i])) {
                    bad = (i >> 2) * 16 + 4 * g + (i & 3);
                    vf[i] = 0;
                }
            bad = min(bad, __shfl_xor(bad, 16));
            bad = min(bad, __shfl_xor(bad, 32));
        }

        if (FULL) {
            // ---- O^T += V^T P^T -------------------------------------------------
            bf8 vt[TERMS], pa[IT][PT];
            #pragma unroll
            for (int it = 0; it < IT; ++it)
                #pragma unroll
                for (int h = 0; h < PT; ++h) pa[it][h] = *(const bf8*)&lds.p[h][(16 * it + m) * L::PS + 8 * g];
            Tk::terms(vf, vt);
            #pragma unroll
            for (int h = 0; h < PT; ++h)
                #pragma unroll
                for (int i = 0; i < TERMS; ++i)
                    if (h + i <= P_ORDER)
                        #pragma unroll
                        for (int it = 0; it < IT; ++it) O[it] = mma(vt[i], pa[it][h], O[it]);
            if (any_bad) {
                rare();
                #pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int first = __shfl(bad, 4 * g + r);
                    #pragma unroll
                    for (int it = 0; it < IT; ++it)
                        if (16 * it + m >= first) O[it][r] = __builtin_nanf("");
                }
            }
            T* const ob = (T*)a.out + (sg.row + t) * a.ot + (long long)pl.head * a.oh;
            const auto bo = buffer(ob, VEC ? ((n - 1) * a.ot + a.dv) * (int)sizeof(T) : 0);
            const int e = pl.e0 + 4 * g;
            #pragma unroll
            for (int it = 0; it < IT; ++it) {
                const int i = 16 * it + m;
                alignas(16) T y[4];
                #pragma unroll
                for (int r = 0; r < 4; ++r) y[r] = (T)O[it][r];
                if (VEC) {
                    const unsigned at = e < a.dv ? (unsigned)(i * (int)a.ot + e) * (unsigned)sizeof(T) : kOut;
                    if constexpr (sizeof(T) == 4) __builtin_amdgcn_raw_buffer_store_b128(*(const u4*)y, bo, at, 0, 0);
                    else __builtin_amdgcn_raw_buffer_store_b64(*(const u2*)y, bo, at, 0, 0);
                } else if (i < n && e + 4 <= a.dv) {
                    __builtin_memcpy(ob + i * a.ot + e, y, sizeof(y));           // at any alignment
                } else if (i < n) {
                    #pragma unroll
                    for (int r = 0; r < 3; ++r)
                        if (e + r < a.dv) ob[i * a.ot + e + r] = y[r];
                }
            }
        }

        // ---- S = exp(b_C) S + K^T (w v): for the next chunk, or as an answer ----
        const float eC = lds.b[buf].end;
        decay *= eC;
        if (!FULL || !pl.last || t + C < sg.t1 || a.s_out) {
            const float* w = &lds.b[buf].w[4 * g];
            bf8 x[3];
            split(Tk::wide(vf) * join(*(const f4*)w, *(const f4*)(w + 16)), x);
            #pragma unroll
            for (int dt = 0; dt < DT; dt += 2) {           // two chains: a product waits for the one before it
                bf8 ka[2][TERMS];              // k^T of two tiles of d
                #pragma unroll
                for (int y = 0; y < 2; ++y) {
                    #pragma unroll
                    for (int i = 0; i < TERMS; ++i) {
                        const __bf16* p = &lds.k[i][(4 * g + (m >> 2)) * L::QS + 16 * dt + 4 * y + 8 * (m & 3)];
                        ka[y][i] = __builtin_bit_cast(bf8, join(tr4(p), tr4(p + 16 * L::QS)));
                    }
                    S[dt + y] *= eC;
                }
                loads_stay_above();
                #pragma unroll
                for (int h = 0; h < 3; ++h)
                    #pragma unroll
                    for (int i = 0; i < TERMS; ++i)
                        if (h + i <= 2)
                            #pragma unroll
                            for (int y = 0; y < 2; ++y) S[dt + y] = mma(ka[y][i], x[h], S[dt + y]);
            }
            if (any_bad) {
                rare();
                if (bad < C) {
                    #pragma unroll
                    for (int dt = 0; dt < DT; ++dt)
                        #pragma unroll
                        for (int r = 0; r < 4; ++r) S[dt][r] = __builtin_nanf("");
                }
            }
        }
        if (t + C < sg.t1 && wave == NW - 1) lds.b[buf ^ 1].set(rg, a.scale, lane);
    }

    if (!FULL && pl.slice == 0 && tid == 0) a.ws_decay[(long long)sg.state * a.heads + pl.head] = decay;
    write_state(S, pl, a, FULL, m, g);
}

template <class T, int DK, int NW>
hipError_t launch_one(const LinAttnArgs& a, bool full, hipStream_t st) {
    const void* f = full ? (a.vec ? (const void*)k_linattn<T, DK, NW, true, true>
                                  : (const void*)k_linattn<T, DK, NW, true, false>)
                         : (a.vec ? (const void*)k_linattn<T, DK, NW, false, true>
                                  : (const void*)k_linattn<T, DK, NW, false, false>);
    return linattn_launch(f, a, NW, sizeof(Lds<T, DK, NW>), st);
}

template <class T, int DK>
hipError_t launch_dk(const LinAttnArgs& a, bool full, hipStream_t st) {
    if constexpr (DK > 128) {
        return launch_one<T, DK, 4>(a, full, st);
    } else {
        switch (linattn_waves(a.dk, a.dv)) {
            case 4: return launch_one<T, DK, 4>(a, full, st);
            case 6: return launch_one<T, DK, 6>(a, full, st);
            default: return launch_one<T, DK, 8>(a, full, st);
        }
    }
}

template <class T>
hipError_t launch(const LinAttnArgs& a, bool full, hipStream_t st) {
    if (a.dk <= 32) return launch_dk<T, 32>(a, full, st);
    if (a.dk <= 64) return launch_dk<T, 64>(a, full, st);
    if (a.dk <= 96) return launch_dk<T, 96>(a, full, st);
    if (a.dk <= 128) return launch_dk<T, 128>(a, full, st);
    return launch_dk<T, 256>(a, full, st);
}

}  // namespace chunk
}  // namespace ssla
