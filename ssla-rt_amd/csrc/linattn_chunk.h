// linattn_chunk.h -- what the chunked linear-attention kernels share: which
// segment, head and columns a workgroup has, a chunk's rows on their way from
// memory, its decays, and the state at both ends.
#pragma once

#include "linattn.h"

namespace ssla {
namespace chunk {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));

constexpr unsigned kOut = 0x7ffffff0u;     // an offset past every buffer's end

// Raw buffer of `bytes` bytes: loads past its end give zeros, stores there nothing.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* p, long long bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)bytes, 0x00020000);
}

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// x + x of the lane that the DPP pattern names (0 where it names none).
template <int CTRL, int ROWS>
__device__ __forceinline__ double plus_dpp(double x) {
    const u2 v = __builtin_bit_cast(u2, x);
    u2 w;
    w[0] = __builtin_amdgcn_update_dpp(0u, v[0], CTRL, ROWS, 0xf, false);
    w[1] = __builtin_amdgcn_update_dpp(0u, v[1], CTRL, ROWS, 0xf, false);
    return x + __builtin_bit_cast(double, w);
}
// Inclusive sum over the wave's lanes.
__device__ __forceinline__ double running_sum(double x) {
    x = plus_dpp<0x111, 0xf>(x);       // row_shr 1, 2, 4, 8: within 16 lanes
    x = plus_dpp<0x112, 0xf>(x);
    x = plus_dpp<0x114, 0xf>(x);
    x = plus_dpp<0x118, 0xf>(x);
    x = plus_dpp<0x142, 0xa>(x);       // lane 15 of rows 0 and 2 to rows 1 and 3
    x = plus_dpp<0x143, 0xc>(x);       // lane 31 to rows 2 and 3
    return x;
}

// Waves of a SIMD that the chunked kernels' registers leave room for: four (two
// workgroups of eight or six waves a compute unit) as far as that spills little
// (fp32, heads of 96: three waves' registers spill nothing, but then two workgroups
// of six waves seldom fit, 72 against 60 us; bf16, heads of 256: 368 us with one,
// 262 with two, but fp16 129 with one, 138 with two).
constexpr int waves_per_simd(int dk, int terms) {
    return dk > 128 ? terms == 1 ? 2 : 1 : terms == 3 && dk > 96 ? 2 : 4;
}

// Keeps a branch a branch: its body is not computed and selected every time.
__device__ __forceinline__ void rare() { asm volatile(""); }

// LDS reads written before this are issued before it; arithmetic may pass.  The
// scheduler otherwise sinks each read to its product and waits for it there.
__device__ __forceinline__ void loads_stay_above() { __builtin_amdgcn_sched_barrier(0x40f); }

// Decays of a chunk's tokens, in powers of two: b_i = hi + lo (the sum of g up to
// token i as two floats, since b_i - b_j is small where b is large), exp(b_i)
// times the output's scale, exp(b_C - b_i), and exp(b_C).
template <int C>
struct alignas(16) Decays {
    float hi[C], lo[C], eb[C], w[C], end;

    // By one wave whose lane i holds g_i; lanes from C on hold 0.
    __device__ __forceinline__ void set(float g, float scale, int lane) {
        const double b = running_sum((g < kMinLogDecay ? kMinLogDecay : g) * 1.4426950408889634);
        const u2 bits = __builtin_bit_cast(u2, b);
        u2 last;
        last[0] = __builtin_amdgcn_readlane(bits[0], 63);
        last[1] = __builtin_amdgcn_readlane(bits[1], 63);
        if (lane < C) {
            const float h = (float)b, e = exp2_(h);
            hi[lane] = h;
            lo[lane] = (float)(b - (double)h);
            eb[lane] = scale * e;
            w[lane] = exp2_((float)(__builtin_bit_cast(double, last) - b));
            if (lane == C - 1) end = e;
        }
    }
};

// Where a workgroup of NW waves works; the waves own 16 columns each.
template <class T, int NW>
struct Place {
    Segment sg;
    int head, slice, slot, e0;                 // e0: the wave's first column
    bool last;                                 // of its sequence's segments
    const T *q, *k, *v;
    const float* g;
    long long state;                           // of the head in a slot

    // Whether there is anything to do.
    __device__ __forceinline__ bool find(const LinAttnArgs& a, bool full, int wave, int lane) {
        // Blocks go to the eight XCDs, each with an L2 of its own, in turn; those that
        // read the same q and k (the heads that share them, the slices of a head)
        // are put eight apart.
        const int sharers = a.rep * a.slices, groups = a.heads / a.rep;
        const int all = a.n_segs * groups, set = 8 * sharers;
        const int at = blockIdx.x / set, width = min(8, all - 8 * at), in = blockIdx.x - at * set;
        const int sharer = in / width, group = 8 * at + in - sharer * width;
        const int j_seg = group / groups;
        const int member = sharer / a.slices;
        slice = sharer - member * a.slices;
        head = (group - j_seg * groups) * a.rep + member;
        sg = linattn_segment(a, j_seg, lane);
        last = sg.t1 >= sg.len;
        if (!sg.ok || (!full && last)) return false;       // nothing follows the last segment
        slot = linattn_slot(a, sg.seq);
        if (slot < 0) return false;
        const int c0 = slice * 16 * NW;
        e0 = c0 + 16 * wave;
        q = (const T*)a.q + (long long)(head / a.rep) * a.qh;
        k = (const T*)a.k + (long long)(head / a.rep) * a.kh;
        v = (const T*)a.v + (long long)head * a.vh + c0;
        g = a.g + (long long)head * a.gh;
        state = (long long)head * a.dk * a.dv;
        return true;
    }
    __device__ __forceinline__ float* segment_state(const LinAttnArgs& a) const {
        return a.ws_state + (long long)sg.state * a.heads * a.dk * a.dv + state;
    }
    // Where the state comes from (null: zeros) and goes to (null: nowhere).  Of a
    // cut sequence every segment's comes from the workspace, the first one's too:
    // s_out may be s_in, and the last segment's workgroup may end before the
    // first one's begins.
    __device__ __forceinline__ const float* source(const LinAttnArgs& a, bool full) const {
        if (!full) return nullptr;
        if (sg.index > 0 || !last) return segment_state(a);
        return a.s_in ? a.s_in + (long long)slot * a.s_stride + state : nullptr;
    }
    __device__ __forceinline__ float* sink(const LinAttnArgs& a, bool full) const {
        if (!full) return segment_state(a);
        return last && a.s_out ? a.s_out + (long long)slot * a.s_stride + state : nullptr;
    }
    // Byte of the state's value (d, e0 + lane's column); past the end for d >= dk or
    // a column >= dv.
    __device__ __forceinline__ unsigned state_at(const LinAttnArgs& a, int d, int m) const {
        return e0 + m < a.dv ? (unsigned)(d * a.dv + e0 + m) * 4u : kOut;
    }
};

// The state in registers: S[dt][r] of lane 16 g + m is (d, column m) with the d of
// two tiles such that a lane has eight neighbouring ones.
__device__ __forceinline__ int state_row(int dt, int r, int g) {
    return 16 * (dt & ~1) + 8 * g + 4 * (dt & 1) + r;
}
template <int DT, class P>
__device__ __forceinline__ void read_state(f4 (&S)[DT], const P& pl, const LinAttnArgs& a, bool full, int m, int g) {
    const float* src = pl.source(a, full);
    const auto b = buffer(src, src ? 4ll * a.dk * a.dv : 0);
    #pragma unroll
    for (int dt = 0; dt < DT; ++dt)
        #pragma unroll
        for (int r = 0; r < 4; ++r)
            S[dt][r] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(
                                                     b, pl.state_at(a, state_row(dt, r, g), m), 0, 0));
}
template <int DT, class P>
__device__ __forceinline__ void write_state(const f4 (&S)[DT], const P& pl, const LinAttnArgs& a, bool full, int m,
                                            int g) {
    float* dst = pl.sink(a, full);
    const auto b = buffer(dst, dst ? 4ll * a.dk * a.dv : 0);
    #pragma unroll
    for (int dt = 0; dt < DT; ++dt)
        #pragma unroll
        for (int r = 0; r < 4; ++r)
            __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, (float)S[dt][r]), b,
                                                  pl.state_at(a, state_row(dt, r, g), m), 0, 0);
}

// A tensor's rows of a chunk of C tokens on their way to LDS: W columns (the
// first `cols` are the tensor's) as 16-byte pieces dealt over NT threads.  VEC:
// buffer loads; a piece's offset from the chunk's first row never changes, and
// what lies past the rows or columns comes back as zero.  Where a thread's
// pieces are whole rows apart, one offset serves them all.  Else (odd sizes,
// strides or addresses): 16-byte loads at any alignment within the row.
// 16 sequences of 2000 tokens, 16 heads of 127 in bf16: 204 us (heads of 128 184; by
// single values the former took 496).
template <class T, int W, int C, int NT, bool VEC>
struct Rows {
    static constexpr int E = 16 / sizeof(T);               // elements of a piece
    static constexpr int PER = W / E, N = (C * PER + NT - 1) / NT;
    static constexpr bool STEPS = NT % PER == 0 && C % (NT / PER) == 0;
    static constexpr int STEP = STEPS ? NT / PER : 0;
    u4 x[N];
    unsigned at[STEPS ? 1 : N];

    static __device__ __forceinline__ int row(int p, int tid) { return (tid + p * NT) / PER; }
    static __device__ __forceinline__ int col(int p, int tid) { return (tid + p * NT) % PER * E; }

    __device__ __forceinline__ void init(long long stride, int cols, int tid) {
        #pragma unroll
        for (int p = 0; p < (STEPS ? 1 : N); ++p) {
            const int r = row(p, tid), c = col(p, tid);
            at[p] = r < C && c < cols ? (unsigned)(r * (int)stride + c) * (unsigned)sizeof(T) : kOut;
        }
    }
    __device__ __forceinline__ void load(const T* base, long long stride, int cols, int n, int tid) {
        if (VEC && n == C) {
            // every row is there: the steps between a thread's pieces are scalar
            // offsets, which no bound is checked with
            const auto b = buffer(base, kOut);
            #pragma unroll
            for (int p = 0; p < N; ++p)
                x[p] = __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(
                                                  b, at[STEPS ? 0 : p], p * STEP * (int)stride * (int)sizeof(T), 0));
        } else if (VEC) {
            #pragma unroll
            for (int p = 0; p < N; ++p) {
                const int left = n - p * STEP;
                const auto b = buffer(base + p * STEP * stride,
                                      left > 0 ? ((left - 1) * stride + cols) * (int)sizeof(T) : 0);
                x[p] = __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(b, at[STEPS ? 0 : p], 0, 0));
            }
        } else {
            #pragma unroll
            for (int p = 0; p < N; ++p) {
                const int r = row(p, tid), c = col(p, tid);
                x[p] = u4{0, 0, 0, 0};
                if (r < n && c < cols) {
                    const T* from = base + r * stride;
                    if (cols >= E) {
                        // one load at any alignment; a row's last piece is the row's
                        // last E values, shifted by settle()
                        __builtin_memcpy(&x[p], from + min(c, cols - E), 16);
                    } else {
                        alignas(16) T y[E];
                        #pragma unroll
                        for (int i = 0; i < E; ++i) y[i] = i < cols ? from[i] : (T)0.0f;
                        x[p] = *(const u4*)y;
                    }
                }
            }
        }
    }
    // Once the pieces are there, before their use.
    __device__ __forceinline__ void settle(int cols, int tid) {
        if (VEC) return;
        #pragma unroll
        for (int p = 0; p < N; ++p) {
            const int over = col(p, tid) + E - cols;         // values of the piece past the row's end
            if (over > 0 && over < E && cols >= E)
                x[p] = __builtin_bit_cast(u4, __builtin_bit_cast(unsigned __int128, x[p]) >> (8 * sizeof(T) * over));
        }
    }
};

}  // namespace chunk
}  // namespace ssla
