// linattn_step.hip -- linear attention for one token of every sequence.
//
// Each state is read and written once: 8 bytes a value against four
// operations, so memory bounds it.  A workgroup owns a head of a sequence, or a
// stretch of its columns where there are few of them; a thread owns W
// neighbouring columns (16 bytes) and every `lanes`-th row, eight rows in
// flight.  Rows' q and k wait in LDS, so that the state's first loads are out
// before them; the products with q are summed over the row lanes through LDS.
// 64 sequences of 16 heads of 128 x 128 (134 MB) take 23.4 us, 5.8 TB/s out of the
// caches; 1021 of 8 heads of 96 x 80 (502 MB) 101 us, 5.0 TB/s, as a large copy; one
// of 16 heads 5 us, which is the launch and two dependent loads.
#include "linattn.h"

namespace ssla {
namespace {

constexpr int NT = 256;
constexpr int BATCH = 8;         // rows a thread has in flight

template <int W>
struct alignas(4 * W) Cols {
    float v[W];
};

template <class T, int W>
__global__ __launch_bounds__(NT) void k_linattn_step(const LinAttnArgs a, int cols, int parts) {
    __shared__ float qk[2][kLinAttnMaxDim];
    __shared__ float sums[NT * W];
    const int tid = threadIdx.x;
    const int sh = blockIdx.x / parts, part = blockIdx.x - sh * parts;
    const int seq = sh / a.heads, head = sh - seq * a.heads;
    const int slot = linattn_slot(a, seq);
    if (slot < 0) return;
    const int e0 = part * cols, ne = min(cols, a.dv - e0);       // the workgroup's columns
    const int wide = ne / W, lanes = min(NT / wide, a.dk);       // threads along a row, rows at a time
    const int y = tid / wide, x = tid - y * wide;
    const bool on = y < lanes;
    const long long at = (long long)slot * a.s_stride + (long long)head * a.dk * a.dv + e0 + x * W;
    const float* src = a.s_in + at;
    float* dst = a.s_out + at;

    Cols<W> s[BATCH];
    auto load = [&](int d0) {
        #pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int d = d0 + i * lanes;
            if (on && d < a.dk) s[i] = *(const Cols<W>*)(src + d * a.dv);
        }
    };
    load(y);
    const T* q = (const T*)a.q + seq * a.qt + (long long)(head / a.rep) * a.qh;
    const T* k = (const T*)a.k + seq * a.kt + (long long)(head / a.rep) * a.kh;
    const T* vp = (const T*)a.v + seq * a.vt + (long long)head * a.vh + e0 + x * W;
    if (tid < a.dk) {
        qk[0][tid] = (float)q[tid];
        qk[1][tid] = (float)k[tid];
    }
    float v[W], o[W];
    #pragma unroll
    for (int i = 0; i < W; ++i) {
        v[i] = on ? (float)vp[i] : 0.0f;
        o[i] = 0.0f;
    }
    const float decay = expf(a.g[seq * a.gt + (long long)head * a.gh]);
    __syncthreads();
    for (int d0 = y; d0 < a.dk; d0 += BATCH * lanes) {
        #pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int d = d0 + i * lanes;
            if (on && d < a.dk) {
                const float qd = qk[0][d], kd = qk[1][d];
                #pragma unroll
                for (int c = 0; c < W; ++c) {
                    s[i].v[c] = fmaf(kd, v[c], decay * s[i].v[c]);
                    o[c] = fmaf(qd, s[i].v[c], o[c]);
                }
                *(Cols<W>*)(dst + d * a.dv) = s[i];
            }
        }
        if (d0 + BATCH * lanes < a.dk) load(d0 + BATCH * lanes);
    }
    if (on) {
        #pragma unroll
        for (int c = 0; c < W; ++c) sums[y * ne + x * W + c] = o[c];
    }
    __syncthreads();
    // a column's sums by up to four threads, and theirs by the first
    const int c = tid >> 2, l = tid & 3;
    T* out = (T*)a.out + seq * a.ot + (long long)head * a.oh + e0;
    for (int e = c; e < ne; e += NT / 4) {
        float t = 0.0f;
        for (int i = l; i < lanes; i += 4) t += sums[i * ne + e];
        t += __shfl_xor(t, 1);
        t += __shfl_xor(t, 2);
        if (l == 0) out[e] = (T)(a.scale * t);
    }
}

template <class T>
hipError_t launch(const LinAttnArgs& a, hipStream_t st) {
    const bool wide = a.dv % 4 == 0 && a.s_stride % 4 == 0 && (size_t)a.s_in % 16 == 0 && (size_t)a.s_out % 16 == 0;
    const int w = wide ? 4 : 1;
    // Columns of a workgroup: all, or down to 16 (64 bytes of a row) while the
    // heads alone leave most of the 256 CUs idle.
    const long long heads = (long long)a.n_seqs * a.heads;
    int parts = 1;
    while (parts < 16 && heads * parts < 512 && a.dv / (2 * parts) >= 16) parts *= 2;
    int cols = (a.dv + parts - 1) / parts;
    cols = (cols + w - 1) / w * w;
    parts = (a.dv + cols - 1) / cols;
    LinAttnArgs args = a;
    void* pa[] = {&args, &cols, &parts};
    return hipLaunchKernel(wide ? (const void*)k_linattn_step<T, 4> : (const void*)k_linattn_step<T, 1>,
                           dim3((unsigned)(heads * parts)), dim3(NT), pa, 0, st);
}

}  // namespace

hipError_t linattn_launch_step(const LinAttnArgs& a, int dtype, hipStream_t st) {
    if (dtype == SSLA_F32) return launch<float>(a, st);
    if (dtype == SSLA_BF16) return launch<__bf16>(a, st);
    return launch<_Float16>(a, st);
}

}  // namespace ssla
