// ops.cpp -- C ABI of the sequence operators (include/ssla_hip.h): argument
// checks, how a call is cut into workgroups, launches.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <exception>
#include <string>

#include "drain_scan.h"
#include "groupnorm.h"
#include "linattn.h"
#include "ssla_hip.h"

namespace ssla {
namespace {

int refuse(const std::string& msg) {
    set_error(msg);
    return SSLA_ERR_ARG;
}

int hip_failed(const char* what, hipError_t e) {
    set_error(std::string(what) + ": " + hipGetErrorString(e));
    return SSLA_ERR_HIP;
}

size_t element(int dtype) { return dtype == SSLA_F32 ? 4 : 2; }

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Whether n0 x n1 pieces of `width` elements at strides s0, s1 are apart.
bool apart(long long n0, long long s0, long long n1, long long s1, long long width) {
    if (n0 <= 1) return n1 <= 1 || s1 >= width;
    if (n1 <= 1) return s0 >= width;
    if (s0 < s1) return s0 >= width && (s1 - width) / s0 >= n0 - 1;
    return s1 >= width && (s0 - width) / s1 >= n1 - 1;
}

// Whether a launch of a * b * c workgroups fits: HIP counts a grid's threads in 32 bits.
bool launchable(long long a, long long b, long long c, int threads) {
    return (__int128)a * b * c <= 0xffffffffll / threads;
}

// Kernels count tokens, rows and channels in 32 bits and step past the last one.
constexpr int kMaxCount = 0x7fff0000;
constexpr long long kMaxStride = 1ll << 40;      // offsets stay within 64 bits

// ---- linear attention ----------------------------------------------------------

int check_linattn(const SslaHipLinAttn* d, bool step, const char* fn) {
    const std::string f = std::string(fn) + ": ";
    if (!d) return refuse(f + "null descriptor");
    if (d->dtype != SSLA_F32 && d->dtype != SSLA_BF16 && d->dtype != SSLA_F16)
        return refuse(f + "dtype must be SSLA_F32, SSLA_BF16 or SSLA_F16");
    if (d->heads < 1 || d->qk_heads < 1 || d->heads % d->qk_heads)
        return refuse(f + "heads must be a positive multiple of qk_heads");
    if (d->dk < 1 || d->dk > kLinAttnMaxDim || d->dv < 1 || d->dv > kLinAttnMaxDim)
        return refuse(f + "dk and dv must be 1 .. 256");
    if (d->n_seqs < 0 || d->n_slots < 0) return refuse(f + "negative count");
    const long long* strides[5] = {d->q_stride, d->k_stride, d->v_stride, d->decay_stride, d->out_stride};
    for (const long long* s : strides)
        if (s[0] < 0 || s[1] < 0 || s[0] > kMaxStride || s[1] > kMaxStride)
            return refuse(f + "strides must be 0 .. 2^40");
    long long tokens = d->n_seqs;
    if (!step) {
        if (d->n_tokens < 0 || d->n_tokens > kMaxCount || d->max_len < 0)
            return refuse(f + "n_tokens must be 0 .. 2^31 - 2^16, max_len not negative");
        if (!d->cu_seqlens && d->n_tokens != (long long)d->n_seqs * d->max_len)
            return refuse(f + "without cu_seqlens n_tokens must be n_seqs * max_len");
        tokens = d->n_tokens;
    }
    const size_t e = element(d->dtype);
    if (tokens > 0 && d->n_seqs > 0) {
        if (!d->q || !d->k || !d->v || !d->log_decay || !d->out) return refuse(f + "null tensor");
        if (!apart(tokens, d->out_stride[0], d->heads, d->out_stride[1], d->dv))
            return refuse(f + "rows of out overlap");
        if (d->out == d->q || d->out == d->k || d->out == d->v) return refuse(f + "out is an input");
    }
    if (!aligned(d->q, e) || !aligned(d->k, e) || !aligned(d->v, e) || !aligned(d->out, e) ||
        !aligned(d->log_decay, 4) || !aligned(d->cu_seqlens, 4) || !aligned(d->slots, 4) ||
        !aligned(d->state_in, 4) || !aligned(d->state_out, 4))
        return refuse(f + "a pointer is not aligned to its element");
    if (step && d->n_seqs > 0 && (!d->state_in || !d->state_out))
        return refuse(f + "state_in and state_out are needed");
    const long long state = (long long)d->heads * d->dk * d->dv;
    if (d->state_in || d->state_out) {
        if (d->state_stride < state || d->state_stride > kMaxStride)
            return refuse(f + "state_stride must be heads * dk * dv .. 2^40");
        if (!d->slots && d->n_slots < d->n_seqs) return refuse(f + "fewer slots than sequences");
        const uintptr_t a = (uintptr_t)d->state_in, b = (uintptr_t)d->state_out;
        const uintptr_t span = d->n_slots ? 4 * (uintptr_t)((d->n_slots - 1) * d->state_stride + state) : 0;
        // floats from a slot of the lower pool to the next one of the higher: the slots of
        // two pools may lie in turn
        const uintptr_t next = (a < b ? b - a : a - b) / 4 % (uintptr_t)d->state_stride;
        const bool in_turn = next >= (uintptr_t)state && next + state <= (uintptr_t)d->state_stride;
        if (a && b && a != b && a < b + span && b < a + span && !in_turn)
            return refuse(f + "state_in and state_out overlap without being the same");
    }
    return SSLA_OK;
}

// Rows that buffer loads of 16-byte pieces can take: the address, both strides
// and the row's end are whole pieces, rows are apart (what lies past a chunk's
// last row must lie past the buffer's end) and 64 of them span less than 2^31
// bytes.
bool pieces(const void* p, const long long* s, long long width, size_t e) {
    const long long n = 16 / (long long)e;
    return aligned(p, 16) && s[0] % n == 0 && s[1] % n == 0 && width % n == 0 && s[0] >= width &&
           s[0] < (1 << 22);
}

// Segment length.  A workgroup takes one segment of a head; cutting a sequence
// costs its k and v a second reading and a state written, chained and read for
// each segment.  Whole sequences are taken where none is longer than 256 tokens
// (200 tokens of 4 heads of 24: 11.9 us whole, 12.2 cut; 300 of 16 heads of 128:
// 26 whole, 21 cut), and while none holds more than one and a half of a compute
// unit's share of all tokens and heads (16 sequences of 8192 tokens, 16 heads of
// 128, one workgroup a compute unit: 0.69 ms whole, 0.84 cut in two, on one card).  Else
// segments are the smallest power of two, from 64 tokens on, that leaves a
// sequence at most 128 (they are chained in turn: 20000 tokens of one head of 64,
// 60 us in 313 segments, 38 in 79), and each of the 256 compute units two (one
// sequence of 8192, 16 heads of 128: 83 us, with one each 85), or one and a half
// where segments are shorter than 256 (2000 tokens of 16 heads of 128: 43 us in 500
// workgroups, 35 in 250).  False where the segments cannot be counted.
bool cut(const SslaHipLinAttn* d, LinAttnArgs& a) {
    const long long rows = d->n_tokens * d->heads * a.slices;
    int shift = 6;
    while ((rows >> shift) > (shift < 8 ? kCUs + kCUs / 2 : 2 * kCUs) || (a.max_len >> shift) > 128) ++shift;
    if (a.max_len <= 256 || a.max_len <= (1ll << shift) || 2 * kCUs * (long long)a.max_len <= 3 * rows) {
        a.seg_shift = 31;                              // no sequence is cut
        a.n_segs = d->n_seqs;
        a.n_states = 0;
        a.by_length = d->cu_seqlens && d->n_seqs > 1 && d->n_seqs <= 64 &&
                      (long long)d->n_seqs * a.max_len > d->n_tokens;
        return true;
    }
    a.seg_shift = shift;
    const long long segs = d->cu_seqlens ? (d->n_tokens >> shift) + d->n_seqs
                                         : d->n_seqs * ((a.max_len + (1ll << shift) - 1) >> shift);
    const long long pairs = 2 * (d->n_tokens >> shift);      // see linattn_states
    a.n_segs = (int)segs;
    a.paired = d->cu_seqlens && pairs < segs;
    a.n_states = (int)(a.paired ? pairs : segs);
    return segs <= 0x7fffffff;
}

LinAttnArgs linattn_args(const SslaHipLinAttn* d) {
    LinAttnArgs a{};
    a.q = d->q, a.k = d->k, a.v = d->v, a.out = d->out, a.g = d->log_decay;
    a.qt = d->q_stride[0], a.qh = d->q_stride[1];
    a.kt = d->k_stride[0], a.kh = d->k_stride[1];
    a.vt = d->v_stride[0], a.vh = d->v_stride[1];
    a.gt = d->decay_stride[0], a.gh = d->decay_stride[1];
    a.ot = d->out_stride[0], a.oh = d->out_stride[1];
    a.cu = d->cu_seqlens, a.slots = d->slots;
    a.s_in = d->state_in, a.s_out = d->state_out, a.s_stride = d->state_stride;
    a.n_tokens = d->n_tokens;
    a.n_seqs = d->n_seqs, a.n_slots = d->n_slots;
    a.max_len = (int)(d->max_len < d->n_tokens ? d->max_len : d->n_tokens);
    a.heads = d->heads, a.rep = d->heads / d->qk_heads, a.dk = d->dk, a.dv = d->dv;
    const int cols = 16 * linattn_waves(d->dk, d->dv);
    a.slices = (d->dv + cols - 1) / cols;
    const size_t e = element(d->dtype);
    a.vec = pieces(d->q, d->q_stride, d->dk, e) && pieces(d->k, d->k_stride, d->dk, e) &&
            pieces(d->v, d->v_stride, d->dv, e) && pieces(d->out, d->out_stride, d->dv, e);
    a.scale = d->scale;
    return a;
}

size_t linattn_bytes(const LinAttnArgs& a) {
    return (size_t)a.n_states * a.heads * ((size_t)a.dk * a.dv + 1) * 4;
}

// ---- group norm ------------------------------------------------------------------

int check_group_norm(const SslaHipGroupNorm* d) {
    const std::string f = "ssla_hip_group_norm: ";
    if (!d) return refuse(f + "null descriptor");
    if (d->dtype != SSLA_F32 && d->dtype != SSLA_BF16 && d->dtype != SSLA_F16)
        return refuse(f + "dtype must be SSLA_F32, SSLA_BF16 or SSLA_F16");
    if (d->n < 0 || d->rows < 0 || d->channels < 0) return refuse(f + "negative size");
    if (d->rows > kMaxCount || d->channels > kMaxCount)
        return refuse(f + "rows and channels must be at most 2^31 - 2^16");
    if (d->groups < 1 || d->channels % d->groups) return refuse(f + "groups must divide channels");
    if (d->act < SSLA_ACT_NONE || d->act > SSLA_ACT_RELU) return refuse(f + "unknown activation");
    if (!(d->eps >= 0.0f)) return refuse(f + "eps must not be negative");
    const long long* strides[3] = {d->x_stride, d->gate_stride, d->out_stride};
    for (const long long* s : strides)
        if (s[0] < 0 || s[1] < 0 || s[0] > kMaxStride || s[1] > kMaxStride)
            return refuse(f + "strides must be 0 .. 2^40");
    const size_t e = element(d->dtype);
    if (!aligned(d->x, e) || !aligned(d->gate, e) || !aligned(d->out, e) || !aligned(d->weight, e) ||
        !aligned(d->bias, e))
        return refuse(f + "a pointer is not aligned to its element");
    if (d->n && d->rows && d->channels) {
        if (!d->x || !d->out) return refuse(f + "null tensor");
        if (!apart(d->n, d->out_stride[0], d->rows, d->out_stride[1], d->channels))
            return refuse(f + "rows of out overlap");
        if ((d->out == d->x && (d->out_stride[0] != d->x_stride[0] || d->out_stride[1] != d->x_stride[1])) ||
            (d->out == d->gate &&
             (d->out_stride[0] != d->gate_stride[0] || d->out_stride[1] != d->gate_stride[1])))
            return refuse(f + "out in an input's place needs that input's strides");
    }
    return SSLA_OK;
}

GroupNormArgs group_norm_args(const SslaHipGroupNorm* d) {
    GroupNormArgs a{};
    a.x = d->x, a.gate = d->gate, a.weight = d->weight, a.bias = d->bias, a.out = d->out;
    a.xn = d->x_stride[0], a.xr = d->x_stride[1];
    a.gn = d->gate_stride[0], a.gr = d->gate_stride[1];
    a.on = d->out_stride[0], a.orow = d->out_stride[1];
    a.n = d->n, a.rows = d->rows, a.channels = d->channels, a.groups = d->groups, a.act = d->act;
    a.eps = d->eps;
    group_norm_plan(a, d->dtype);
    return a;
}

size_t group_norm_bytes(const GroupNormArgs& a) {
    return (size_t)a.parts * a.n * a.groups * 2 * sizeof(double);
}

}  // namespace
}  // namespace ssla

using namespace ssla;

extern "C" {

int ssla_hip_ops_layout(long long* out, int cap) {
    if (!out || cap < 2) {
        set_error("ssla_hip_ops_layout: need 2 slots");
        return SSLA_ERR_ARG;
    }
    out[0] = sizeof(SslaHipLinAttn);
    out[1] = sizeof(SslaHipGroupNorm);
    return SSLA_OK;
}

int ssla_hip_linattn_workspace(const SslaHipLinAttn* d, size_t* nbytes) try {
    if (!nbytes) return refuse("ssla_hip_linattn_workspace: null argument");
    *nbytes = 0;
    if (const int rc = check_linattn(d, false, "ssla_hip_linattn_workspace")) return rc;
    LinAttnArgs a = linattn_args(d);
    if (!cut(d, a)) return refuse("ssla_hip_linattn_workspace: too many sequences");
    *nbytes = linattn_bytes(a);
    return SSLA_OK;
} catch (const std::exception&) {
    return SSLA_ERR_ARG;
}

int ssla_hip_linattn(const SslaHipLinAttn* d, void* workspace, size_t workspace_bytes, void* stream) try {
    if (const int rc = check_linattn(d, false, "ssla_hip_linattn")) return rc;
    if (d->n_seqs == 0) return SSLA_OK;
    LinAttnArgs a = linattn_args(d);
    if (!cut(d, a)) return refuse("ssla_hip_linattn: too many sequences");
    const size_t need = linattn_bytes(a);
    if (!launchable(a.n_segs, a.heads, a.slices, 64 * linattn_waves(a.dk, a.dv)) ||
        (need && !launchable(a.n_seqs, a.heads, (a.dk * a.dv + 255) / 256, 256)))
        return refuse("ssla_hip_linattn: too many sequences and heads");
    if (need) {
        if (!workspace || workspace_bytes < need || !aligned(workspace, 16))
            return refuse("ssla_hip_linattn: the workspace is missing, too small or not 16-byte aligned");
        a.ws_state = (float*)workspace;
        a.ws_decay = a.ws_state + (size_t)a.n_states * a.heads * a.dk * a.dv;
    }
    const hipStream_t st = (hipStream_t)stream;
    hipError_t (*run)(const LinAttnArgs&, bool, hipStream_t) =
        d->dtype == SSLA_F32 ? linattn_launch_f32 : d->dtype == SSLA_BF16 ? linattn_launch_bf16 : linattn_launch_f16;
    hipError_t e = hipSuccess;
    if (need) {
        e = run(a, false, st);
        if (e == hipSuccess) e = linattn_launch_chain(a, st);
    }
    if (e == hipSuccess) e = run(a, true, st);
    return e == hipSuccess ? SSLA_OK : hip_failed("ssla_hip_linattn", e);
} catch (const std::exception&) {
    return SSLA_ERR_HIP;
}

int ssla_hip_linattn_step(const SslaHipLinAttn* d, void* stream) try {
    if (const int rc = check_linattn(d, true, "ssla_hip_linattn_step")) return rc;
    if (d->n_seqs == 0) return SSLA_OK;
    const LinAttnArgs a = linattn_args(d);
    if (!launchable(a.n_seqs, a.heads, 1, 256))
        return refuse("ssla_hip_linattn_step: too many sequences and heads");
    const hipError_t e = linattn_launch_step(a, d->dtype, (hipStream_t)stream);
    return e == hipSuccess ? SSLA_OK : hip_failed("ssla_hip_linattn_step", e);
} catch (const std::exception&) {
    return SSLA_ERR_HIP;
}

int ssla_hip_group_norm_workspace(const SslaHipGroupNorm* d, size_t* nbytes) try {
    if (!nbytes) return refuse("ssla_hip_group_norm_workspace: null argument");
    *nbytes = 0;
    if (const int rc = check_group_norm(d)) return rc;
    if (d->n && d->rows && d->channels) *nbytes = group_norm_bytes(group_norm_args(d));
    return SSLA_OK;
} catch (const std::exception&) {
    return SSLA_ERR_ARG;
}

int ssla_hip_group_norm(const SslaHipGroupNorm* d, void* workspace, size_t workspace_bytes, void* stream) try {
    if (const int rc = check_group_norm(d)) return rc;
    if (!d->n || !d->rows || !d->channels) return SSLA_OK;
    GroupNormArgs a = group_norm_args(d);
    const size_t need = group_norm_bytes(a);
    if (a.kind == kGroupLanes ? !launchable(a.n, a.groups, a.reps, 1)
                              : !launchable(a.n, a.parts ? a.parts : 1, a.blocks, a.threads))
        return refuse("ssla_hip_group_norm: too many items and groups");
    if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
        return refuse("ssla_hip_group_norm: the workspace is missing, too small or not 16-byte aligned");
    a.ws = (double*)workspace;
    const hipError_t e = group_norm_launch(a, d->dtype, (hipStream_t)stream);
    return e == hipSuccess ? SSLA_OK : hip_failed("ssla_hip_group_norm", e);
} catch (const std::exception&) {
    return SSLA_ERR_HIP;
}

}  // extern "C"
