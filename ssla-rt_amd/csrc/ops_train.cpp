// ops_train.cpp -- C ABI of the operators that have gradients
// (include/ssla_hip.h): argument checks, launches.
#include <exception>
#include <string>

#include "layernorm.h"
#include "linrec.h"
#include "ops_check.h"

namespace ssla {
namespace {

// ---- gated linear recurrence -----------------------------------------------------

// Floats of a pool of n slots.
uintptr_t pool_bytes(long long n, long long stride, long long width) {
    return n ? 4 * (uintptr_t)((n - 1) * stride + width) : 0;
}

int check_pools(const SslaHipLinRec* d, const std::string& f) {
    for (const long long s : {d->state_in ? d->state_in_stride : d->channels,
                              d->state_out ? d->state_out_stride : d->channels})
        if (s < d->channels || s > kMaxStride) return refuse(f + "state strides must be channels .. 2^40");
    if (!d->slots && (d->state_in || d->state_out) && d->n_slots < d->n_seqs)
        return refuse(f + "fewer slots than sequences");
    const uintptr_t a = (uintptr_t)d->state_in, b = (uintptr_t)d->state_out;
    if (!a || !b) return SSLA_OK;
    const long long c = d->channels, si = d->state_in_stride, so = d->state_out_stride;
    if (a == b) return si == so || d->n_slots < 2 ? SSLA_OK : refuse(f + "a pool in its own place needs one stride");
    // the slots of two pools may lie in turn
    const uintptr_t next = (a < b ? b - a : a - b) / 4 % (uintptr_t)si;
    const bool in_turn = si == so && next >= (uintptr_t)c && next + c <= (uintptr_t)si;
    if (a < b + pool_bytes(d->n_slots, so, c) && b < a + pool_bytes(d->n_slots, si, c) && !in_turn)
        return refuse(f + "state_in and state_out overlap without being the same");
    return SSLA_OK;
}

enum Call { kForward, kBackward, kStep, kSizes };      // kSizes: before there is an out

int check_linrec(const SslaHipLinRec* d, Call call, const char* fn) {
    const bool step = call == kStep, writes = call == kForward || step;
    const std::string f = std::string(fn) + ": ";
    if (!d) return refuse(f + "null descriptor");
    if (!is_dtype(d->dtype)) return refuse(f + "dtype must be SSLA_F32, SSLA_BF16 or SSLA_F16");
    if (d->channels < 1 || d->channels > kMaxCount) return refuse(f + "channels must be 1 .. 2^31 - 2^16");
    if (d->n_seqs < 0 || d->n_slots < 0) return refuse(f + "negative count");
    if (d->wait_us > 1000000) return refuse(f + "wait_us must be at most 10^6");
    if (d->n_seqs > kMaxCount) return refuse(f + "n_seqs must be at most 2^31 - 2^16");
    if (!is_stride(d->gate_stride) || !is_stride(d->v_stride) || !is_stride(d->q_stride) || !is_stride(d->out_stride))
        return refuse(f + "strides must be 0 .. 2^40");
    long long tokens = d->n_seqs;
    if (!step) {
        if (d->n_tokens < 0 || d->n_tokens > kMaxCount) return refuse(f + "n_tokens must be 0 .. 2^31 - 2^16");
        if (!d->cu_seqlens && (d->n_seqs ? d->n_tokens % d->n_seqs : d->n_tokens))
            return refuse(f + "without cu_seqlens n_tokens must be a multiple of n_seqs");
        tokens = d->n_tokens;
    }
    const size_t e = element(d->dtype);
    if (tokens > 0) {
        if (!d->gate || !d->v || (writes && !d->out)) return refuse(f + "null tensor");
        if (writes) {
            if (tokens > 1 && d->out_stride < d->channels) return refuse(f + "rows of out overlap");
            if (d->out == d->gate || d->out == d->v || d->out == d->q) return refuse(f + "out is an input");
        } else if (call == kBackward && !d->carries) {
            return refuse(f + "no carries");
        }
    }
    if (!aligned(d->gate, e) || !aligned(d->v, e) || !aligned(d->q, e) || (writes && !aligned(d->out, e)) ||
        !aligned(d->cu_seqlens, 4) || !aligned(d->slots, 4) || !aligned(d->state_in, 4) ||
        !aligned(d->state_out, 4) || !aligned(d->carries, 4))
        return refuse(f + "a pointer is not aligned to its element");
    if (step && d->n_seqs > 0 && (!d->state_in || !d->state_out))
        return refuse(f + "state_in and state_out are needed");
    if (d->slots && (call == kBackward || (call == kForward && d->carries)))
        return refuse(f + "there are no gradients by slots");
    if (writes) return check_pools(d, f);
    if (d->state_in && (d->state_in_stride < d->channels || d->state_in_stride > kMaxStride))
        return refuse(f + "state strides must be channels .. 2^40");
    return SSLA_OK;
}

int check_linrec_grad(const SslaHipLinRec* d, const SslaHipLinRecGrad* g) {
    const std::string f = "ssla_hip_linrec_backward: ";
    if (!g) return refuse(f + "null descriptor");
    const size_t e = element(d->dtype);
    if (!is_stride(g->dout_stride)) return refuse(f + "strides must be 0 .. 2^40");
    const void* const out[3] = {g->dgate, g->dv, g->dq};
    const long long stride[3] = {g->dgate_stride, g->dv_stride, g->dq_stride};
    for (int i = 0; i < 3; ++i) {
        if (!out[i]) continue;
        if (!is_stride(stride[i])) return refuse(f + "strides must be 0 .. 2^40");
        if (d->n_tokens > 1 && stride[i] < d->channels) return refuse(f + "rows of a gradient overlap");
        if (!aligned(out[i], e)) return refuse(f + "a pointer is not aligned to its element");
        if (out[i] == d->gate || out[i] == d->v || out[i] == d->q || out[i] == g->dout)
            return refuse(f + "a gradient is an input");
    }
    if (g->dq && !d->q) return refuse(f + "dq without q");
    if (!aligned(g->dout, e) || !aligned(g->dstate_out, 4) || !aligned(g->dstate_in, 4))
        return refuse(f + "a pointer is not aligned to its element");
    if ((g->dstate_out && (g->dstate_out_stride < 0 || g->dstate_out_stride > kMaxStride)) ||
        (g->dstate_in && (g->dstate_in_stride > kMaxStride || g->dstate_in_stride < d->channels)))
        return refuse(f + "state strides must be channels .. 2^40");
    if (g->dstate_in && (g->dstate_in == g->dstate_out || g->dstate_in == d->state_in))
        return refuse(f + "a gradient is an input");
    return SSLA_OK;
}

LinRecArgs linrec_args(const SslaHipLinRec* d, const SslaHipLinRecGrad* g) {
    LinRecArgs a{};
    a.g = d->gate, a.v = d->v, a.q = d->q, a.out = d->out;
    a.gt = d->gate_stride, a.vt = d->v_stride, a.qt = d->q_stride, a.ot = d->out_stride;
    a.cu = d->cu_seqlens, a.slots = d->slots;
    a.s_in = d->state_in, a.s_out = d->state_out, a.si = d->state_in_stride, a.so = d->state_out_stride;
    a.carries = d->carries;
    a.patience = d->wait_us < 0 ? 0 : (d->wait_us ? d->wait_us : 200) * 100u;
    a.alone = d->wait_us == SSLA_LINREC_ALONE;
    a.n_tokens = d->n_tokens, a.n_seqs = d->n_seqs, a.n_slots = d->n_slots, a.channels = d->channels;
    if (!d->slots && !d->state_in && !d->state_out) a.n_slots = d->n_seqs;
    a.seq_len = d->n_seqs ? (int)(d->n_tokens / d->n_seqs) : 0;
    if (g) {
        a.out = nullptr, a.s_out = nullptr;
        a.n_slots = d->n_seqs;
        a.dout = g->dout, a.ds_out = g->dstate_out, a.dg = g->dgate, a.dv = g->dv, a.dq = g->dq, a.ds_in = g->dstate_in;
        a.dot = g->dout_stride, a.dgt = g->dgate_stride, a.dvt = g->dv_stride, a.dqt = g->dq_stride;
        a.dso = g->dstate_out_stride, a.dsi = g->dstate_in_stride;
    }
    linrec_plan(a, d->dtype, g != nullptr);
    return a;
}

// Workspace of either pass.
size_t linrec_need(const SslaHipLinRec* d) {
    const SslaHipLinRecGrad none{};
    const size_t one = linrec_bytes(linrec_args(d, nullptr), false), other = linrec_bytes(linrec_args(d, &none), true);
    return one > other ? one : other;
}

// The grid's limit, and the workspace.
int bind_linrec(LinRecArgs& a, const SslaHipLinRec* d, void* workspace, size_t bytes, const char* fn) {
    if (!launchable(a.tiles, a.blocks, 1, kLinRecThreads) ||
        !launchable((long long)a.tiles * a.blocks + a.n_seqs / linrec_threads(a) + 1, 1, 1, kLinRecThreads))
        return refuse(std::string(fn) + ": too many tokens and channels");
    const size_t need = linrec_need(d);
    if (!need) return SSLA_OK;
    if (!workspace || bytes < need || !aligned(workspace, 16))
        return refuse(std::string(fn) + ": the workspace is missing, too small or not 16-byte aligned");
    linrec_bind(a, workspace);
    if (a.firsts && !launchable(a.tiles + 1024ll, 1, 1, kLinRecThreads)) return refuse(std::string(fn) + ": too many tokens");
    return SSLA_OK;
}

// ---- layer norm --------------------------------------------------------------------

int check_layer_norm(const SslaHipLayerNorm* d, bool backward, const char* fn) {
    const std::string f = std::string(fn) + ": ";
    if (!d) return refuse(f + "null descriptor");
    if (!is_dtype(d->dtype)) return refuse(f + "dtype must be SSLA_F32, SSLA_BF16 or SSLA_F16");
    if (d->weight_dtype != d->dtype && d->weight_dtype != SSLA_F32)
        return refuse(f + "weight_dtype must be dtype or SSLA_F32");
    if (d->rows < 0 || d->channels < 0) return refuse(f + "negative size");
    if (d->rows > kMaxCount || d->channels > kMaxCount)
        return refuse(f + "rows and channels must be at most 2^31 - 2^16");
    if (!(d->eps >= 0.0f)) return refuse(f + "eps must not be negative");
    if (!is_stride(d->x_stride) || !is_stride(d->residual_stride) || (!backward && !is_stride(d->out_stride)))
        return refuse(f + "strides must be 0 .. 2^40");
    const size_t e = element(d->dtype), ew = element(d->weight_dtype);
    if (!aligned(d->x, e) || !aligned(d->residual, e) || (!backward && !aligned(d->out, e)) ||
        !aligned(d->weight, ew) || (!backward && !aligned(d->bias, ew)) || !aligned(d->stats, 4))
        return refuse(f + "a pointer is not aligned to its element");
    if (!d->rows || !d->channels) return SSLA_OK;
    if (!d->x) return refuse(f + "null tensor");
    if (backward) return d->stats ? SSLA_OK : refuse(f + "no stats");
    if (!d->out) return refuse(f + "null tensor");
    if (d->rows > 1 && d->out_stride < d->channels) return refuse(f + "rows of out overlap");
    if ((d->out == d->x && d->rows > 1 && d->out_stride != d->x_stride) ||
        (d->out == d->residual && d->rows > 1 && d->out_stride != d->residual_stride))
        return refuse(f + "out in an input's place needs that input's stride");
    return SSLA_OK;
}

int check_layer_norm_grad(const SslaHipLayerNorm* d, const SslaHipLayerNormGrad* g, const char* fn) {
    const std::string f = std::string(fn) + ": ";
    if (!g) return refuse(f + "null descriptor");
    const size_t e = element(d->dtype), ew = element(d->weight_dtype);
    if (!is_stride(g->dout_stride) || !is_stride(g->dx_stride)) return refuse(f + "strides must be 0 .. 2^40");
    if (!aligned(g->dout, e) || !aligned(g->dx, e) || !aligned(g->dweight, ew) || !aligned(g->dbias, ew))
        return refuse(f + "a pointer is not aligned to its element");
    if (!d->rows || !d->channels) return SSLA_OK;
    if (!g->dout) return refuse(f + "null tensor");
    if (g->dx && d->rows > 1 && g->dx_stride < d->channels) return refuse(f + "rows of dx overlap");
    for (const void* p : {(const void*)g->dx, (const void*)g->dweight, (const void*)g->dbias})
        if (p && (p == d->x || p == d->residual || p == d->weight || p == g->dout))
            return refuse(f + "a gradient is an input");
    return SSLA_OK;
}

LayerNormArgs layer_norm_args(const SslaHipLayerNorm* d, const SslaHipLayerNormGrad* g) {
    LayerNormArgs a{};
    a.x = d->x, a.res = d->residual, a.weight = d->weight, a.bias = d->bias, a.out = d->out, a.stats = d->stats;
    a.xr = d->x_stride, a.rr = d->residual_stride, a.orow = d->out_stride;
    a.rows = d->rows, a.channels = d->channels, a.wide = d->weight_dtype == SSLA_F32, a.eps = d->eps;
    if (g) {
        a.dout = g->dout, a.dx = g->dx, a.dw = g->dweight, a.db = g->dbias;
        a.dor = g->dout_stride, a.dxr = g->dx_stride;
    }
    layer_norm_plan(a, d->dtype, g != nullptr);
    return a;
}

// Grids of the backward pass: the rows', and those of the sums over them.
bool layer_norm_fits(const LayerNormArgs& a) {
    return launchable(a.wgs, 1, 1, a.threads) && launchable((a.channels - 1) / 256 + 1, a.reps ? 1 : a.parts, 1, 256) &&
           launchable((2ll * a.channels - 1) / 16 + 1, a.dw || a.db ? 1 : 0, 1, 1024);
}

size_t layer_norm_bytes(const LayerNormArgs& a) { return (size_t)a.parts * 2 * a.channels * 4; }

}  // namespace
}  // namespace ssla

using namespace ssla;

extern "C" {

int ssla_hip_train_layout(long long* out, int cap) {
    if (!out || cap < 4) {
        set_error("ssla_hip_train_layout: need 4 slots");
        return SSLA_ERR_ARG;
    }
    out[0] = sizeof(SslaHipLinRec);
    out[1] = sizeof(SslaHipLinRecGrad);
    out[2] = sizeof(SslaHipLayerNorm);
    out[3] = sizeof(SslaHipLayerNormGrad);
    return SSLA_OK;
}

int ssla_hip_linrec_carries(const SslaHipLinRec* d, size_t* nbytes) try {
    if (!nbytes) return refuse("ssla_hip_linrec_carries: null argument");
    *nbytes = 0;
    if (const int rc = check_linrec(d, kSizes, "ssla_hip_linrec_carries")) return rc;
    *nbytes = linrec_carries(linrec_args(d, nullptr));
    return SSLA_OK;
} catch (const std::exception&) {
    return SSLA_ERR_ARG;
}

int ssla_hip_linrec_workspace(const SslaHipLinRec* d, size_t* nbytes) try {
    if (!nbytes) return refuse("ssla_hip_linrec_workspace: null argument");
    *nbytes = 0;
    if (const int rc = check_linrec(d, kSizes, "ssla_hip_linrec_workspace")) return rc;
    *nbytes = linrec_need(d);
    return SSLA_OK;
} catch (const std::exception&) {
    return SSLA_ERR_ARG;
}

int ssla_hip_linrec(const SslaHipLinRec* d, void* workspace, size_t workspace_bytes, void* stream) try {
    const char* fn = "ssla_hip_linrec";
    if (const int rc = check_linrec(d, kForward, fn)) return rc;
    LinRecArgs a = linrec_args(d, nullptr);
    if (const int rc = bind_linrec(a, d, workspace, workspace_bytes, fn)) return rc;
    const hipError_t e = linrec_launch(a, d->dtype, (hipStream_t)stream);
    return e == hipSuccess ? SSLA_OK : hip_failed(fn, e);
} catch (const std::exception&) {
    return SSLA_ERR_HIP;
}

int ssla_hip_linrec_backward(const SslaHipLinRec* d, const SslaHipLinRecGrad* g, void* workspace,
                             size_t workspace_bytes, void* stream) try {
    const char* fn = "ssla_hip_linrec_backward";
    if (const int rc = check_linrec(d, kBackward, fn)) return rc;
    if (const int rc = check_linrec_grad(d, g)) return rc;
    LinRecArgs a = linrec_args(d, g);
    if (const int rc = bind_linrec(a, d, workspace, workspace_bytes, fn)) return rc;
    const hipError_t e = linrec_launch_backward(a, d->dtype, (hipStream_t)stream);
    return e == hipSuccess ? SSLA_OK : hip_failed(fn, e);
} catch (const std::exception&) {
    return SSLA_ERR_HIP;
}

int ssla_hip_linrec_step(const SslaHipLinRec* d, void* stream) try {
    if (const int rc = check_linrec(d, kStep, "ssla_hip_linrec_step")) return rc;
    if (d->n_seqs == 0) return SSLA_OK;
    const LinRecArgs a = linrec_args(d, nullptr);
    // a thread 16 bytes of values, but where there are few
    if (!launchable((long long)a.n_seqs * ((a.channels - 1) / (d->dtype == SSLA_F32 ? 4 : 8) + 1) + kLinRecThreads, 1, 1, 1))
        return refuse("ssla_hip_linrec_step: too many sequences and channels");
    const hipError_t e = linrec_launch_step(a, d->dtype, (hipStream_t)stream);
    return e == hipSuccess ? SSLA_OK : hip_failed("ssla_hip_linrec_step", e);
} catch (const std::exception&) {
    return SSLA_ERR_HIP;
}

int ssla_hip_layer_norm(const SslaHipLayerNorm* d, void* stream) try {
    if (const int rc = check_layer_norm(d, false, "ssla_hip_layer_norm")) return rc;
    if (!d->rows || !d->channels) return SSLA_OK;
    const LayerNormArgs a = layer_norm_args(d, nullptr);
    if (!launchable(a.wgs, 1, 1, a.threads)) return refuse("ssla_hip_layer_norm: too many rows");
    const hipError_t e = layer_norm_launch(a, d->dtype, (hipStream_t)stream);
    return e == hipSuccess ? SSLA_OK : hip_failed("ssla_hip_layer_norm", e);
} catch (const std::exception&) {
    return SSLA_ERR_HIP;
}

int ssla_hip_layer_norm_backward_workspace(const SslaHipLayerNorm* d, const SslaHipLayerNormGrad* g,
                                           size_t* nbytes) try {
    const char* fn = "ssla_hip_layer_norm_backward_workspace";
    if (!nbytes) return refuse(std::string(fn) + ": null argument");
    *nbytes = 0;
    if (const int rc = check_layer_norm(d, true, fn)) return rc;
    if (const int rc = check_layer_norm_grad(d, g, fn)) return rc;
    *nbytes = layer_norm_bytes(layer_norm_args(d, g));
    return SSLA_OK;
} catch (const std::exception&) {
    return SSLA_ERR_ARG;
}

int ssla_hip_layer_norm_backward(const SslaHipLayerNorm* d, const SslaHipLayerNormGrad* g, void* workspace,
                                 size_t workspace_bytes, void* stream) try {
    const char* fn = "ssla_hip_layer_norm_backward";
    if (const int rc = check_layer_norm(d, true, fn)) return rc;
    if (const int rc = check_layer_norm_grad(d, g, fn)) return rc;
    if (!d->channels) return SSLA_OK;
    LayerNormArgs a = layer_norm_args(d, g);
    if (!layer_norm_fits(a)) return refuse(std::string(fn) + ": too many rows and channels");
    const size_t need = layer_norm_bytes(a);
    if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
        return refuse(std::string(fn) + ": the workspace is missing, too small or not 16-byte aligned");
    a.ws = (float*)workspace;
    const hipError_t e = layer_norm_launch_backward(a, d->dtype, (hipStream_t)stream);
    return e == hipSuccess ? SSLA_OK : hip_failed(fn, e);
} catch (const std::exception&) {
    return SSLA_ERR_HIP;
}

}  // extern "C"
