// ops_train_torch.cpp -- the operators that have gradients (include/ssla_hip.h)
// on torch tensors: the gated linear recurrence and layer norm, as functions of
// torch's autograd where it records one.  The functions are C++ ones: a call
// that records takes as long as one that does not, plus autograd's own node.
#include "ops_torch.h"

#include <c10/hip/HIPGraphsC10Utils.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/variable.h>

namespace ssla_torch {
namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// (rows, channels) with contiguous channels: the stride between rows.
long long matrix(const char* fn, const char* name, const at::Tensor& t, at::ScalarType type, at::Device dev,
                 at::IntArrayRef shape, bool backward) {
    alike(fn, name, t, type, dev, backward);
    shaped(fn, name, t, shape);
    if (t.stride(1) != 1 && shape[1] > 1) refuse(fn, std::string(name) + "'s channels must be contiguous");
    return shape[0] > 1 ? t.stride(0) : shape[1];
}

// (..., channels) with contiguous channels, whose other dimensions fold into rows.
long long folded(const char* fn, const char* name, const at::Tensor& t, at::ScalarType type, at::Device dev,
                 at::IntArrayRef shape, bool backward) {
    alike(fn, name, t, type, dev, backward);
    shaped(fn, name, t, shape);
    const int64_t n = t.dim(), c = shape[n - 1];
    if (t.stride(n - 1) != 1 && c > 1) refuse(fn, std::string(name) + "'s channels must be contiguous");
    if (t.numel() == 0) return c;
    int64_t stride = -1, want = 0;
    for (int64_t i = n - 2; i >= 0; --i) {
        if (t.size(i) == 1) continue;
        if (stride < 0) stride = t.stride(i);
        else if (t.stride(i) != want) refuse(fn, std::string(name) + "'s rows must lie at one stride");
        want = t.stride(i) * t.size(i);
    }
    return stride < 0 ? c : stride;
}

bool wanted(const at::Tensor* t) { return t && t->requires_grad(); }

// Autograd adds up a leaf's gradient on the stream that was current when the leaf
// was first recorded, for as long as any graph of it lives.  Where that is the default
// stream, which cannot be captured, a backward pass in a capture ends the process.
void capturable(const char* fn, const char* name, const at::Tensor* t) {
    if (!wanted(t) || !t->is_leaf()) return;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
    const auto on = node ? node->stream() : std::nullopt;
    if (on && on->id() == 0)
        refuse(fn, std::string(name) + " has a graph that was recorded on the default stream and still lives: "
                                       "drop it before the capture");
}
bool capturing(at::Device dev) {
    const c10::DeviceGuard guard(dev);
    return c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None;
}

// A gradient that autograd hands over, as the kernels take it.
at::Tensor usable(const at::Tensor& t) {
    if (!t.defined()) return t;
    const int64_t n = t.dim();
    at::Tensor r = t.is_neg() ? t.resolve_neg() : t;
    bool rows = r.layout() == at::kStrided && (r.size(n - 1) <= 1 || r.stride(n - 1) == 1);
    int64_t want = -1;
    for (int64_t i = n - 2; rows && i >= 0; --i) {
        if (r.size(i) == 1) continue;
        rows = want < 0 || r.stride(i) == want;
        want = r.stride(i) * r.size(i);
    }
    return rows ? r : r.contiguous();
}
long long row_stride(const at::Tensor& t) {
    for (int64_t i = t.dim() - 2; i >= 0; --i)
        if (t.size(i) != 1) return t.stride(i);
    return t.size(t.dim() - 1);
}

// Arguments of a function that may be absent.  Autograd counts the edges of those
// that are there only.
typedef std::optional<at::Tensor> Maybe;

Maybe maybe(const at::Tensor* t) { return t ? Maybe(*t) : Maybe(); }
const at::Tensor* some(const Maybe& t) { return t ? &*t : nullptr; }
const at::Tensor* some(const at::Tensor& t) { return t.defined() ? &t : nullptr; }
at::Tensor plain(const Maybe& t) { return t ? *t : at::Tensor(); }

void once(const char* fn) {
    if (at::GradMode::is_enabled())
        refuse(fn, "there are no second derivatives: call without create_graph");
}

// ---- gated linear recurrence ---------------------------------------------------------

// gate, v, q and cu_seqlens of a call.
void recurrence(const char* fn, SslaHipLinRec& d, const at::Tensor& gate, const at::Tensor& v, const at::Tensor* q,
                bool backward) {
    d.dtype = dtype_of(fn, "gate", gate);
    if (gate.dim() != 2) refuse(fn, "gate must have the shape (tokens, channels)");
    const auto type = gate.scalar_type();
    const auto dev = gate.device();
    const auto shape = gate.sizes();
    if (shape[0] > 0x7fffffff || shape[1] > 0x7fffffff) refuse(fn, "gate is too large");
    if (shape[1] < 1) refuse(fn, "there must be at least one channel");
    d.n_tokens = shape[0];
    d.channels = (int)shape[1];
    d.gate_stride = matrix(fn, "gate", gate, type, dev, shape, backward);
    d.v_stride = matrix(fn, "v", v, type, dev, shape, backward);
    d.gate = gate.const_data_ptr();
    d.v = v.const_data_ptr();
    if (q) {
        d.q_stride = matrix(fn, "q", *q, type, dev, shape, backward);
        d.q = q->const_data_ptr();
    }
}

// A pool of states (slots, channels): floats between slots.
long long states(const char* fn, const char* name, const at::Tensor& t, at::Device dev, const SslaHipLinRec& d,
                 bool backward) {
    if (t.dim() != 2) refuse(fn, std::string(name) + " must have the shape (slots, channels)");
    const int64_t want[2] = {t.size(0), d.channels};
    if (t.size(0) > 0x7fffffff) refuse(fn, std::string(name) + " has too many slots");
    return matrix(fn, name, t, at::kFloat, dev, want, backward);
}

at::Tensor new_rows(const at::Tensor& like, int64_t rows, at::ScalarType type) {
    return at::empty({rows, like.size(1)}, like.options().dtype(type).requires_grad(false));
}

void run(SslaHipLinRec& d, at::Device dev) {
    const c10::DeviceGuard guard(dev);
    size_t bytes = 0;
    check(ssla_hip_linrec_workspace(&d, &bytes), "ssla_hip_linrec_workspace");
    const at::Tensor ws = workspace(dev, bytes);
    check(ssla_hip_linrec(&d, bytes ? ws.data_ptr() : nullptr, bytes, stream_of(dev)), "ssla_hip_linrec");
}

struct Recurrence : torch::autograd::Function<Recurrence> {
    static constexpr const char* fn = "linear_recurrence";

    static SslaHipLinRec describe(const at::Tensor& gate, const at::Tensor& v, const at::Tensor& q,
                                  const at::Tensor& state_in, const at::Tensor& cu, int64_t n_seqs) {
        SslaHipLinRec d{};
        recurrence(fn, d, gate, v, q.defined() ? &q : nullptr, true);
        d.n_seqs = d.n_slots = (int)n_seqs;
        if (cu.defined()) d.cu_seqlens = cu.const_data_ptr<int>();
        if (state_in.defined()) {
            d.state_in_stride = states(fn, "state_in", state_in, gate.device(), d, true);
            d.state_in = state_in.const_data_ptr<float>();
        }
        return d;
    }

    static variable_list forward(AutogradContext* ctx, const at::Tensor& gate, const at::Tensor& v, const Maybe& maybe_q,
                                 const Maybe& maybe_in, const Maybe& maybe_cu, int64_t n_seqs, bool last) {
        const at::Tensor q = plain(maybe_q), state_in = plain(maybe_in), cu = plain(maybe_cu);
        SslaHipLinRec d = describe(gate, v, q, state_in, cu, n_seqs);
        const auto dev = gate.device();
        const at::Tensor out = new_rows(gate, d.n_tokens, gate.scalar_type());
        d.out = out.mutable_data_ptr();
        d.out_stride = d.channels;
        at::Tensor state;
        if (last) {
            state = new_rows(gate, n_seqs, at::kFloat);
            d.state_out = state.mutable_data_ptr<float>();
            d.state_out_stride = d.channels;
        }
        size_t bytes = 0;
        check(ssla_hip_linrec_carries(&d, &bytes), "ssla_hip_linrec_carries");
        const at::Tensor carries = workspace(dev, bytes);
        d.carries = bytes ? (float*)carries.data_ptr() : nullptr;
        run(d, dev);
        ctx->save_for_backward({gate, v, q, state_in, cu, carries});
        ctx->saved_data["n_seqs"] = n_seqs;
        ctx->set_materialize_grads(false);
        return last ? variable_list{out, state} : variable_list{out};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once(fn);
        const auto saved = ctx->get_saved_variables();
        const at::Tensor &gate = saved[0], &v = saved[1], &q = saved[2], &state_in = saved[3], &cu = saved[4],
                         &carries = saved[5];
        const int64_t n_seqs = ctx->saved_data["n_seqs"].toInt();
        SslaHipLinRec d = describe(gate, v, q, state_in, cu, n_seqs);
        const auto dev = gate.device();
        d.carries = carries.defined() ? (float*)carries.data_ptr() : nullptr;
        const at::Tensor dout = usable(grads[0]);
        const at::Tensor dstate = grads.size() > 1 ? usable(grads[1]) : at::Tensor();
        SslaHipLinRecGrad g{};
        if (dout.defined()) {
            g.dout = dout.const_data_ptr();
            g.dout_stride = row_stride(dout);
        }
        if (dstate.defined()) {
            g.dstate_out = dstate.const_data_ptr<float>();
            g.dstate_out_stride = row_stride(dstate);
        }
        variable_list out(7);
        int edge = 0;
        auto rows = [&](int i, void*& p, long long& stride) {
            if (!ctx->needs_input_grad(edge++)) return;
            out[i] = new_rows(gate, d.n_tokens, gate.scalar_type());
            p = out[i].mutable_data_ptr();
            stride = d.channels;
        };
        rows(0, g.dgate, g.dgate_stride);
        rows(1, g.dv, g.dv_stride);
        if (q.defined()) rows(2, g.dq, g.dq_stride);
        if (state_in.defined() && ctx->needs_input_grad(edge)) {
            out[3] = new_rows(gate, n_seqs, at::kFloat);
            g.dstate_in = out[3].mutable_data_ptr<float>();
            g.dstate_in_stride = d.channels;
        }
        const c10::DeviceGuard guard(dev);
        size_t bytes = 0;
        check(ssla_hip_linrec_workspace(&d, &bytes), "ssla_hip_linrec_workspace");
        const at::Tensor ws = workspace(dev, bytes);
        check(ssla_hip_linrec_backward(&d, &g, bytes ? ws.data_ptr() : nullptr, bytes, stream_of(dev)),
              "ssla_hip_linrec_backward");
        return out;
    }
};

// linear_recurrence(gate, v, q, out, cu_seqlens, n_seqs, state_in, state_out, slots, return_state)
std::vector<at::Tensor> linear_recurrence(const Args& a) {
    const char* fn = a.fn;
    const at::Tensor &gate = a.tensor(0, "gate"), &v = a.tensor(1, "v");
    const at::Tensor *q = a.optional(2, "q"), *given = a.optional(3, "out"), *cu = a.optional(4, "cu_seqlens"),
                     *in = a.optional(6, "state_in"), *to = a.optional(7, "state_out"), *slots = a.optional(8, "slots");
    const bool last = a.count(9, "return_state") != 0;
    const bool record = at::GradMode::is_enabled() && (wanted(&gate) || wanted(&v) || wanted(q) || wanted(in));
    SslaHipLinRec d{};
    recurrence(fn, d, gate, v, q, true);
    const auto dev = gate.device();
    const int64_t n = d.n_tokens;
    if (cu) {
        if (cu->numel() < 1 || cu->numel() > 0x7fffffff) refuse(fn, "cu_seqlens must have at least one value");
        d.n_seqs = (int)cu->numel() - 1;
        d.cu_seqlens = index(fn, "cu_seqlens", *cu, dev, cu->numel());
    } else {
        d.n_seqs = a.count(5, "n_seqs");
        if ((n && !d.n_seqs) || (d.n_seqs && n % d.n_seqs))
            refuse(fn, std::to_string(n) + " tokens are not " + std::to_string(d.n_seqs) + " sequences of the same length");
    }
    d.n_slots = d.n_seqs;
    if (in) {
        d.state_in_stride = states(fn, "state_in", *in, dev, d, true);
        d.n_slots = (int)in->size(0);
        d.state_in = in->const_data_ptr<float>();
    }
    if (last && (to || slots)) refuse(fn, "return_state gives every sequence's state: it goes without state_out and slots");
    if (record) {
        if (given || to || slots)
            refuse(fn, "out, state_out and slots have no gradients: call under torch.no_grad(), or with return_state");
        if (in && in->size(0) != d.n_seqs) refuse(fn, "state_in must have one row for every sequence");
        if (capturing(dev)) {
            capturable(fn, "gate", &gate);
            capturable(fn, "v", &v);
            capturable(fn, "q", q);
            capturable(fn, "state_in", in);
        }
        return Recurrence::apply(gate, v, maybe(q), maybe(in), maybe(cu), (int64_t)d.n_seqs, last);
    }
    if (to) {
        d.state_out_stride = states(fn, "state_out", *to, dev, d, false);
        if (in && to->size(0) != in->size(0)) refuse(fn, "state_in and state_out must have the same number of slots");
        d.n_slots = (int)to->size(0);
        d.state_out = to->mutable_data_ptr<float>();
    }
    if (slots) d.slots = index(fn, "slots", *slots, dev, d.n_seqs);
    else if (d.n_slots < d.n_seqs) refuse(fn, "there must be a state slot for every sequence");
    const at::Tensor out = given ? *given : new_rows(gate, n, gate.scalar_type());
    d.out_stride = matrix(fn, "out", out, gate.scalar_type(), dev, gate.sizes(), false);
    d.out = out.mutable_data_ptr();
    std::vector<at::Tensor> got{out};
    if (last) {
        got.push_back(new_rows(gate, d.n_seqs, at::kFloat));
        d.state_out = got[1].mutable_data_ptr<float>();
        d.state_out_stride = d.channels;
        d.n_slots = d.n_seqs;
    }
    run(d, dev);
    written(out);
    if (to) written(*to);
    return got;
}

// linear_recurrence_step(gate, v, state, q, out, slots)
at::Tensor linear_recurrence_step(const Args& a) {
    const char* fn = a.fn;
    const at::Tensor &gate = a.tensor(0, "gate"), &v = a.tensor(1, "v"), &state = a.tensor(2, "state");
    const at::Tensor *q = a.optional(3, "q"), *given = a.optional(4, "out"), *slots = a.optional(5, "slots");
    SslaHipLinRec d{};
    recurrence(fn, d, gate, v, q, false);
    const auto dev = gate.device();
    d.n_seqs = (int)d.n_tokens;
    d.state_in_stride = d.state_out_stride = states(fn, "state", state, dev, d, false);
    d.n_slots = (int)state.size(0);
    d.state_in = d.state_out = state.mutable_data_ptr<float>();
    if (slots) d.slots = index(fn, "slots", *slots, dev, d.n_seqs);
    else if (d.n_slots < d.n_seqs) refuse(fn, "there must be a state slot for every sequence");
    const at::Tensor out = given ? *given : new_rows(gate, d.n_tokens, gate.scalar_type());
    d.out_stride = matrix(fn, "out", out, gate.scalar_type(), dev, gate.sizes(), false);
    d.out = out.mutable_data_ptr();
    const c10::DeviceGuard guard(dev);
    check(ssla_hip_linrec_step(&d, stream_of(dev)), "ssla_hip_linrec_step");
    written(out);
    written(state);
    return out;
}

// ---- layer norm ------------------------------------------------------------------------

SslaHipLayerNorm describe_norm(const char* fn, const at::Tensor& x, const at::Tensor* res, const at::Tensor* w,
                               const at::Tensor* b, double eps) {
    SslaHipLayerNorm d{};
    d.dtype = dtype_of(fn, "x", x);
    if (x.dim() < 1) refuse(fn, "x must have the shape (..., channels)");
    const auto dev = x.device();
    const int64_t c = x.size(x.dim() - 1);
    int64_t rows = 1;
    for (int64_t i = 0; i + 1 < x.dim(); ++i) rows *= x.size(i);
    if (c > 0x7fffffff || rows > 0x7fffffff) refuse(fn, "x is too large");
    d.rows = (int)rows;
    d.channels = (int)c;
    d.eps = (float)eps;
    d.x_stride = folded(fn, "x", x, x.scalar_type(), dev, x.sizes(), true);
    d.x = x.const_data_ptr();
    if (res) {
        d.residual_stride = folded(fn, "residual", *res, x.scalar_type(), dev, x.sizes(), true);
        d.residual = res->const_data_ptr();
    }
    const auto wt = w ? w->scalar_type() : b ? b->scalar_type() : x.scalar_type();
    if (wt != x.scalar_type() && wt != at::kFloat) refuse(fn, "weight and bias must be of x's type or float32");
    auto vector = [&](const char* name, const at::Tensor* t) -> const void* {
        if (!t) return nullptr;
        alike(fn, name, *t, wt, dev, true);
        if (t->dim() != 1 || t->size(0) != c || (c > 1 && t->stride(0) != 1))
            refuse(fn, std::string(name) + " must be " + std::to_string(c) + " contiguous values");
        return t->const_data_ptr();
    };
    d.weight = vector("weight", w);
    d.bias = vector("bias", b);
    d.weight_dtype = wt == at::kFloat ? SSLA_F32 : d.dtype;
    return d;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static constexpr const char* fn = "layer_norm";

    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const Maybe& res, const Maybe& w,
                              const Maybe& b, double eps) {
        SslaHipLayerNorm d = describe_norm(fn, x, some(res), some(w), some(b), eps);
        const auto dev = x.device();
        const at::Tensor out = at::empty(x.sizes(), x.options().requires_grad(false));
        d.out = out.mutable_data_ptr();
        d.out_stride = d.channels;
        const c10::DeviceGuard guard(dev);
        const at::Tensor stats = at::empty({(int64_t)d.rows * 3}, x.options().dtype(at::kFloat).requires_grad(false));
        d.stats = stats.mutable_data_ptr<float>();
        check(ssla_hip_layer_norm(&d, stream_of(dev)), "ssla_hip_layer_norm");
        // of the bias only its type is needed
        ctx->save_for_backward({x, plain(res), plain(w), stats});
        ctx->saved_data["bias"] = b.has_value();
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["wide"] = d.weight_dtype == SSLA_F32;
        ctx->set_materialize_grads(false);
        return out;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once(fn);
        variable_list out(5);
        if (!grads[0].defined()) return out;
        const auto saved = ctx->get_saved_variables();
        const at::Tensor &x = saved[0], &res = saved[1], &w = saved[2], &stats = saved[3];
        SslaHipLayerNorm d = describe_norm(fn, x, some(res), some(w), nullptr, ctx->saved_data["eps"].toDouble());
        const auto dev = x.device();
        const bool wide = ctx->saved_data["wide"].toBool();
        d.weight_dtype = wide ? SSLA_F32 : d.dtype;
        d.stats = stats.mutable_data_ptr<float>();
        const at::Tensor dout = usable(grads[0]);
        SslaHipLayerNormGrad g{};
        g.dout = dout.const_data_ptr();
        g.dout_stride = row_stride(dout);
        const auto options = x.options().requires_grad(false);
        int edge = 0;
        const bool of_x = ctx->needs_input_grad(edge++), of_res = res.defined() && ctx->needs_input_grad(edge++);
        if (of_x || of_res) {
            const at::Tensor dx = at::empty(x.sizes(), options);
            g.dx = dx.mutable_data_ptr();
            g.dx_stride = d.channels;
            if (of_x) out[0] = dx;
            if (of_res) out[1] = dx;
        }
        auto vector = [&](int i, bool there, void*& p) {
            if (!there || !ctx->needs_input_grad(edge++)) return;
            out[i] = at::empty({(int64_t)d.channels}, wide ? options.dtype(at::kFloat) : options);
            p = out[i].mutable_data_ptr();
        };
        vector(2, w.defined(), g.dweight);
        vector(3, ctx->saved_data["bias"].toBool(), g.dbias);
        const c10::DeviceGuard guard(dev);
        size_t bytes = 0;
        check(ssla_hip_layer_norm_backward_workspace(&d, &g, &bytes), "ssla_hip_layer_norm_backward_workspace");
        const at::Tensor ws = workspace(dev, bytes);
        check(ssla_hip_layer_norm_backward(&d, &g, bytes ? ws.data_ptr() : nullptr, bytes, stream_of(dev)),
              "ssla_hip_layer_norm_backward");
        return out;
    }
};

// layer_norm(x, weight, bias, out, eps, residual)
at::Tensor layer_norm(const Args& a) {
    const char* fn = a.fn;
    const at::Tensor& x = a.tensor(0, "x");
    const at::Tensor *w = a.optional(1, "weight"), *b = a.optional(2, "bias"), *given = a.optional(3, "out"),
                     *res = a.optional(5, "residual");
    const double eps = a.real(4, "eps");
    SslaHipLayerNorm d = describe_norm(fn, x, res, w, b, eps);
    if (at::GradMode::is_enabled() && (wanted(&x) || wanted(res) || wanted(w) || wanted(b))) {
        if (given) refuse(fn, "out has no gradient: call under torch.no_grad()");
        if (capturing(x.device())) {
            capturable(fn, "x", &x);
            capturable(fn, "residual", res);
            capturable(fn, "weight", w);
            capturable(fn, "bias", b);
        }
        return LayerNorm::apply(x, maybe(res), maybe(w), maybe(b), eps);
    }
    const auto dev = x.device();
    const at::Tensor out = given ? *given : at::empty(x.sizes(), x.options().requires_grad(false));
    d.out_stride = folded(fn, "out", out, x.scalar_type(), dev, x.sizes(), false);
    d.out = out.mutable_data_ptr();
    const c10::DeviceGuard guard(dev);
    check(ssla_hip_layer_norm(&d, stream_of(dev)), "ssla_hip_layer_norm");
    written(out);
    return out;
}

}  // namespace

PyObject* py_linear_recurrence(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return call<linear_recurrence>("linear_recurrence", 10, v, n);
}
PyObject* py_linear_recurrence_step(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return call<linear_recurrence_step>("linear_recurrence_step", 6, v, n);
}
PyObject* py_layer_norm(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return call<layer_norm>("layer_norm", 6, v, n);
}

}  // namespace ssla_torch
