// ops_torch.cpp -- the sequence operators (include/ssla_hip.h) on torch tensors:
// the Python module ssla_hip._ops, which ssla_hip/ops.py presents.  Checks the
// tensors, fills the C ABI's descriptors, takes outputs and workspaces from
// torch's allocator and queues the call on torch's current stream.
//
// The same in Python over ctypes took 10 to 12.5 us a call, twice what the small
// calls take on the GPU; here one takes 5 to 6.
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <stdexcept>
#include <string>

#include "ssla_hip.h"

namespace {

PyObject* g_error = nullptr;     // ssla_hip.lib.SslaHipError

[[noreturn]] void refuse(const char* fn, const std::string& what) {
    throw std::invalid_argument(std::string(fn) + ": " + what);
}

struct LibraryError : std::runtime_error {
    using std::runtime_error::runtime_error;
};

void check(int rc, const char* entry) {
    if (rc < 0)
        throw LibraryError(std::string(entry) + " failed (" + std::to_string(rc) + "): " + ssla_hip_last_error());
}

// The arguments of a call, which ops.py passes by position.
struct Args {
    const char* fn;
    PyObject* const* v;

    const at::Tensor& tensor(int i, const char* name) const {
        if (!THPVariable_Check(v[i])) refuse(fn, std::string(name) + " must be a tensor");
        return THPVariable_Unpack(v[i]);
    }
    const at::Tensor* optional(int i, const char* name) const {
        return v[i] == Py_None ? nullptr : &tensor(i, name);
    }
    long long integer(int i, const char* name) const {
        const long long x = PyLong_AsLongLong(v[i]);
        if (x == -1 && PyErr_Occurred()) {
            PyErr_Clear();
            refuse(fn, std::string(name) + " must be an integer");
        }
        return x;
    }
    int count(int i, const char* name) const {
        const long long x = integer(i, name);
        if (x < 0 || x > 0x7fffffff) refuse(fn, std::string(name) + " must be 0 .. 2^31 - 1");
        return (int)x;
    }
    double real(int i, const char* name) const {
        const double x = PyFloat_AsDouble(v[i]);
        if (x == -1.0 && PyErr_Occurred()) {
            PyErr_Clear();
            refuse(fn, std::string(name) + " must be a number");
        }
        return x;
    }
};

int dtype_of(const char* fn, const char* name, const at::Tensor& t) {
    if (!t.is_cuda()) refuse(fn, std::string(name) + " must be on a GPU");
    switch (t.scalar_type()) {
        case at::kFloat: return SSLA_F32;
        case at::kBFloat16: return SSLA_BF16;
        case at::kHalf: return SSLA_F16;
        default: refuse(fn, std::string(name) + " must be float32, bfloat16 or float16");
    }
}

// Type and device of a tensor of the call; there are no gradients, backward or forward.
void alike(const char* fn, const char* name, const at::Tensor& t, at::ScalarType type, at::Device dev) {
    if (t.scalar_type() != type || t.device() != dev || t.layout() != at::kStrided)
        refuse(fn, std::string(name) + " must be a " + c10::toString(type) + " tensor on " + dev.str());
    if (t.is_neg()) refuse(fn, std::string(name) + " is a negated view: call resolve_neg()");
    if (t.requires_grad() && at::GradMode::is_enabled())
        refuse(fn, std::string(name) + " requires a gradient, which there is none of: call under torch.no_grad()");
    if (t._fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode())
        refuse(fn, std::string(name) + " carries a forward gradient, which there is none of: call with its primal");
}

// A call has written to t: autograd notices, should it have kept t.  Inference
// tensors have no version.
void written(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

void shaped(const char* fn, const char* name, const at::Tensor& t, at::IntArrayRef shape) {
    if (t.sizes() != shape)
        refuse(fn, std::string(name) + " must have the shape " + c10::str(shape) + ", not " + c10::str(t.sizes()));
}

// (tokens, heads, size) with the last dimension contiguous: strides of the others.
void rows(const char* fn, const char* name, const at::Tensor& t, at::ScalarType type, at::Device dev,
          at::IntArrayRef shape, long long* stride) {
    alike(fn, name, t, type, dev);
    shaped(fn, name, t, shape);
    if (t.stride(2) != 1 && shape[2] > 1) refuse(fn, std::string(name) + "'s last dimension must be contiguous");
    stride[0] = t.stride(0);
    stride[1] = t.stride(1);
}

// A pool of states (slots, heads, dk, dv): floats between slots.
long long pool(const char* fn, const char* name, const at::Tensor& t, at::Device dev, const SslaHipLinAttn& d) {
    alike(fn, name, t, at::kFloat, dev);
    if (t.dim() != 4) refuse(fn, std::string(name) + " must have the shape (slots, heads, dk, dv)");
    const int64_t want[4] = {t.size(0), d.heads, d.dk, d.dv};
    shaped(fn, name, t, want);
    const long long slot = (long long)d.heads * d.dk * d.dv;
    if ((t.stride(3) != 1 && d.dv > 1) || (t.stride(2) != d.dv && d.dk > 1) ||
        (t.stride(1) != (long long)d.dk * d.dv && d.heads > 1))
        refuse(fn, std::string(name) + ": a slot must be contiguous");
    if (t.size(0) > 0x7fffffff) refuse(fn, std::string(name) + " has too many slots");
    return t.size(0) > 1 ? t.stride(0) : slot;
}

const int* index(const char* fn, const char* name, const at::Tensor& t, at::Device dev, int64_t n) {
    alike(fn, name, t, at::kInt, dev);
    if (t.dim() != 1 || t.size(0) != n || (n > 1 && t.stride(0) != 1))
        refuse(fn, std::string(name) + " must be " + std::to_string(n) + " contiguous int32 values");
    return t.const_data_ptr<int>();
}

// q, k, v, log_decay and out of a call; out is made where there is none.
at::Tensor tokens(const char* fn, SslaHipLinAttn& d, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                  const at::Tensor& g, const at::Tensor* out) {
    d.dtype = dtype_of(fn, "q", q);
    if (q.dim() != 3 || v.dim() != 3) refuse(fn, "q, k and v must have the shape (tokens, heads, size)");
    const auto type = q.scalar_type();
    const auto dev = q.device();
    const int64_t n = q.size(0), qk_heads = q.size(1), dk = q.size(2), heads = v.size(1), dv = v.size(2);
    if (v.size(0) != n) refuse(fn, "q, k and v must have the same number of tokens");
    if (dk < 1 || dk > SSLA_LINATTN_MAX_DIM || dv < 1 || dv > SSLA_LINATTN_MAX_DIM)
        refuse(fn, "head sizes must be 1 .. " + std::to_string(SSLA_LINATTN_MAX_DIM));
    if (qk_heads < 1 || heads < 1 || heads % qk_heads || heads > 0x7fffffff)
        refuse(fn, "v's heads must be a multiple of q's and k's");
    rows(fn, "q", q, type, dev, q.sizes(), d.q_stride);
    rows(fn, "k", k, type, dev, q.sizes(), d.k_stride);
    rows(fn, "v", v, type, dev, v.sizes(), d.v_stride);
    alike(fn, "log_decay", g, at::kFloat, dev);
    if (g.dim() == 2 && g.size(0) == n && g.size(1) == heads) {
        d.decay_stride[0] = g.stride(0);
        d.decay_stride[1] = g.stride(1);
    } else if (g.dim() == 1 && g.size(0) == heads) {
        d.decay_stride[0] = 0;
        d.decay_stride[1] = g.stride(0);
    } else {
        refuse(fn, "log_decay must have the shape (heads,) or (tokens, heads)");
    }
    at::Tensor o = out ? *out : at::empty(v.sizes(), q.options().requires_grad(false));
    rows(fn, "out", o, type, dev, v.sizes(), d.out_stride);
    d.heads = (int)heads;
    d.qk_heads = (int)qk_heads;
    d.dk = (int)dk;
    d.dv = (int)dv;
    d.n_tokens = n;
    d.q = q.const_data_ptr();
    d.k = k.const_data_ptr();
    d.v = v.const_data_ptr();
    d.log_decay = g.const_data_ptr<float>();
    d.out = o.mutable_data_ptr();
    return o;
}

void* stream_of(at::Device dev) { return c10::hip::getCurrentHIPStream(dev.index()).stream(); }

at::Tensor workspace(at::Device dev, size_t bytes) {
    return bytes ? at::empty({(int64_t)bytes}, at::TensorOptions().dtype(at::kByte).device(dev)) : at::Tensor();
}

// linear_attention(q, k, v, log_decay, out, scale, cu_seqlens, max_len, n_seqs, state_in, state_out, slots)
at::Tensor linear_attention(const Args& a) {
    const char* fn = a.fn;
    const at::Tensor &q = a.tensor(0, "q"), &k = a.tensor(1, "k"), &v = a.tensor(2, "v"),
                     &g = a.tensor(3, "log_decay");
    SslaHipLinAttn d{};
    at::Tensor out = tokens(fn, d, q, k, v, g, a.optional(4, "out"));
    const auto dev = q.device();
    d.scale = (float)a.real(5, "scale");
    if (d.n_tokens > 0x7fffffff) refuse(fn, "too many tokens");
    const bool bounded = a.v[7] != Py_None;
    if (const at::Tensor* cu = a.optional(6, "cu_seqlens")) {
        if (cu->numel() < 1 || cu->numel() > 0x7fffffff) refuse(fn, "cu_seqlens must have at least one value");
        d.n_seqs = (int)cu->numel() - 1;
        d.cu_seqlens = index(fn, "cu_seqlens", *cu, dev, cu->numel());
        d.max_len = bounded ? a.count(7, "max_len") : (int)d.n_tokens;
    } else {
        d.n_seqs = a.count(8, "n_seqs");
        if ((d.n_tokens && !d.n_seqs) || (d.n_seqs && d.n_tokens % d.n_seqs))
            refuse(fn, std::to_string(d.n_tokens) + " tokens are not " + std::to_string(d.n_seqs) +
                           " sequences of the same length");
        d.max_len = d.n_seqs ? (int)(d.n_tokens / d.n_seqs) : 0;
        if (bounded && a.count(7, "max_len") != d.max_len) refuse(fn, "max_len goes with cu_seqlens");
    }
    d.n_slots = d.n_seqs;
    const at::Tensor *in = a.optional(9, "state_in"), *to = a.optional(10, "state_out");
    if (in) {
        d.state_stride = pool(fn, "state_in", *in, dev, d);
        d.n_slots = (int)in->size(0);
        d.state_in = in->const_data_ptr<float>();
    }
    if (to) {
        const long long s = pool(fn, "state_out", *to, dev, d);
        if (in && (to->size(0) != in->size(0) || s != d.state_stride))
            refuse(fn, "state_in and state_out must have the same layout");
        d.state_stride = s;
        d.n_slots = (int)to->size(0);
        d.state_out = to->mutable_data_ptr<float>();
    }
    if (const at::Tensor* slots = a.optional(11, "slots")) d.slots = index(fn, "slots", *slots, dev, d.n_seqs);
    else if (d.n_slots < d.n_seqs) refuse(fn, "there must be a state slot for every sequence");
    const c10::DeviceGuard guard(dev);
    size_t bytes = 0;
    check(ssla_hip_linattn_workspace(&d, &bytes), "ssla_hip_linattn_workspace");
    const at::Tensor ws = workspace(dev, bytes);
    check(ssla_hip_linattn(&d, bytes ? ws.data_ptr() : nullptr, bytes, stream_of(dev)), "ssla_hip_linattn");
    written(out);
    if (to) written(*to);
    return out;
}

// linear_attention_step(q, k, v, log_decay, state, out, scale, slots)
at::Tensor linear_attention_step(const Args& a) {
    const char* fn = a.fn;
    const at::Tensor &q = a.tensor(0, "q"), &k = a.tensor(1, "k"), &v = a.tensor(2, "v"),
                     &g = a.tensor(3, "log_decay"), &state = a.tensor(4, "state");
    SslaHipLinAttn d{};
    at::Tensor out = tokens(fn, d, q, k, v, g, a.optional(5, "out"));
    const auto dev = q.device();
    d.scale = (float)a.real(6, "scale");
    if (d.n_tokens > 0x7fffffff) refuse(fn, "too many sequences");
    d.n_seqs = (int)d.n_tokens;
    d.max_len = 1;
    d.state_stride = pool(fn, "state", state, dev, d);
    d.n_slots = (int)state.size(0);
    d.state_in = d.state_out = state.mutable_data_ptr<float>();
    if (const at::Tensor* slots = a.optional(7, "slots")) d.slots = index(fn, "slots", *slots, dev, d.n_seqs);
    else if (d.n_slots < d.n_seqs) refuse(fn, "there must be a state slot for every sequence");
    const c10::DeviceGuard guard(dev);
    check(ssla_hip_linattn_step(&d, stream_of(dev)), "ssla_hip_linattn_step");
    written(out);
    written(state);
    return out;
}

// Item and row stride of a channels-last tensor (n, ..., channels): the
// dimensions between must fold into rows at one stride.
void items(const char* fn, const char* name, const at::Tensor& t, const at::Tensor& like, long long* stride) {
    alike(fn, name, t, like.scalar_type(), like.device());
    shaped(fn, name, t, like.sizes());
    const int64_t n = t.dim(), c = t.size(n - 1);
    if (t.stride(n - 1) != 1 && c > 1) refuse(fn, std::string(name) + "'s channels must be contiguous");
    stride[0] = t.stride(0);
    stride[1] = c;
    bool first = true;
    int64_t want = 0;
    for (int64_t i = n - 2; i > 0; --i) {
        if (t.size(i) == 1) continue;
        if (first) stride[1] = t.stride(i);
        else if (t.stride(i) != want) refuse(fn, std::string(name) + "'s rows must lie at one stride");
        want = t.stride(i) * t.size(i);
        first = false;
    }
}

// group_norm(x, groups, weight, bias, out, eps, act, gate)
at::Tensor group_norm(const Args& a) {
    const char* fn = a.fn;
    const at::Tensor& x = a.tensor(0, "x");
    SslaHipGroupNorm d{};
    d.dtype = dtype_of(fn, "x", x);
    if (x.dim() < 2) refuse(fn, "x must have the shape (n, ..., channels)");
    const auto dev = x.device();
    const int64_t n = x.size(0), c = x.size(x.dim() - 1);
    int64_t between = 1;
    for (int64_t i = 1; i + 1 < x.dim(); ++i) between *= x.size(i);
    if (n > 0x7fffffff || c > 0x7fffffff || between > 0x7fffffff) refuse(fn, "x is too large");
    d.n = (int)n;
    d.rows = (int)between;
    d.channels = (int)c;
    d.groups = a.count(1, "groups");
    if (d.groups < 1 || c % d.groups) refuse(fn, "groups must divide channels");
    d.act = a.count(6, "act");
    d.eps = (float)a.real(5, "eps");
    const at::Tensor *w = a.optional(2, "weight"), *b = a.optional(3, "bias"), *gate = a.optional(7, "gate");
    auto vector = [&](const char* name, const at::Tensor* t) -> const void* {
        if (!t) return nullptr;
        alike(fn, name, *t, x.scalar_type(), dev);
        if (t->dim() != 1 || t->size(0) != c || (c > 1 && t->stride(0) != 1))
            refuse(fn, std::string(name) + " must be " + std::to_string(c) + " contiguous values");
        return t->const_data_ptr();
    };
    d.weight = vector("weight", w);
    d.bias = vector("bias", b);
    items(fn, "x", x, x, d.x_stride);
    if (gate) {
        items(fn, "gate", *gate, x, d.gate_stride);
        d.gate = gate->const_data_ptr();
    }
    const at::Tensor* given = a.optional(4, "out");
    at::Tensor out = given ? *given : at::empty(x.sizes(), x.options().requires_grad(false));
    items(fn, "out", out, x, d.out_stride);
    d.x = x.const_data_ptr();
    d.out = out.mutable_data_ptr();
    const c10::DeviceGuard guard(dev);
    size_t bytes = 0;
    check(ssla_hip_group_norm_workspace(&d, &bytes), "ssla_hip_group_norm_workspace");
    const at::Tensor ws = workspace(dev, bytes);
    check(ssla_hip_group_norm(&d, bytes ? ws.data_ptr() : nullptr, bytes, stream_of(dev)), "ssla_hip_group_norm");
    written(out);
    return out;
}

// C++ exceptions end here, as Python ones.
template <at::Tensor (*F)(const Args&)>
PyObject* call(const char* fn, int want, PyObject* const* v, Py_ssize_t n) {
    try {
        if (n != want) refuse(fn, "wrong number of arguments");
        return THPVariable_Wrap(F(Args{fn, v}));
    } catch (const std::invalid_argument& e) {
        PyErr_SetString(PyExc_ValueError, e.what());
    } catch (const LibraryError& e) {
        PyErr_SetString(g_error, e.what());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
    }
    return nullptr;
}

PyObject* py_linear_attention(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return call<linear_attention>("linear_attention", 12, v, n);
}
PyObject* py_linear_attention_step(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return call<linear_attention_step>("linear_attention_step", 8, v, n);
}
PyObject* py_group_norm(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return call<group_norm>("group_norm", 8, v, n);
}

PyMethodDef g_methods[] = {
    {"linear_attention", (PyCFunction)(void (*)())py_linear_attention, METH_FASTCALL, nullptr},
    {"linear_attention_step", (PyCFunction)(void (*)())py_linear_attention_step, METH_FASTCALL, nullptr},
    {"group_norm", (PyCFunction)(void (*)())py_group_norm, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_ops", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ops(void) {
    PyObject* lib = PyImport_ImportModule("ssla_hip.lib");
    if (!lib) return nullptr;
    g_error = PyObject_GetAttrString(lib, "SslaHipError");
    Py_DECREF(lib);
    return g_error ? PyModule_Create(&g_module) : nullptr;
}
