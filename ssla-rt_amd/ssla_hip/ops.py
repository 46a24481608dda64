"""Sequence operators of libssla_hip.so on torch device tensors.

  linear_attention       whole sequences (packed, ragged), states in and out
  linear_attention_step  one token of every sequence, states updated in a pool
  group_norm             group norm with an activation, channels last

The formulas, layouts and limits are those of include/ssla_hip.h (sequence
operators).  Calls are queued on torch's current stream of the tensors'
device, which need not be the current device; outputs and workspaces come
from torch's allocator, so calls can be captured into a graph.  There is no
fallback: without the library, or for tensors off the GPU, a call raises.
"""
from __future__ import annotations

import ctypes
import struct
from typing import Optional

import torch

from . import abi, lib

_DTYPES = {torch.float32: abi.SSLA_F32, torch.bfloat16: abi.SSLA_BF16, torch.float16: abi.SSLA_F16}
_ACTS = {"none": abi.SSLA_ACT_NONE, None: abi.SSLA_ACT_NONE, "silu": abi.SSLA_ACT_SILU,
         "sigmoid": abi.SSLA_ACT_SIGMOID, "relu": abi.SSLA_ACT_RELU}

# the descriptors' fields in order, in native alignment (abi.SslaHipLinAttn, SslaHipGroupNorm);
# a call packs one in about a microsecond, where filling the ctypes form takes five
_LINATTN = struct.Struct("@8i q 5P 10q 4P q f 0q")
_NORM = struct.Struct("@6i 5P 6q f 0q")
assert _LINATTN.size == ctypes.sizeof(abi.SslaHipLinAttn)
assert _NORM.size == ctypes.sizeof(abi.SslaHipGroupNorm)


_raw_stream = torch._C._cuda_getCurrentRawStream      # current_stream(...).cuda_stream in 0.1 us, not 2
_size_t = ctypes.c_size_t
_L = None


def _bad(fn: str, what: str):
    raise ValueError(f"{fn}: {what}")


def _call(entry: str, dev: int, desc: bytes, workspace: Optional[str] = None) -> None:
    """One library call on device `dev` and torch's current stream there."""
    global _L
    if _L is None:
        _L = lib.load()
    if torch.cuda.current_device() != dev:
        with torch.cuda.device(dev):
            return _call(entry, dev, desc, workspace)
    if workspace is None:
        rc = getattr(_L, entry)(desc, _raw_stream(dev))
    else:
        n = _size_t()
        rc = getattr(_L, workspace)(desc, ctypes.byref(n))
        if rc == 0:
            n = n.value
            ws = torch.empty(n, dtype=torch.uint8, device=dev).data_ptr() if n else None
            rc = getattr(_L, entry)(desc, ws, n, _raw_stream(dev))
    if rc:
        lib.check(rc, entry)


def _check_rows(fn, name, t, dtype, dev, shape):
    """Why t is no (tokens, heads, size) tensor of the call, if it is none."""
    if t.dtype != dtype or t.get_device() != dev:
        _bad(fn, f"{name} must be a {dtype} tensor on cuda:{dev}")
    if t.shape != shape:
        _bad(fn, f"{name} must have the shape {tuple(shape)}, not {tuple(t.shape)}")
    if t.stride(2) != 1 and shape[2] > 1:
        _bad(fn, f"{name}'s last dimension must be contiguous")


def _pool(fn, name, t, dev, heads, dk, dv):
    """Floats between the slots of a pool of states."""
    if t.dtype != torch.float32 or t.get_device() != dev:
        _bad(fn, f"{name} must be a float32 tensor on cuda:{dev}")
    if t.dim() != 4 or t.shape[1:] != (heads, dk, dv):
        _bad(fn, f"{name} must have the shape (slots, {heads}, {dk}, {dv}), not {tuple(t.shape)}")
    slot = heads * dk * dv
    if t.is_contiguous():
        return slot
    s, h, d, e = t.stride()
    if (e != 1 and dv > 1) or (d != dv and dk > 1) or (h != dk * dv and heads > 1):
        _bad(fn, f"{name}: a slot must be contiguous")
    return s if t.shape[0] > 1 else slot


def _index(fn, name, t, dev, n):
    if t.dtype != torch.int32 or t.get_device() != dev or t.shape != (n,):
        _bad(fn, f"{name} must be {n} int32 values on cuda:{dev}")
    if n > 1 and t.stride(0) != 1:
        _bad(fn, f"{name} must be contiguous")
    return t.data_ptr()


def _linattn(fn, dev, q, k, v, log_decay, out, scale, n_seqs, max_len, cu, slots, state_in, state_out):
    dtype, qshape, vshape = q.dtype, q.shape, v.shape
    if dev < 0 or dtype not in _DTYPES:
        _bad(fn, "q must be a float32, bfloat16 or float16 tensor on a GPU")
    if len(qshape) != 3 or len(vshape) != 3:
        _bad(fn, "q, k and v must have the shape (tokens, heads, size)")
    tokens, qk_heads, dk = qshape
    t, heads, dv = vshape
    if t != tokens:
        _bad(fn, "q, k and v must have the same number of tokens")
    if not (0 < dk <= abi.LINATTN_MAX_DIM and 0 < dv <= abi.LINATTN_MAX_DIM):
        _bad(fn, f"head sizes must be 1 .. {abi.LINATTN_MAX_DIM}")
    if qk_heads < 1 or heads < 1 or heads % qk_heads:
        _bad(fn, "v's heads must be a multiple of q's and k's")
    _check_rows(fn, "q", q, dtype, dev, qshape)
    _check_rows(fn, "k", k, dtype, dev, qshape)
    _check_rows(fn, "v", v, dtype, dev, vshape)
    if log_decay.dtype != torch.float32 or log_decay.get_device() != dev:
        _bad(fn, f"log_decay must be a float32 tensor on cuda:{dev}")
    if log_decay.shape == (tokens, heads):
        g0, g1 = log_decay.stride()
    elif log_decay.shape == (heads,):
        g0, g1 = 0, log_decay.stride(0)
    else:
        _bad(fn, f"log_decay must have the shape ({heads},) or ({tokens}, {heads})")
    if out is None:
        out = q.new_empty(vshape)
    else:
        _check_rows(fn, "out", out, dtype, dev, vshape)
    stride, n_slots, p_in, p_out = heads * dk * dv, n_seqs, 0, 0
    if state_in is not None:
        stride, n_slots = _pool(fn, "state_in", state_in, dev, heads, dk, dv), state_in.shape[0]
        p_in = state_in.data_ptr()
    if state_out is state_in:
        p_out = p_in
    elif state_out is not None:
        s = _pool(fn, "state_out", state_out, dev, heads, dk, dv)
        if state_in is not None and (state_out.shape[0] != n_slots or s != stride):
            _bad(fn, "state_in and state_out must have the same layout")
        stride, n_slots, p_out = s, state_out.shape[0], state_out.data_ptr()
    if slots is not None:
        slots = _index(fn, "slots", slots, dev, n_seqs)
    elif n_slots < n_seqs:
        _bad(fn, f"{n_seqs} sequences need as many state slots, not {n_slots}")
    q0, q1, _ = q.stride()
    k0, k1, _ = k.stride()
    v0, v1, _ = v.stride()
    o0, o1, _ = out.stride()
    return out, _LINATTN.pack(
        _DTYPES[dtype], heads, qk_heads, dk, dv, n_seqs, max_len, n_slots, tokens,
        q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), out.data_ptr(),
        q0, q1, k0, k1, v0, v1, g0, g1, o0, o1, cu, slots or 0, p_in, p_out, stride, scale)


def linear_attention(q, k, v, log_decay, out=None, *, scale: float = 1.0, cu_seqlens=None,
                     max_len: Optional[int] = None, n_seqs: int = 1, state_in=None,
                     state_out=None, slots=None) -> torch.Tensor:
    """S_t = exp(log_decay_t) S_{t-1} + k_t v_t^T, out_t = scale q_t^T S_t over
    packed sequences.

    q, k        (tokens, qk_heads, dk), v (tokens, heads, dv): any strides with
                the last dimension contiguous; qk_heads divides heads
    log_decay   float32 (tokens, heads), or (heads,): one for each head
    cu_seqlens  int32 (sequences + 1,) on the device: the sequences' first
                tokens and the last one's end; max_len bounds their lengths
                (default: all tokens; a tight bound spares work).  None:
                n_seqs sequences of the same length
    state_in, state_out  float32 (slots, heads, dk, dv) pools, read from
                (None: zeros) and written to; may be the same
    slots       int32 (sequences,) slots of the sequences, each its own (None:
                slot s for sequence s); a sequence with a negative slot is
                passed over
    Returns out (tokens, heads, dv) in q's type; rows of no sequence are left
    as they are (uninitialised where out is made here)."""
    fn, cu, dev = "linear_attention", 0, q.get_device()
    tokens = q.shape[0]
    if cu_seqlens is not None:
        n_seqs = cu_seqlens.numel() - 1
        if n_seqs < 0:
            _bad(fn, "cu_seqlens must have at least one value")
        cu = _index(fn, "cu_seqlens", cu_seqlens, dev, n_seqs + 1)
        max_len = tokens if max_len is None else max_len
    else:
        if n_seqs < 0 or (tokens and not n_seqs) or (n_seqs and tokens % n_seqs):
            _bad(fn, f"{tokens} tokens are not {n_seqs} sequences of the same length")
        if max_len is not None and n_seqs and max_len != tokens // n_seqs:
            _bad(fn, "max_len goes with cu_seqlens")
        max_len = tokens // n_seqs if n_seqs else 0
    out, desc = _linattn(fn, dev, q, k, v, log_decay, out, scale, n_seqs, max_len, cu, slots,
                         state_in, state_out)
    _call("ssla_hip_linattn", dev, desc, "ssla_hip_linattn_workspace")
    return out


def linear_attention_step(q, k, v, log_decay, state, out=None, *, scale: float = 1.0,
                          slots=None) -> torch.Tensor:
    """One token of every sequence: row s of q, k (sequences, qk_heads, dk),
    v (sequences, heads, dv) and log_decay ((sequences, heads), or (heads,))
    belongs to sequence s.  Its state, slot slots[s] (None: s) of `state`
    (float32 (slots, heads, dk, dv)), is updated in place; out[s] is read from
    the new one.  A row with a negative slot is passed over.  Returns out."""
    fn, dev = "linear_attention_step", q.get_device()
    out, desc = _linattn(fn, dev, q, k, v, log_decay, out, scale, q.shape[0], 1, 0, slots, state,
                         state)
    _call("ssla_hip_linattn_step", dev, desc)
    return out


def _items(fn, name, t, like):
    """(item stride, row stride) of a channels-last tensor (n, ..., channels)."""
    if t.dtype != like.dtype or t.get_device() != like.get_device() or t.shape != like.shape:
        _bad(fn, f"{name} must have x's shape, type and device")
    st, sh = t.stride(), t.shape
    if st[-1] != 1 and sh[-1] > 1:
        _bad(fn, f"{name}'s channels must be contiguous")
    if len(sh) == 2:
        return st[0], sh[1]
    if len(sh) == 3:
        return st[0], st[1] if sh[1] > 1 else sh[2]
    row, want = None, None
    for i in range(len(sh) - 2, 0, -1):          # the dimensions between must fold into one
        if sh[i] == 1:
            continue
        if row is None:
            row, want = st[i], st[i] * sh[i]
        elif st[i] != want:
            _bad(fn, f"{name}'s rows must lie at one stride")
        else:
            want *= sh[i]
    return st[0], sh[-1] if row is None else row


def group_norm(x, groups: int, weight=None, bias=None, out=None, *, eps: float = 1e-5,
               act: Optional[str] = None, gate=None) -> torch.Tensor:
    """Group norm of x (n, ..., channels), channels last, over the dimensions
    between and the channels / groups neighbouring channels of a group; then
    act ("none", "silu", "sigmoid", "relu") of it, or, with `gate` (of x's
    shape), the norm times act(gate).  (tokens, channels) normalises each
    token's groups by themselves, as behind an attention's heads.  weight, bias
    (channels,) in x's type.  out may be x.  Returns out (x's shape and type)."""
    fn, dev, dtype, shape = "group_norm", x.get_device(), x.dtype, x.shape
    if len(shape) < 2 or dev < 0 or dtype not in _DTYPES:
        _bad(fn, "x must be a float32, bfloat16 or float16 tensor (n, ..., channels) on a GPU")
    if act not in _ACTS:
        _bad(fn, f"act must be one of {[a for a in _ACTS if a]}")
    n, c = shape[0], shape[-1]
    if groups < 1 or c % groups:
        _bad(fn, "groups must divide channels")
    pw = pb = pg = 0
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            if t.dtype != dtype or t.get_device() != dev or t.shape != (c,) or (c > 1 and t.stride(0) != 1):
                _bad(fn, f"{name} must be {c} contiguous values of x's type and device")
            if name == "weight":
                pw = t.data_ptr()
            else:
                pb = t.data_ptr()
    if out is None:
        out = x.new_empty(shape)
    rows = 1
    for s in shape[1:-1]:
        rows *= s
    if n == 0 or rows == 0 or c == 0:
        return out
    (xn, xr), (on, orow), (gn, gr) = _items(fn, "x", x, x), _items(fn, "out", out, x), (0, 0)
    if gate is not None:
        gn, gr = _items(fn, "gate", gate, x)
        pg = gate.data_ptr()
    desc = _NORM.pack(_DTYPES[dtype], n, rows, c, groups, _ACTS[act], x.data_ptr(), pg, pw, pb,
                      out.data_ptr(), xn, xr, gn, gr, on, orow, eps)
    _call("ssla_hip_group_norm", dev, desc, "ssla_hip_group_norm_workspace")
    return out
