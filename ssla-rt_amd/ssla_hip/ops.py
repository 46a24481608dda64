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


def _bad(fn: str, what: str):
    raise ValueError(f"{fn}: {what}")


def _call(fn: str, dev: torch.device, desc: bytes, workspace_of=None) -> None:
    L = lib.load()
    if torch.cuda.current_device() != dev.index:
        with torch.cuda.device(dev):
            return _call(fn, dev, desc, workspace_of)
    stream = torch.cuda.current_stream(dev).cuda_stream
    if workspace_of is None:
        lib.check(getattr(L, fn)(desc, stream), fn)
        return
    n = ctypes.c_size_t()
    lib.check(workspace_of(L)(desc, ctypes.byref(n)), fn)
    ws = torch.empty(n.value, dtype=torch.uint8, device=dev) if n.value else None
    lib.check(getattr(L, fn)(desc, ws.data_ptr() if ws is not None else None, n.value, stream), fn)


def _rows(fn, name, t, dtype, dev, heads, width):
    if t.dtype != dtype or t.device != dev:
        _bad(fn, f"{name} must be a {dtype} tensor on {dev}")
    if t.dim() != 3 or t.shape[1] != heads or t.shape[2] != width:
        _bad(fn, f"{name} must have the shape (tokens, {heads}, {width}), not {tuple(t.shape)}")
    s0, s1, s2 = t.stride()
    if s2 != 1 and width > 1:
        _bad(fn, f"{name}'s last dimension must be contiguous")
    return s0, s1


def _pool(fn, name, t, dev, heads, dk, dv):
    if t.dtype != torch.float32 or t.device != dev:
        _bad(fn, f"{name} must be a float32 tensor on {dev}")
    if t.dim() != 4 or tuple(t.shape[1:]) != (heads, dk, dv):
        _bad(fn, f"{name} must have the shape (slots, {heads}, {dk}, {dv}), not {tuple(t.shape)}")
    if t.shape[0] and not t[0].is_contiguous():
        _bad(fn, f"{name}: a slot must be contiguous")
    return t.stride(0) if t.shape[0] > 1 else heads * dk * dv


def _index(fn, name, t, dev, n):
    if t.dtype != torch.int32 or t.device != dev or t.dim() != 1 or t.shape[0] != n:
        _bad(fn, f"{name} must be {n} int32 values on {dev}")
    if not t.is_contiguous():
        _bad(fn, f"{name} must be contiguous")
    return t.data_ptr()


def _linattn(fn, q, k, v, log_decay, out, scale, n_seqs, max_len, cu, slots, state_in, state_out):
    if q.dim() != 3 or v.dim() != 3:
        _bad(fn, "q, k and v must have the shape (tokens, heads, size)")
    dtype, dev = q.dtype, q.device
    if dev.type != "cuda" or dtype not in _DTYPES:
        _bad(fn, "q must be a float32, bfloat16 or float16 tensor on a GPU")
    tokens, qk_heads, dk = q.shape
    heads, dv = v.shape[1], v.shape[2]
    if not (0 < dk <= abi.LINATTN_MAX_DIM and 0 < dv <= abi.LINATTN_MAX_DIM):
        _bad(fn, f"head sizes must be 1 .. {abi.LINATTN_MAX_DIM}")
    if qk_heads < 1 or heads < 1 or heads % qk_heads:
        _bad(fn, "v's heads must be a multiple of q's and k's")
    if k.shape[0] != tokens or v.shape[0] != tokens:
        _bad(fn, "q, k and v must have the same number of tokens")
    qs = _rows(fn, "q", q, dtype, dev, qk_heads, dk)
    ks = _rows(fn, "k", k, dtype, dev, qk_heads, dk)
    vs = _rows(fn, "v", v, dtype, dev, heads, dv)
    if log_decay.dtype != torch.float32 or log_decay.device != dev:
        _bad(fn, f"log_decay must be a float32 tensor on {dev}")
    if log_decay.shape == (tokens, heads) and log_decay.dim() == 2:
        gs = log_decay.stride()
    elif log_decay.dim() == 1 and log_decay.shape[0] == heads:
        gs = (0, log_decay.stride(0))
    else:
        _bad(fn, f"log_decay must have the shape ({heads},) or ({tokens}, {heads})")
    if out is None:
        out = torch.empty((tokens, heads, dv), dtype=dtype, device=dev)
    elif out.shape[0] != tokens:
        _bad(fn, "out must have as many tokens as q")
    os = _rows(fn, "out", out, dtype, dev, heads, dv)
    stride = heads * dk * dv
    n_slots = n_seqs
    if state_in is not None:
        stride = _pool(fn, "state_in", state_in, dev, heads, dk, dv)
        n_slots = state_in.shape[0]
    if state_out is not None:
        s = _pool(fn, "state_out", state_out, dev, heads, dk, dv)
        if state_in is not None and (state_out.shape[0] != n_slots or s != stride):
            _bad(fn, "state_in and state_out must have the same layout")
        stride, n_slots = s, state_out.shape[0]
    if slots is None and n_slots < n_seqs:
        _bad(fn, f"{n_seqs} sequences need as many state slots, not {n_slots}")
    return out, _LINATTN.pack(
        _DTYPES[dtype], heads, qk_heads, dk, dv, n_seqs, max_len, n_slots, tokens,
        q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), out.data_ptr(),
        *qs, *ks, *vs, *gs, *os, cu,
        _index(fn, "slots", slots, dev, n_seqs) if slots is not None else 0,
        state_in.data_ptr() if state_in is not None else 0,
        state_out.data_ptr() if state_out is not None else 0, stride, scale)


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
    fn, cu = "linear_attention", 0
    tokens = q.shape[0]
    if cu_seqlens is not None:
        n_seqs = cu_seqlens.numel() - 1
        if n_seqs < 0:
            _bad(fn, "cu_seqlens must have at least one value")
        cu = _index(fn, "cu_seqlens", cu_seqlens, q.device, n_seqs + 1)
        max_len = tokens if max_len is None else max_len
    else:
        if n_seqs < 0 or (tokens and not n_seqs) or (n_seqs and tokens % n_seqs):
            _bad(fn, f"{tokens} tokens are not {n_seqs} sequences of the same length")
        if max_len is not None and n_seqs and max_len != tokens // n_seqs:
            _bad(fn, "max_len goes with cu_seqlens")
        max_len = tokens // n_seqs if n_seqs else 0
    out, desc = _linattn(fn, q, k, v, log_decay, out, scale, n_seqs, max_len, cu, slots, state_in,
                         state_out)
    _call("ssla_hip_linattn", q.device, desc, lambda L: L.ssla_hip_linattn_workspace)
    return out


def linear_attention_step(q, k, v, log_decay, state, out=None, *, scale: float = 1.0,
                          slots=None) -> torch.Tensor:
    """One token of every sequence: row s of q, k (sequences, qk_heads, dk),
    v (sequences, heads, dv) and log_decay ((sequences, heads), or (heads,))
    belongs to sequence s.  Its state, slot slots[s] (None: s) of `state`
    (float32 (slots, heads, dk, dv)), is updated in place; out[s] is read from
    the new one.  A row with a negative slot is passed over.  Returns out."""
    fn = "linear_attention_step"
    out, desc = _linattn(fn, q, k, v, log_decay, out, scale, q.shape[0], 1, 0, slots, state, state)
    _call("ssla_hip_linattn_step", q.device, desc)
    return out


def _items(fn, name, t, like):
    """(item stride, row stride) of a channels-last tensor (n, ..., channels)."""
    if t.dtype != like.dtype or t.device != like.device or t.shape != like.shape:
        _bad(fn, f"{name} must have x's shape, type and device")
    st, sh = t.stride(), t.shape
    if st[-1] != 1 and sh[-1] > 1:
        _bad(fn, f"{name}'s channels must be contiguous")
    if t.dim() == 2:
        return st[0], sh[1]
    row, want = None, None
    for i in range(t.dim() - 2, 0, -1):          # the dimensions between must fold into one
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
    fn = "group_norm"
    if x.dim() < 2 or x.device.type != "cuda" or x.dtype not in _DTYPES:
        _bad(fn, "x must be a float32, bfloat16 or float16 tensor (n, ..., channels) on a GPU")
    if act not in _ACTS:
        _bad(fn, f"act must be one of {[a for a in _ACTS if a]}")
    n, c = x.shape[0], x.shape[-1]
    if groups < 1 or c % groups:
        _bad(fn, "groups must divide channels")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and (t.dtype != x.dtype or t.device != x.device or tuple(t.shape) != (c,)
                              or (c > 1 and t.stride(0) != 1)):
            _bad(fn, f"{name} must be {c} contiguous values of x's type and device")
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    rows = 1
    for s in x.shape[1:-1]:
        rows *= s
    if x.numel() == 0:
        return out
    xs, os = _items(fn, "x", x, x), _items(fn, "out", out, x)
    gs = _items(fn, "gate", gate, x) if gate is not None else (0, 0)
    desc = _NORM.pack(_DTYPES[x.dtype], n, rows, c, groups, _ACTS[act], x.data_ptr(),
                      gate.data_ptr() if gate is not None else 0,
                      weight.data_ptr() if weight is not None else 0,
                      bias.data_ptr() if bias is not None else 0, out.data_ptr(), *xs, *gs, *os, eps)
    _call("ssla_hip_group_norm", x.device, desc, lambda L: L.ssla_hip_group_norm_workspace)
    return out
