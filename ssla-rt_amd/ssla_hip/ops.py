"""Sequence operators of libssla_hip.so on torch device tensors.

  linear_attention       whole sequences (packed, ragged), states in and out
  linear_attention_step  one token of every sequence, states updated in a pool
  group_norm             group norm with an activation, channels last
  linear_recurrence      an SSLA layer's recurrence over whole sequences (packed,
                         ragged), states in and out, with gradients
  linear_recurrence_step  its single tokens, states updated in a pool
  layer_norm             layer norm, of a sum with a residual too, with gradients

The formulas, layouts and limits are those of include/ssla_hip.h (sequence
operators).  Calls are queued on torch's current stream of the tensors'
device, which need not be the current device; outputs and workspaces come
from torch's allocator, so calls can be captured into a graph.  Tensors that do
not fit raise ValueError, what the library refuses (values out of range, rows of
out or pools that overlap) lib.SslaHipError, before anything is queued.
linear_recurrence and layer_norm are functions of torch's autograd: where it
records, their outputs are new tensors with first derivatives (second ones are
refused), and a call in a capture refuses leaves given to it whose older graph,
recorded on the default stream, still lives.  The others have no gradients:
tensors that require one are refused while torch records.  Tensors that carry a
forward gradient are refused everywhere; tensors that a call writes to get a new
version.  There is no fallback: without the library, or for tensors off the GPU, a
call raises.

The checks and the calls are in csrc/ops_torch.cpp and csrc/ops_train_torch.cpp
(_ops.so).
"""
from __future__ import annotations

from typing import Optional

import torch

from . import abi

try:
    from . import _ops
except ImportError as e:
    raise ImportError(f"{e}: build the library first (make -C ssla-rt_amd)") from e

_ACTS = {"none": abi.SSLA_ACT_NONE, None: abi.SSLA_ACT_NONE, "silu": abi.SSLA_ACT_SILU,
         "sigmoid": abi.SSLA_ACT_SIGMOID, "relu": abi.SSLA_ACT_RELU}


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
                (None: zeros) and written to; may be the same (no slot of one
                may overlap one of the other otherwise)
    slots       int32 (sequences,) slots of the sequences, each its own (None:
                slot s for sequence s); a sequence with a negative slot is
                passed over
    Returns out (tokens, heads, dv) in q's type; rows of no sequence are left
    as they are (uninitialised where out is made here)."""
    return _ops.linear_attention(q, k, v, log_decay, out, scale, cu_seqlens, max_len, n_seqs,
                                 state_in, state_out, slots)


def linear_attention_step(q, k, v, log_decay, state, out=None, *, scale: float = 1.0,
                          slots=None) -> torch.Tensor:
    """One token of every sequence: row s of q, k (sequences, qk_heads, dk),
    v (sequences, heads, dv) and log_decay ((sequences, heads), or (heads,))
    belongs to sequence s.  Its state, slot slots[s] (None: s) of `state`
    (float32 (slots, heads, dk, dv)), is updated in place; out[s] is read from
    the new one.  A row with a negative slot is passed over.  Returns out."""
    return _ops.linear_attention_step(q, k, v, log_decay, state, out, scale, slots)


def group_norm(x, groups: int, weight=None, bias=None, out=None, *, eps: float = 1e-5,
               act: Optional[str] = None, gate=None) -> torch.Tensor:
    """Group norm of x (n, ..., channels), channels last, over the dimensions
    between and the channels / groups neighbouring channels of a group; then
    act ("none", "silu", "sigmoid", "relu") of it, or, with `gate` (of x's
    shape), the norm times act(gate).  (tokens, channels) normalises each
    token's groups by themselves, as behind an attention's heads.  weight, bias
    (channels,) in x's type.  out may be x.  Returns out (x's shape and type)."""
    if act not in _ACTS:
        raise ValueError(f"group_norm: act must be one of {[a for a in _ACTS if a]}")
    return _ops.group_norm(x, groups, weight, bias, out, eps, _ACTS[act], gate)


def linear_recurrence(gate, v, q=None, out=None, *, cu_seqlens=None, n_seqs: int = 1,
                      state_in=None, state_out=None, slots=None, return_state: bool = False):
    """h_t = sigmoid(gate_t) h_{t-1} + v_t, out_t = q_t h_t (h_t without q),
    channel by channel, over packed sequences.

    gate, v, q  (tokens, channels): any stride between tokens, channels contiguous
    cu_seqlens  int32 (sequences + 1,) on the device: the sequences' first
                tokens and the last one's end.  None: n_seqs sequences of the
                same length
    state_in, state_out  float32 (slots, channels) pools, read from (None: zeros)
                and written to; may be the same (no slot of one may overlap one of
                the other otherwise)
    slots       int32 (sequences,) slots of the sequences, each its own (None:
                slot s for sequence s); a sequence with a negative slot is
                passed over
    return_state  the sequences' last states come with out, float32
                (sequences, channels), in place of state_out
    Returns out (tokens, channels) in gate's type, or (out, state).  Rows of no
    sequence are left as they are (uninitialised where out is made here).

    Where torch records a gradient of gate, v, q or state_in (one row for each
    sequence then), out, state_out and slots must be None; rows of no sequence are
    zeros, and so are their gradients."""
    got = _ops.linear_recurrence(gate, v, q, out, cu_seqlens, n_seqs, state_in, state_out, slots,
                                 return_state)
    return got if return_state else got[0]


def linear_recurrence_step(gate, v, state, q=None, out=None, *, slots=None) -> torch.Tensor:
    """One token of every sequence: row s of gate, v and q (sequences, channels)
    belongs to sequence s.  Its state, slot slots[s] (None: s) of `state` (float32
    (slots, channels)), is updated in place; out[s] is read from the new one.  A
    row with a negative slot is passed over.  Returns out."""
    return _ops.linear_recurrence_step(gate, v, state, q, out, slots)


def layer_norm(x, weight=None, bias=None, out=None, *, eps: float = 1e-5,
               residual=None) -> torch.Tensor:
    """Layer norm of x, or of x + residual, over the last dimension: (s - mean) /
    sqrt(var + eps) * weight + bias.  x (..., channels) and residual (of x's
    shape): channels contiguous, rows at one stride.  weight, bias (channels,)
    in x's type or both in float32.  out may be x or residual.  Returns out (x's
    shape and type).  Where torch records a gradient, out must be None."""
    return _ops.layer_norm(x, weight, bias, out, eps, residual)
