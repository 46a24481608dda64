"""Performance cases of the operators that models around the drain are trained
with: the gated linear recurrence of an SSLA layer (whole sequences, their
gradients, and single tokens) and layer norm with its gradients.

A case is a dict:
  name     listed cases only
  op       "scan"   the recurrence over packed sequences, states in and out
           "train"  the same and its gradients
           "step"   one token of every sequence against a pool of states
           "norm"   layer norm
  dtype    "float32", "bfloat16" or "float16"
scan and train
  seqs     sequences of the call
  tokens   tokens of the call ("cells"), else of the longest sequence
  lengths  "even"   all the same
           "ragged" they differ, some have none
           "cells"  records dealt to the cells of a grid
  channels
  read     whether the states are read out by q
  states   whether states come in, and the last ones go out
  fused    whether gate, v and q are parts of one projection's rows
step
  seqs, channels, read, fused, pool (slots for each sequence)
norm
  rows, channels, affine, residual, grad (the gradients too)
"""
import math
import os
import random
import sys

import torch

own = False
DEV = "cuda:0"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
EPS = 1e-5


def _ops():
    """The framework's operators; imported only where they are measured."""
    path = os.path.join(os.getcwd(), "ssla-rt_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from ssla_hip import ops
    return ops


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _named(name, c):
    return dict(c, name=name) if name else c


def _seq(name, op, dtype, seqs, tokens, channels, lengths="even", read=True, states=False,
         fused=True):
    return _named(name, dict(op=op, dtype=dtype, seqs=seqs, tokens=tokens, channels=channels,
                             lengths=lengths, read=read, states=states, fused=fused))


def _step(name, dtype, seqs, channels, read=True, fused=True, pool=1):
    return _named(name, dict(op="step", dtype=dtype, seqs=seqs, channels=channels, read=read,
                             fused=fused, pool=pool))


def _norm(name, dtype, rows, channels, affine=True, residual=False, grad=True):
    return _named(name, dict(op="norm", dtype=dtype, rows=rows, channels=channels, affine=affine,
                             residual=residual, grad=grad))


def listed():
    return [
        # a few records more of one stream, at the last layers' width: latency
        _seq("scan-1x17x96-f32", "scan", "float32", 1, 17, 96, states=True),
        # one long stream through a wide layer: the work is split along the tokens
        _seq("scan-1x40001x1024", "scan", "bfloat16", 1, 40_001, 1024, states=True),
        # the first drained layer over 200k records of an 80 x 64 camera, sorted by
        # the 20 x 16 grid's cell, the cells' states going in and out
        _seq("scan-cells-320-f32", "scan", "float32", 320, 200_000, 48, "cells", states=True),
        # a small training batch at the last layers' width: latency
        _seq("train-16x100x96-f32", "train", "float32", 16, 100, 96, states=True),
        # one long training sequence of a wide layer
        _seq("train-1x8192x2048", "train", "bfloat16", 1, 8192, 2048),
        # a ragged batch of odd width in half precision, states read as they are
        _seq("train-ragged-48x1531x1001-f16", "train", "float16", 48, 1531, 1001, "ragged",
             read=False, states=True, fused=False),
        # training on 1.25M records of a 640 x 480 camera by the 160 x 120 grid's cells
        _seq("train-cells-19200-f32", "train", "float32", 19_200, 1_250_000, 48, "cells"),
        # one user: latency of a token
        _step("step-1x2048", "bfloat16", 1, 2048),
        # every cell of a 160 x 120 grid, out of a larger pool
        _step("step-19200x96-f32", "float32", 19_200, 96, fused=False, pool=2),
        # the norm behind a contraction alone, on the cells of one grid: latency
        _norm("norm-320x48-f32", "float32", 320, 48, residual=True, grad=False),
        # a training step's norm of 8191 tokens behind a residual branch
        _norm("norm-train-8191x2048", "bfloat16", 8191, 2048, residual=True),
        # a layer's norm over 1.25M records of 96 channels, with its gradients
        _norm("norm-train-1250000x96-f32", "float32", 1_250_000, 96),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, hi):
    """Channels: usual widths and odd ones."""
    if rng.random() < 0.5:
        return rng.choice([c for c in (24, 48, 96, 256, 1024, 2048, 4096) if c <= hi])
    return _log_int(rng, 8, hi)


def draw(rng):
    op = rng.choice(("scan", "train", "train", "step", "norm", "norm"))
    dtype = rng.choice(("float32", "bfloat16", "bfloat16", "float16"))
    if op == "norm":
        channels = _width(rng, 8192)
        return _norm(None, dtype, _log_int(rng, 1, max(1, 90_000_000 // channels)), channels,
                     rng.random() < 0.8, rng.random() < 0.4, rng.random() < 0.7)
    channels = _width(rng, 4096)
    read, fused = rng.random() < 0.7, rng.random() < 0.5
    if op == "step":
        return _step(None, dtype, _log_int(rng, 1, max(1, min(40_000, 20_000_000 // channels))),
                     channels, read, fused, rng.choice((1, 1, 2, 3)))
    states = rng.random() < 0.5
    most = 55_000_000 // channels
    if rng.random() < 0.25:
        seqs = _log_int(rng, 16, min(20_000, most // 8))
        return _seq(None, op, dtype, seqs, max(1, min(most, seqs * _log_int(rng, 2, 600))), channels,
                    "cells", read, states, fused)
    seqs = _log_int(rng, 1, min(64, most))
    return _seq(None, op, dtype, seqs, _log_int(rng, 1, max(1, min(most // seqs, 60_000))), channels,
                rng.choice(("even", "ragged")), read, states, fused)


def _lengths(case):
    """Tokens of every sequence."""
    t, n = case["tokens"], case["seqs"]
    if case["lengths"] == "ragged":
        return [0 if s % 11 == 10 else t - t * (5 * s % 8) // 9 for s in range(n)]
    if case["lengths"] == "cells":
        # some cells see ten times the records of others, many hardly any
        rng = random.Random(n * 1_000_003 + t)
        w = [math.exp(rng.gauss(0.0, 1.0)) for _ in range(n)]
        total, ends, run = sum(w), [], 0.0
        for x in w:
            run += x
            ends.append(int(t * run / total))
        ends[-1] = t
        return [b - a for a, b in zip([0] + ends, ends)]
    return [t] * n


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
class _State:
    pass


def _rows(case, n, gen):
    """gate, v and (with `read`) q (n, channels), of a projection's size; the
    gates remember from a token to a hundred and more."""
    c, t, k = case["channels"], TYPES[case["dtype"]], 3 if case["read"] else 2
    if case["fused"]:
        x = torch.randn(n, k * c, generator=gen, device=DEV)
        x[:, :c].mul_(1.5).add_(2.0)
        parts = x.to(t).split(c, 1)
    else:
        parts = [torch.randn(n, c, generator=gen, device=DEV) for _ in range(k)]
        parts[0].mul_(1.5).add_(2.0)
        parts = [p.to(t) for p in parts]
    return parts[0], parts[1], parts[2] if case["read"] else None


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    s = _State()
    s.case = case
    t, c = TYPES[case["dtype"]], case["channels"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    if case["op"] == "norm":
        n = case["rows"]
        # channels differ in offset and spread, as a contraction's outputs do
        s.x = (normal(n, c) * (0.5 + torch.rand(c, generator=gen, device=DEV)) + normal(c)).to(t)
        s.res = normal(n, c).to(t) if case["residual"] else None
        s.w = (1.0 + 0.2 * normal(c)).to(t) if case["affine"] else None
        s.b = (0.2 * normal(c)).to(t) if case["affine"] else None
        s.dy = normal(n, c).to(t) if case["grad"] else None
        s.leaves = [x for x in (s.x, s.res, s.w, s.b) if x is not None]
    elif case["op"] == "step":
        n, m = case["seqs"], case["seqs"] * case["pool"]
        s.gate, s.v, s.q = _rows(case, n, gen)
        s.pool = normal(m, c)
        s.slots = torch.randperm(m, generator=gen, device=DEV)[:n].to(torch.int32) \
            if case["pool"] > 1 else None
        return s
    else:
        n, lens = case["seqs"], _lengths(case)
        ends = torch.tensor([0] + lens).cumsum(0)
        total = int(ends[-1])
        s.longest = max(lens)
        s.cu = ends.to(torch.int32).to(DEV) if case["lengths"] != "even" else None
        s.gate, s.v, s.q = _rows(case, total, gen)
        s.state_in = normal(n, c) if case["states"] else None
        s.state_out = torch.empty(n, c, device=DEV) if case["states"] else None
        s.dout = normal(total, c).to(t) if case["op"] == "train" else None
        s.dstate = normal(n, c) if case["op"] == "train" and case["states"] else None
        s.leaves = [x for x in (s.gate, s.v, s.q, s.state_in) if x is not None]
    if case["op"] == "train" or case.get("grad"):
        # what a model's layer gets: gradients are wanted, none is kept
        s.leaves = [x.detach().requires_grad_() for x in s.leaves]
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _plain_norm(s):
    x = s.x.float() if s.res is None else s.x.float() + s.res.float()
    d = x - x.mean(1, keepdim=True)
    r = torch.rsqrt((d * d).mean(1, keepdim=True) + EPS)
    xh = d.mul_(r)
    y = xh if s.w is None else xh * s.w.float() + s.b.float()
    y = y.to(s.x.dtype)
    if s.dy is None:
        return y
    dy = s.dy.float()
    u = dy if s.w is None else dy * s.w.float()
    dx = r * (u - u.mean(1, keepdim=True) - xh * (u * xh).mean(1, keepdim=True))
    dx = dx.to(s.x.dtype)
    out = {"y": y, "dx": dx}
    if s.res is not None:
        out["dres"] = dx
    if s.w is not None:
        out["dw"], out["db"] = (dy * xh).sum(0).to(s.w.dtype), dy.sum(0).to(s.b.dtype)
    return out


def _scan(a, x, longest):
    """h_t = a_t h_{t-1} + x_t along the first dimension, in steps of 1, 2, 4 ...
    tokens; a is zero where a sequence begins."""
    n = 1
    while n < longest:
        x = torch.cat([x[:n], x[n:] + a[n:] * x[:-n]])
        if 2 * n < longest:
            a = torch.cat([a[:n], a[n:] * a[:-n]])
        n *= 2
    return x


def _bounds(s, total):
    """First and last token of each sequence that has any, and which those are."""
    if s.cu is None:
        n = s.case["seqs"]
        first = torch.arange(0, total, total // n, device=DEV)
        return first, first + (total // n - 1), torch.arange(n, device=DEV)
    cu = s.cu.long()
    some = torch.nonzero(cu[1:] > cu[:-1])[:, 0]
    return cu[some], cu[some + 1] - 1, some


def _plain_scan(s):
    total, train = s.gate.shape[0], s.case["op"] == "train"
    first, last, some = _bounds(s, total)
    a = torch.sigmoid(s.gate.float())
    x, b = s.v.float(), a.clone()
    if s.state_in is not None:
        x = x.index_add(0, first, a[first] * s.state_in[some])
    b[first] = 0.0
    h = _scan(b, x, s.longest)
    out = {"out": (h if s.q is None else s.q.float() * h).to(s.v.dtype)}
    if s.state_out is not None:
        state = s.state_in.clone()
        state[some] = h[last]
        if train:
            out["state"] = state
        else:
            out["state"] = s.state_out.copy_(state)
    if not train:
        return out
    e = s.dout.float()
    if s.q is not None:
        out["dq"] = (e * h).to(s.v.dtype)
        e = e * s.q.float()
    if s.dstate is not None:
        e = e.index_add(0, last, s.dstate[some])
    # backwards, each token's factor is the next one's gate
    up = torch.cat([b[1:], torch.zeros_like(b[:1])])
    dh = _scan(up.flip(0), e.flip(0), s.longest).flip(0)
    del up, e, b
    before = torch.cat([torch.zeros_like(h[:1]), h[:-1]])
    before[first] = 0.0 if s.state_in is None else s.state_in[some]
    out["dv"] = dh.to(s.v.dtype)
    out["dgate"] = (dh * before * (a * (1.0 - a))).to(s.v.dtype)
    if s.state_in is not None:
        ds = s.dstate.clone()
        ds[some] = a[first] * dh[first]
        out["dstate_in"] = ds
    return out


def _plain_step(s):
    old = s.pool if s.slots is None else s.pool[s.slots.long()]
    new = torch.sigmoid(s.gate.float()) * old + s.v.float()
    out = (new if s.q is None else s.q.float() * new).to(s.v.dtype)
    if s.slots is None:
        s.pool.copy_(new)
    else:
        s.pool.index_copy_(0, s.slots.long(), new)
    return {"out": out, "pool": s.pool}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    case = s.case
    if not own:
        return {"norm": _plain_norm, "step": _plain_step}.get(case["op"], _plain_scan)(s)
    ops = _ops()
    if case["op"] == "step":
        out = ops.linear_recurrence_step(s.gate, s.v, s.pool, s.q, slots=s.slots)
        return {"out": out, "pool": s.pool}
    if case["op"] == "norm":
        left = list(s.leaves)
        x = left.pop(0)
        res = left.pop(0) if s.res is not None else None
        w, b = left or (None, None)
        y = ops.layer_norm(x, w, b, eps=EPS, residual=res)
        if s.dy is None:
            return y
        grads = torch.autograd.grad(y, s.leaves, s.dy)
        names = ["dx"] + ["dres"] * (res is not None) + ["dw", "db"] * (w is not None)
        return dict(zip(names, grads), y=y.detach())
    if case["op"] == "scan":
        out = ops.linear_recurrence(s.gate, s.v, s.q, cu_seqlens=s.cu, n_seqs=case["seqs"],
                                    state_in=s.state_in, state_out=s.state_out)
        return {"out": out} if s.state_out is None else {"out": out, "state": s.state_out}
    left = list(s.leaves)
    gate, v = left.pop(0), left.pop(0)
    q = left.pop(0) if s.q is not None else None
    state = left.pop(0) if left else None
    got = ops.linear_recurrence(gate, v, q, cu_seqlens=s.cu, n_seqs=case["seqs"], state_in=state,
                                return_state=case["states"])
    if case["states"]:
        grads = torch.autograd.grad(got, s.leaves, (s.dout, s.dstate))
        out = {"out": got[0].detach(), "state": got[1].detach()}
    else:
        grads = torch.autograd.grad(got, s.leaves, s.dout)
        out = {"out": got.detach()}
    names = ["dgate", "dv"] + ["dq"] * (q is not None) + ["dstate_in"] * (state is not None)
    return dict(out, **dict(zip(names, grads)))


# ---------------------------------------------------------------------------
# work, and the same in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    e, c = 4 if case["dtype"] == "float32" else 2, case["channels"]
    if case["op"] == "norm":
        n = case["rows"] * c
        tensors = 2 + case["residual"] + 2 * case["grad"]
        return {"bytes": n * e * tensors + (2 + 2 * case["grad"]) * case["affine"] * c * e,
                "flops": n * (24 if case["grad"] else 8)}
    k = 4 if case["read"] else 3                       # gate, v, q and out
    if case["op"] == "step":
        n = case["seqs"] * c
        return {"bytes": n * (k * e + 8), "flops": 8 * n}
    n, train = sum(_lengths(case)) * c, case["op"] == "train"
    states = case["seqs"] * c * 4 * (4 if train else 2) if case["states"] else 0
    # with gradients: out's too, and one of every input
    return {"bytes": n * e * (2 * k if train else k) + states, "flops": n * (24 if train else 8)}


def _exact_norm(s):
    def leaf(x):
        return None if x is None else x.detach().double().requires_grad_(s.dy is not None)

    x, res, w, b = leaf(s.x), leaf(s.res), leaf(s.w), leaf(s.b)
    z = x if res is None else x + res
    m = z.sum(1, keepdim=True) / z.shape[1]
    var = ((z - m) ** 2).sum(1, keepdim=True) / z.shape[1]
    y = (z - m) / (var + EPS).sqrt()
    if w is not None:
        y = y * w + b
    if s.dy is None:
        return y
    names = {"dx": x, "dres": res, "dw": w, "db": b}
    names = {k: t for k, t in names.items() if t is not None}
    grads = torch.autograd.grad(y, list(names.values()), s.dy.double())
    return dict(zip(names, grads), y=y.detach())


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(s)
    a = 1.0 / (1.0 + torch.exp(-s.gate.double()))
    v = s.v.double()
    q = torch.ones_like(v) if s.q is None else s.q.double()
    if case["op"] == "step":
        slots = torch.arange(case["seqs"], device=DEV) if s.slots is None else s.slots.long()
        pool = s.pool.double()
        h = a * pool[slots] + v
        pool[slots] = h
        return {"out": q * h, "pool": pool}
    # token by token, the longest sequences first, so that those with a token left
    # are the first ones
    lens = torch.tensor(_lengths(case))
    n, c = case["seqs"], case["channels"]
    if s.longest * (60 + n * c / 2e5) > 4e6:           # microseconds, or so
        return None
    order = torch.argsort(lens, descending=True)
    first = (lens.cumsum(0) - lens)[order].to(DEV)
    sizes = lens[order].tolist()
    order = order.to(DEV)
    zero = torch.zeros(n, c, dtype=torch.float64, device=DEV)
    start = zero if s.state_in is None else s.state_in.double()
    state = start[order]
    hs = torch.empty_like(v)
    left, lefts = n, []
    for t in range(s.longest):
        while sizes[left - 1] <= t:
            left -= 1
        lefts.append(left)
        at = first[:left] + t
        state[:left] = a[at] * state[:left] + v[at]
        hs[at] = state[:left]
    out = {"out": q * hs}
    if case["states"]:
        out["state"] = torch.empty_like(state)
        out["state"][order] = state
    if case["op"] == "scan":
        return out
    do = s.dout.double()
    # what comes to h_t from behind; for a sequence's last token its state's gradient
    back = (zero if s.dstate is None else s.dstate.double())[order]
    dv, dgate = torch.empty_like(v), torch.empty_like(v)
    for t in range(s.longest - 1, -1, -1):
        left = lefts[t]
        at = first[:left] + t
        dh = q[at] * do[at] + back[:left]
        dv[at] = dh
        before = hs[at - 1] if t else start[order[:left]]
        dgate[at] = dh * before * a[at] * (1.0 - a[at])
        back[:left] = a[at] * dh
    out.update(dv=dv, dgate=dgate)
    if s.q is not None:
        out["dq"] = do * hs
    if s.state_in is not None:
        out["dstate_in"] = torch.empty_like(back)
        out["dstate_in"][order] = back
    return out
