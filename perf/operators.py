"""Performance cases of the sequence operators: linear attention with a decay
for each head (whole prompts and single tokens) and group norm with an
activation over channels-last data.

A case is a dict:
  name     listed cases only
  op       "prompt"  chunked linear attention over packed sequences
           "step"    one token of every sequence against a pool of states
           "norm"    group norm
  dtype    "float32", "bfloat16" or "float16"
prompt and step
  seqs     sequences of the call
  tokens   tokens of the longest sequence (prompt)
  ragged   whether the sequences differ in length (prompt)
  heads, qk_heads, dk, dv
  decay    "head"  one decay a head
           "token" one a token and head
  states   whether states come in (prompt; they always go out)
  fused    whether q, k and v are parts of one projection's rows
  pool     slots of the state pool for each sequence (step)
norm
  n, rows, channels, groups, act, gate
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda:0"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


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
def _prompt(name, dtype, seqs, tokens, heads, dk, dv, qk_heads=None, decay="token", ragged=False,
            states=True, fused=True):
    c = dict(op="prompt", dtype=dtype, seqs=seqs, tokens=tokens, ragged=ragged, heads=heads,
             qk_heads=qk_heads or heads, dk=dk, dv=dv, decay=decay, states=states, fused=fused)
    return dict(c, name=name) if name else c


def _step(name, dtype, seqs, heads, dk, dv, qk_heads=None, decay="token", fused=True, pool=1):
    c = dict(op="step", dtype=dtype, seqs=seqs, heads=heads, qk_heads=qk_heads or heads, dk=dk,
             dv=dv, decay=decay, fused=fused, pool=pool)
    return dict(c, name=name) if name else c


def _norm(name, dtype, n, rows, channels, groups, act="silu", gate=False):
    c = dict(op="norm", dtype=dtype, n=n, rows=rows, channels=channels, groups=groups, act=act,
             gate=gate)
    return dict(c, name=name) if name else c


def listed():
    return [
        # a few tokens appended to one sequence: an interactive turn, at the
        # channel width of the first layer's input
        _prompt("prompt-1x17-h4-24", "float32", 1, 17, 4, 24, 24, decay="head"),
        # one long prompt: the work has to be split along the sequence
        _prompt("prompt-1x8192-h16-128", "bfloat16", 1, 8192, 16, 128, 128),
        # sixteen streams of features at the last layers' width, full precision
        _prompt("prompt-16x2000-h4-96-f32", "float32", 16, 2000, 4, 96, 96, decay="head",
                fused=False),
        # prompts of a serving batch: ragged, shared queries and keys, half precision
        _prompt("prompt-ragged-48x1531-f16", "float16", 48, 1531, 16, 64, 64, qk_heads=4,
                ragged=True),
        # a large prefill batch
        _prompt("prompt-16x8192-h16-128", "bfloat16", 16, 8192, 16, 128, 128, states=False),
        # one user: latency of a token
        _step("step-1-h16-128", "bfloat16", 1, 16, 128, 128),
        # a serving batch out of a larger pool
        _step("step-64-h16-128", "bfloat16", 64, 16, 128, 128, qk_heads=8, pool=2),
        # many streams, the last layers' width, full precision, ragged head sizes
        _step("step-1021-h8-96x80-f32", "float32", 1021, 8, 96, 80, decay="head", fused=False),
        # one small grid: 20 x 16 cells of 48 channels
        _norm("norm-1x320x48", "float32", 1, 320, 48, 8),
        # the norm behind the attention's heads, gated, one row a token
        _norm("norm-8191x1x2048-gate", "bfloat16", 8191, 1, 2048, 16, gate=True),
        # sixteen quarter-resolution grids of 160 x 120 cells of 96 channels
        _norm("norm-16x19200x96", "float32", 16, 19200, 96, 8),
        # one such grid alone: few groups, many rows, an odd group width
        _norm("norm-1x19200x48-f16", "float16", 1, 19200, 48, 16, act="none"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    qk = rng.choice((1, 2, 3, 4, 8, 16))
    return qk * rng.choice((1, 1, 2, 4)) if qk < 16 else 16, qk


def _size(rng):
    """A head's size: usual ones and odd ones."""
    return rng.choice((24, 48, 64, 96, 128)) if rng.random() < 0.6 else _log_int(rng, 8, 256)


def draw(rng):
    op = rng.choice(("prompt", "step", "norm"))
    dtype = rng.choice(("float32", "bfloat16", "bfloat16", "float16"))
    decay, fused = rng.choice(("head", "token")), rng.random() < 0.5
    if op == "norm":
        act = rng.choice(("silu", "silu", "relu", "sigmoid", "none"))
        groups = rng.choice((1, 2, 4, 8, 16, 32))
        channels = groups * _log_int(rng, 1, 2048 // groups)
        rows = 1 if rng.random() < 0.3 else _log_int(rng, 2, 40_000)
        most = max(1, 29_000_000 // (channels * rows))
        return _norm(None, dtype, _log_int(rng, 1, min(most, 16_000)), rows, channels, groups,
                     act, act != "none" and rng.random() < 0.4)
    heads, qk = _heads(rng)
    dk, dv = _size(rng), _size(rng)
    if op == "step":
        most = max(1, 300_000_000 // (heads * dk * dv))
        return _step(None, dtype, _log_int(rng, 1, min(most, 2000)), heads, dk, dv, qk, decay,
                     fused, rng.choice((1, 1, 2, 3)))
    seqs = _log_int(rng, 1, 64)
    most = max(1, 100_000_000 // (heads * (dk + dv)) // seqs)
    return _prompt(None, dtype, seqs, _log_int(rng, 1, min(most, 12_000)), heads, dk, dv, qk, decay,
                   rng.random() < 0.5, rng.random() < 0.5, fused)


def _lengths(case):
    """Tokens of every sequence: with `ragged` they differ, and some have none."""
    t, n = case["tokens"], case["seqs"]
    if not case["ragged"]:
        return [t] * n
    return [0 if s % 11 == 10 else t - t * (5 * s % 8) // 9 for s in range(n)]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
class _State:
    pass


def _rows(case, n, gen):
    """q, k (n, qk_heads, dk) and v (n, heads, dv), of a projection's size."""
    h, hq, dk, dv = case["heads"], case["qk_heads"], case["dk"], case["dv"]
    widths, t = (hq * dk, hq * dk, h * dv), TYPES[case["dtype"]]

    def normal(w):
        return torch.randn(n, w, generator=gen, device=DEV).to(t)

    parts = normal(sum(widths)).split(widths, 1) if case["fused"] else [normal(w) for w in widths]
    return (parts[0].unflatten(1, (hq, dk)), parts[1].unflatten(1, (hq, dk)),
            parts[2].unflatten(1, (h, dv)))


def _decay(case, n, gen):
    """log(decay): fixed ones from a few tokens' memory to hundreds, or a gate's."""
    h = case["heads"]
    if case["decay"] == "head":
        jitter = torch.rand(h, generator=gen, device=DEV)
        return -torch.exp2(-1.0 - 7.0 * (torch.arange(h, device=DEV) + jitter) / h)
    return torch.nn.functional.logsigmoid(
        2.0 + 1.5 * torch.randn(n, h, generator=gen, device=DEV))


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    s = _State()
    s.case = case
    t = TYPES[case["dtype"]]
    if case["op"] == "norm":
        n, r, c = case["n"], case["rows"], case["channels"]
        # channels differ in offset and spread, as a convolution's outputs do
        off = torch.randn(c, generator=gen, device=DEV)
        amp = 0.5 + torch.rand(c, generator=gen, device=DEV)
        s.x = (torch.randn(n, r, c, generator=gen, device=DEV) * amp + off).to(t)
        s.w = (1.0 + 0.2 * torch.randn(c, generator=gen, device=DEV)).to(t)
        s.b = (0.2 * torch.randn(c, generator=gen, device=DEV)).to(t)
        s.gate = torch.randn(n, r, c, generator=gen, device=DEV).to(t) if case["gate"] else None
        return s
    h, dk, dv, n = case["heads"], case["dk"], case["dv"], case["seqs"]
    s.scale = dk ** -0.5
    if case["op"] == "step":
        s.q, s.k, s.v = _rows(case, n, gen)
        s.g = _decay(case, n, gen)
        m = n * case["pool"]
        s.pool = torch.randn(m, h, dk, dv, generator=gen, device=DEV)
        s.slots = torch.randperm(m, generator=gen, device=DEV)[:n].to(torch.int32) \
            if case["pool"] > 1 else None
        return s
    lens = _lengths(case)
    ends = [sum(lens[:i]) for i in range(n + 1)]
    s.cu = torch.tensor(ends, dtype=torch.int32, device=DEV)
    s.longest = max(lens)
    s.q, s.k, s.v = _rows(case, ends[-1], gen)
    s.g = _decay(case, ends[-1], gen)
    s.state_in = torch.randn(n, h, dk, dv, generator=gen, device=DEV) if case["states"] else None
    s.state_out = torch.empty(n, h, dk, dv, device=DEV)
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _plain_norm(s):
    case = s.case
    n, r, c, g = case["n"], case["rows"], case["channels"], case["groups"]
    x = s.x.float().view(n, r, g, c // g)
    d = x - x.mean((1, 3), keepdim=True)
    y = d * torch.rsqrt((d * d).mean((1, 3), keepdim=True) + 1e-5)
    y = y.view(n, r, c) * s.w.float() + s.b.float()
    a = y if s.gate is None else s.gate.float()
    if case["act"] == "silu":
        a = a / (1.0 + torch.exp(-a))
    elif case["act"] == "sigmoid":
        a = 1.0 / (1.0 + torch.exp(-a))
    elif case["act"] == "relu":
        a = torch.clamp(a, min=0.0)
    return (a if s.gate is None else y * a).to(s.x.dtype)


def _spread(x, heads):
    """float32, every head its own (queries and keys may be shared)."""
    x = x.float()
    return x if x.shape[1] == heads else x.repeat_interleave(heads // x.shape[1], 1)


def _plain_step(s):
    h = s.case["heads"]
    q, k, v = _spread(s.q, h), _spread(s.k, h), s.v.float()
    old = s.pool if s.slots is None else s.pool[s.slots.long()]
    new = torch.exp(s.g).expand(q.shape[0], h)[..., None, None] * old + k[..., :, None] * v[..., None, :]
    out = (s.scale * torch.matmul(q[..., None, :], new)[..., 0, :]).to(s.q.dtype)
    if s.slots is None:
        s.pool.copy_(new)
    else:
        s.pool.index_copy_(0, s.slots.long(), new)
    return {"out": out, "pool": s.pool}


CHUNK = 64


def _plain_prompt(s):
    """Chunks of 64 tokens: products inside the chunks, the states before them
    from the chunks' own by one more product.  Exponents in 64 bits."""
    case = s.case
    h, dk, dv, nb = case["heads"], case["dk"], case["dv"], case["seqs"]
    total = s.q.shape[0]
    nc = -(-s.longest // CHUNK)
    # sequences side by side, filled up with zeros (which change no state)
    at = s.cu[:-1, None].long() + torch.arange(nc * CHUNK, device=DEV)
    real = at < s.cu[1:, None]
    at = at.clamp(max=total - 1)

    def chunks(x):
        x = torch.where(real[..., None, None], x[at], 0.0)
        return x.view(nb, nc, CHUNK, h, x.shape[-1]).transpose(2, 3)        # (nb, nc, h, C, d)

    q, k, v = chunks(_spread(s.q, h)), chunks(_spread(s.k, h)), chunks(s.v.float())
    g = torch.where(real[..., None], s.g.expand(total, h)[at].double(), 0.0)
    b = g.view(nb, nc, CHUNK, h).cumsum(2).transpose(2, 3)                  # (nb, nc, h, C)
    i = torch.arange(CHUNK, device=DEV)
    w = torch.where(i[:, None] >= i, b[..., :, None] - b[..., None, :], -math.inf).float().exp_()
    out = torch.matmul(torch.matmul(q, k.transpose(3, 4)).mul_(w), v)
    del w
    end = b[..., -1]                                                        # (nb, nc, h)
    local = torch.matmul((k * torch.exp(end[..., None] - b).float()[..., None]).transpose(3, 4), v)
    # state before chunk n, and behind the last: sum over m < n of decay(m + 1 .. n - 1) local(m)
    run = torch.cat([torch.zeros_like(end[:, :1]), end.cumsum(1)], 1).transpose(1, 2)  # (nb, h, nc + 1)
    n, m = torch.arange(nc + 1, device=DEV), torch.arange(nc, device=DEV)
    d = torch.where(n[:, None] > m, run[..., :, None] - run[..., None, 1:], -math.inf).float().exp_()
    before = torch.matmul(d, local.transpose(1, 2).reshape(nb, h, nc, dk * dv))
    del local, d
    if s.state_in is not None:
        before += torch.exp(run).float()[..., None] * s.state_in.reshape(nb, h, 1, dk * dv)
    before = before.view(nb, h, nc + 1, dk, dv).transpose(1, 2)
    s.state_out.copy_(before[:, -1])
    out += torch.exp(b).float()[..., None] * torch.matmul(q, before[:, :-1])
    out = (s.scale * out).transpose(2, 3).reshape(nb, nc * CHUNK, h, dv)
    return {"out": out[real].to(s.q.dtype), "state": s.state_out}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    case = s.case
    if not own:
        return {"norm": _plain_norm, "step": _plain_step, "prompt": _plain_prompt}[case["op"]](s)
    ops = _ops()
    if case["op"] == "norm":
        return ops.group_norm(s.x, case["groups"], s.w, s.b, eps=1e-5, act=case["act"],
                              gate=s.gate)
    if case["op"] == "step":
        out = ops.linear_attention_step(s.q, s.k, s.v, s.g, s.pool, scale=s.scale, slots=s.slots)
        return {"out": out, "pool": s.pool}
    out = ops.linear_attention(s.q, s.k, s.v, s.g, scale=s.scale, cu_seqlens=s.cu,
                               max_len=s.longest, state_in=s.state_in, state_out=s.state_out)
    return {"out": out, "state": s.state_out}


# ---------------------------------------------------------------------------
# work, and the same in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    e = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "norm":
        n = case["n"] * case["rows"] * case["channels"]
        return {"bytes": n * e * (3 if case["gate"] else 2) + 2 * case["channels"] * e,
                "flops": 10 * n}
    h, hq, dk, dv, n = (case[x] for x in ("heads", "qk_heads", "dk", "dv", "seqs"))
    t = n if case["op"] == "step" else sum(_lengths(case))
    rows = t * (2 * hq * dk + 2 * h * dv) * e + 4 * h * (t if case["decay"] == "token" else 1)
    states = n * h * dk * dv * 4 * (2 if case["op"] == "step" or case["states"] else 1)
    return {"bytes": rows + states, "flops": 4 * t * h * dk * dv}


def _exact_norm(s):
    """One channel's sums at a time, the groups' from them."""
    case = s.case
    g, c, r = case["groups"], case["channels"], case["rows"]
    x = s.x.double()
    m = c // g * r
    s1 = x.sum(1).view(-1, g, c // g).sum(2)
    mean = (s1 / m).repeat_interleave(c // g, 1)[:, None]
    s2 = (x - mean).pow(2).sum(1).view(-1, g, c // g).sum(2)
    y = (x - mean) / (s2 / m + 1e-5).sqrt().repeat_interleave(c // g, 1)[:, None]
    y = y * s.w.double() + s.b.double()
    a = y if s.gate is None else s.gate.double()
    a = {"silu": lambda z: z * torch.sigmoid(z), "sigmoid": torch.sigmoid, "relu": torch.relu,
         "none": lambda z: z}[case["act"]](a)
    return a if s.gate is None else y * a


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(s)
    h, dk, dv, nb = case["heads"], case["dk"], case["dv"], case["seqs"]
    rep = h // case["qk_heads"]
    q, k = (x.double().repeat_interleave(rep, 1) for x in (s.q, s.k))
    v = s.v.double()
    a = torch.exp(s.g.double())

    def token(state, rows):
        """One token of the sequences: their new states and outputs."""
        decay = a[rows] if a.dim() == 2 else a.expand(rows.numel(), h)
        state = state * decay[..., None, None] + k[rows][..., None] * v[rows][:, :, None]
        return state, s.scale * (q[rows][..., None] * state).sum(2)

    if case["op"] == "step":
        slots = torch.arange(nb, device=DEV) if s.slots is None else s.slots.long()
        new, out = token(s.pool[slots].double(), torch.arange(nb, device=DEV))
        pool = s.pool.double()
        pool[slots] = new
        return {"out": out, "pool": pool}
    if s.longest * (200 + nb * h * dk * dv / 5e4) > 15e6:        # about a microsecond a unit
        return None
    lens = torch.tensor(_lengths(case), device=DEV)
    state = torch.zeros(nb, h, dk, dv, dtype=torch.float64, device=DEV) if s.state_in is None \
        else s.state_in.double()
    out = torch.zeros(q.shape[0], h, dv, dtype=torch.float64, device=DEV)
    # the longest sequences first, so that those with a token t left are the first ones
    order = torch.argsort(lens, descending=True)
    starts, state = s.cu[:-1].long()[order], state[order]
    sizes = lens[order].tolist()
    left = nb
    for t in range(s.longest):
        while sizes[left - 1] <= t:
            left -= 1
        state[:left], out[starts[:left] + t] = token(state[:left], starts[:left] + t)
    back = torch.empty_like(state)
    back[order] = state
    return {"out": out, "state": back}
