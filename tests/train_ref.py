"""Plain 64-bit forms of the operators with gradients, and the error their kernels
may have, from counts of fp32 roundings (U32 each)."""
import torch

from seq_ref import TYPES, U32, half_step, tiny  # noqa: F401


def f64(t):
    return None if t is None else t.detach().cpu().double()


def recurrence(gate, v, q, bounds, state_in=None, dout=None, dstate=None):
    """Token by token.  bounds: [(first, end)] of the sequences.  Returns a dict of
    values, and one of the errors allowed before an output's own rounding.

    A step's own error is at most k U32 of the magnitude that comes out of it: the
    gate's exponential has an argument off by half a step (|gate| U32), and some ten
    roundings of its quotient, the products and sums; joining maps of several tokens
    takes a rounding more a token.  Errors go through the steps as the values do."""
    g, v = f64(gate), f64(v)
    T, C = v.shape
    q_ = torch.ones_like(v) if q is None else f64(q)
    a, s = torch.sigmoid(g), torch.sigmoid(-g.abs())
    k = (g.abs() + 16) * U32
    n = len(bounds)
    h, M, E = (torch.zeros(T, C, dtype=torch.float64) for _ in range(3))
    first = torch.zeros(n, C, dtype=torch.float64) if state_in is None else f64(state_in)
    last, lastM, lastE = first.clone(), first.abs(), torch.zeros_like(first)
    hb, Mb, Eb = (torch.zeros(T, C, dtype=torch.float64) for _ in range(3))     # before a token
    for i, (t0, t1) in enumerate(bounds):
        x, m, e = first[i], first[i].abs(), torch.zeros(C, dtype=torch.float64)
        for t in range(t0, t1):
            hb[t], Mb[t], Eb[t] = x, m, e
            x = a[t] * x + v[t]
            m = a[t] * m + v[t].abs()
            e = a[t] * e + k[t] * m
            h[t], M[t], E[t] = x, m, e
        if t1 > t0:
            last[i], lastM[i], lastE[i] = x, m, e
    val = {"out": q_ * h, "state": last}
    tol = {"out": q_.abs() * (E + 2 * U32 * M), "state": lastE + 2 * U32 * lastM}
    if dout is None and dstate is None:
        return val, tol
    do = torch.zeros_like(v) if dout is None else f64(dout)
    dh, D, F = (torch.zeros(T, C, dtype=torch.float64) for _ in range(3))
    dfirst = torch.zeros(n, C, dtype=torch.float64) if dstate is None else f64(dstate).clone()
    tfirst = torch.zeros_like(dfirst)
    for i, (t0, t1) in enumerate(bounds):
        x = dfirst[i].clone()
        m, e = x.abs(), torch.zeros(C, dtype=torch.float64)
        for t in range(t1 - 1, t0 - 1, -1):
            x = x + q_[t] * do[t]
            m = m + (q_[t] * do[t]).abs()
            e = e + k[t] * m
            dh[t], D[t], F[t] = x, m, e
            x, m, e = a[t] * x, a[t] * m, a[t] * (e + k[t] * m)
        dfirst[i], tfirst[i] = x, e + (2 * U32 * m if t1 > t0 else 0)
    slope = s * (1 - s)
    val.update(dgate=dh * hb * slope, dv=dh, dstate_in=dfirst)
    tol.update(dgate=slope * (F * Mb + D * Eb + 2 * k * D * Mb), dv=F + 2 * U32 * D, dstate_in=tfirst)
    if q is not None:
        val["dq"], tol["dq"] = do * h, do.abs() * (E + 2 * U32 * M)
    return val, tol


def check(name, got, val, tol):
    """`got` against the value, rounded once to its type."""
    assert torch.isfinite(got).all(), f"{name} is not finite"
    t = 1.01 * tol + half_step(got.dtype) * (1 + 2.0 ** -8) * val.abs() + tiny(got.dtype)
    err = (f64(got) - val).abs()
    worst = (err / t).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.3g} of the tolerance"


def layer_norm(x, res, w, b, eps, dy=None):
    """Values and errors.  x + residual is rounded once; the mean is off by 2^-48 of
    itself, and by what that sum's rounding adds; the square root by 4 roundings; sums
    of the backward pass by at most 96 (the roundings that a value can go through:
    32 in a lane, 10 between lanes and waves, four products, twice), those over rows by
    one a row."""
    x64 = f64(x) + (0 if res is None else f64(res))
    C = x64.shape[-1]
    shape = x64.shape
    x64 = x64.reshape(-1, C)
    mean = x64.mean(1, keepdim=True)
    d = x64 - mean
    var = (d * d).mean(1, keepdim=True)
    r = 1.0 / torch.sqrt(var + eps)
    xh = d * r
    sum_off = torch.zeros_like(x64) if res is None else U32 * x64.abs()
    off = (sum_off + sum_off.mean(1, keepdim=True)) * r
    off = off + 2.0 ** -45 * mean.abs() * r + 8 * U32 * xh.abs()
    # of the variance: from the summands' errors
    off = off + xh.abs() * (2 * (d.abs() * sum_off).mean(1, keepdim=True) + (sum_off ** 2).mean(1, keepdim=True)) * r * r
    W = torch.ones(C, dtype=torch.float64) if w is None else f64(w)
    B = torch.zeros(C, dtype=torch.float64) if b is None else f64(b)
    y = xh * W + B
    val = {"y": y.reshape(shape)}
    tol = {"y": (off * W.abs() + 4 * U32 * (y.abs() + B.abs())).reshape(shape)}
    if dy is None:
        return val, tol
    g = f64(dy).reshape(-1, C)
    u = g * W
    c1, c2 = u.mean(1, keepdim=True), (u * xh).mean(1, keepdim=True)
    dx = r * (u - c1 - xh * c2)
    n = 96 * U32
    t = (4 * U32 * u.abs() + n * (u.abs().mean(1, keepdim=True) + xh.abs() * (u * xh).abs().mean(1, keepdim=True))
         + off * c2.abs() + xh.abs() * (u.abs() * off).mean(1, keepdim=True))
    rel = 16 * U32 + (2 * (d.abs() * sum_off).mean(1, keepdim=True)) * r * r
    val["dx"], tol["dx"] = dx.reshape(shape), (r * t + rel * (dx.abs() + r * u.abs())).reshape(shape)
    rows = (x64.shape[0] + 16) * U32
    val["dw"], val["db"] = (g * xh).sum(0), g.sum(0)
    tol["dw"] = rows * (g * xh).abs().sum(0) + (g.abs() * off).sum(0)
    tol["db"] = rows * g.abs().sum(0)
    return val, tol
