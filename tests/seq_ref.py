"""Plain 64-bit forms of the sequence operators and the error their kernels may
have, from counts of roundings."""
import torch

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half a step of the type's subnormal numbers (fp32's normal ones for the
    wider types: products below them may be flushed)."""
    return 2.0 ** -25 if dtype == torch.float16 else 1e-36


def linear_attention(q, k, v, g, lens, scale, state=None):
    """Token by token in 64 bits on the CPU.  Returns (out, |out| with every
    term's magnitude, states, their magnitudes)."""
    q, k, v, g = (t.detach().cpu().double() for t in (q, k, v, g))
    T, H, dv = v.shape
    rep = H // q.shape[1]
    q, k = q.repeat_interleave(rep, 1), k.repeat_interleave(rep, 1)
    if g.dim() == 1:
        g = g.expand(T, H)
    a = torch.exp(g)
    out, mag = torch.zeros(T, H, dv, dtype=torch.float64), torch.zeros(T, H, dv, dtype=torch.float64)
    S_all, M_all = [], []
    t0 = 0
    for s, n in enumerate(lens):
        S = torch.zeros(H, q.shape[2], dv, dtype=torch.float64) if state is None \
            else state[s].detach().cpu().double().clone()
        M = S.abs()
        for t in range(t0, t0 + n):
            kv = k[t][:, :, None] * v[t][:, None, :]
            S = a[t][:, None, None] * S + kv
            M = a[t][:, None, None] * M + kv.abs()
            out[t] = scale * (q[t][:, :, None] * S).sum(1)
            mag[t] = abs(scale) * (q[t].abs()[:, :, None] * M).sum(1)
        t0 += n
        S_all.append(S)
        M_all.append(M)
    stack = (lambda x: torch.stack(x) if x else torch.zeros(0, H, q.shape[2], dv, dtype=torch.float64))
    return out, mag, stack(S_all), stack(M_all)


def roundings(dk, longest):
    """fp32 roundings a term of out can go through: the products and sums of q.k
    or of q with the state (dk), of a chunk (64) and of the states of the chunks
    before it (three a chunk); and the error of the decays: the exponential's
    argument, which matters down to exp(-104), is off by half a step, for each
    of the chunks' factors a term takes, and each exponential by two."""
    chunks = longest // 32 + 1
    return dk + 64 + 5 * chunks + 2 * 104 + 16


def check_linear_attention(out, state, ref, dtype, dk, longest):
    r_out, mag, r_state, smag = ref
    n = roundings(dk, longest) * U32
    # 16-bit types: P and the state's copy in two bf16 terms (2^-16 each, of
    # disjoint parts of a sum); fp16 inputs leave out one more product of lower
    # terms (2^-16)
    split = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -15}[dtype]
    tol = (n + split) * mag + half_step(dtype) * (1 + 2.0 ** -8) * r_out.abs() + tiny(dtype)
    err = (out.detach().cpu().double() - r_out).abs()
    assert torch.isfinite(out).all()
    worst = (err / tol).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"out: {worst:.3g} of the tolerance"
    if state is not None:
        # three bf16 terms: 2^-24 and, in fp16, as much again
        err = (state.detach().cpu().double() - r_state).abs()
        tol = (n + 2 * U32) * smag + 1e-36
        worst = (err / tol).max().item() if err.numel() else 0.0
        assert worst <= 1.0, f"state: {worst:.3g} of the tolerance"


def act64(x, act):
    if act == "silu":
        return x * torch.sigmoid(x)
    if act == "sigmoid":
        return torch.sigmoid(x)
    return torch.relu(x) if act == "relu" else x


def group_norm(x, groups, w, b, eps, act, gate=None):
    """In 64 bits on the CPU, and the error an fp32 kernel may have: x - mean, the
    mean being a merge of at most 32 levels, the square root of the variance
    (as far off), the weight, the bias and the activation (slope at most 1.1, the
    sigmoid's at most 1/4; its own exponential and division a few steps)."""
    shape = x.shape
    x64 = x.detach().cpu().double().reshape(shape[0], -1, groups, shape[-1] // groups)
    n = x64.shape[1] * x64.shape[3]
    mean = x64.mean((1, 3), keepdim=True)
    var = ((x64 - mean) ** 2).sum((1, 3), keepdim=True) / n
    rstd = 1.0 / torch.sqrt(var + eps)
    level = 32 * U32
    off = level * (x64.abs() + x64.abs().mean((1, 3), keepdim=True)) * rstd
    y = (x64 - mean) * rstd
    off = off + 2 * level * y.abs()
    # what an error of the mean adds to the variance
    off = off + y.abs() * (level * x64.abs().mean((1, 3), keepdim=True) * rstd) ** 2
    y, off = y.reshape(shape), off.reshape(shape)
    if w is not None:
        y, off = y * w.detach().cpu().double(), off * w.detach().cpu().double().abs()
    if b is not None:
        b = b.detach().cpu().double()
        y, off = y + b, off + U32 * (y.abs() + b.abs())
    if gate is None:
        out = act64(y, act)
        off = 1.1 * off + 8 * U32 * (1.0 + out.abs())
    else:
        s = act64(gate.detach().cpu().double(), act)
        out = y * s
        off = off * s.abs() + y.abs() * 8 * U32 * (1.0 + s.abs())
    return out, off


def check_group_norm(out, ref, dtype):
    want, off = ref
    tol = 1.01 * off + half_step(dtype) * (1 + 2.0 ** -8) * want.abs() + tiny(dtype)
    err = (out.detach().cpu().double() - want).abs()
    assert torch.isfinite(out).all()
    worst = (err / tol).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3g} of the tolerance"
