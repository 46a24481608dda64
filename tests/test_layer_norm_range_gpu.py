"""Layer norm of rows whose spread is small: eps of zero or nearly, in every type and form of
the kernels, with gradients."""
import pytest

torch = pytest.importorskip("torch")

import train_ref as R  # noqa: E402
from test_layer_norm_gpu import grads, normal  # noqa: E402

pytestmark = pytest.mark.gpu


def allowed(x, res, w, b, eps, dy):
    """R.layer_norm's values and errors, and what counts where spreads are small: 2^-16 s - mean
    and the mean's second part are fp32 numbers, 2^-149 apart at least, so that each is off by
    up to 2^-150, or 2^-134 of s; as an error of the normed rows, 2^-133 / sqrt(var + eps)."""
    val, tol = R.layer_norm(x, res, w, b, eps, dy)
    s = R.f64(x) + (0 if res is None else R.f64(res))
    d = s - s.mean(1, keepdim=True)
    r = 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + eps)
    off, xh, g = 2.0 ** -133 * r, d * r, R.f64(dy)
    W = 1.0 if w is None else R.f64(w)
    u = g * W
    tol["y"] = tol["y"] + off * (W.abs() if w is not None else 1.0)
    tol["dx"] = tol["dx"] + r * off * ((u * xh).mean(1, keepdim=True).abs() + xh.abs() * u.abs().mean(1, keepdim=True))
    tol["dw"] = tol["dw"] + (g.abs() * off).sum(0)
    return val, tol


# a value a lane; lanes of a wave, with and without a ragged end; a workgroup; strides
@pytest.mark.parametrize("c", [7, 48, 1000, 1021, 5003, 20000])
@pytest.mark.parametrize("dtype,spread,eps", [
    ("bf16", s, e) for s, e in ((1e-33, 0.0), (1e-30, 0.0), (1e-24, 0.0), (1e-23, 0.0), (1e-22, 0.0), (1e-20, 0.0),
                                (1e-19, 0.0), (1e-15, 0.0), (1e-20, 2.0 ** -130), (1e-30, 2.0 ** -130), (1e-13, 2.0 ** -80),
                                (1e-20, 2.0 ** -60), (1e-10, 2.0 ** -61), (1e-25, 1e-5))] + [
    ("f16", 1e-7, 0.0), ("f16", 1e-5, 0.0), ("f32", 1e-33, 0.0), ("f32", 1e-24, 0.0), ("f32", 1e-20, 2.0 ** -130)])
@pytest.mark.parametrize("residual", [False, True])
def test_small_spreads(dtype, spread, eps, c, residual):
    rows = 9
    x = (normal(41, rows, c) * spread + (normal(42, rows, 1) * spread if dtype != "f16" else 0)).to(R.TYPES[dtype])
    x[4] = normal(43, c).to(x.dtype)                       # beside one of an ordinary row's
    x[5, c // 2] = 3.0                                     # and one value that is
    if dtype == "f16":
        x[:4, 0] = 6e-8                                    # (rows of nothing but zeros have no norm)
    res = (normal(44, rows, c) * spread).to(x.dtype) if residual else None
    w, b = (1 + 0.2 * normal(45, c)).to(x.dtype), (0.2 * normal(46, c)).to(x.dtype)
    dy = normal(47, rows, c).to(x.dtype)
    eps = float(torch.tensor(eps))
    val, tol = allowed(x, res, w, b, eps, dy)
    ok = val["dx"].abs().amax(1) < torch.finfo(x.dtype).max / 4      # a gradient may be past the type's largest
    got = grads(x, res, w, b, dy, eps)
    for n in ("y", "dw", "db"):
        R.check(n, got[n], val[n], tol[n])
    assert ok.any()
    R.check("dx", got["dx"][ok.to(x.device)], val["dx"][ok], tol["dx"][ok])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("c", [8, 96, 2048, 20000])
def test_the_smallest_spread(dtype, c):
    """A deviation of 2^-111 without eps, in powers of two alone: every value is exact.  A row
    of a smaller one is not finite, and the others do not see it."""
    from ssla_hip import ops
    sign = torch.ones(c, device="cuda")
    sign[1::2] = -1.0
    x = (sign * 2.0 ** -111).expand(5, c).to(R.TYPES[dtype]).contiguous()
    x[2] = 0.0
    dy = torch.zeros_like(x)
    dy[:, 0] = 2.0
    norm = ops.layer_norm(x, eps=0.0), ops.group_norm(x, 1, eps=0.0)
    got = grads(x, None, None, None, dy, 0.0)
    rows = [0, 1, 3, 4]
    for y in norm + (got["y"],):
        assert (y[rows] == sign).all() and not torch.isfinite(y[2]).any()
    # dx = 2^111 (dy - 2 / c - sign 2 / c): nothing where sign is -1
    want = (2.0 ** 111 * (dy.double() - 2.0 / c - sign.double() * (2.0 / c)))[rows]
    off = 2.0 ** 111 * 100 * R.U32 * (dy.double() + 4.0 / c)[rows] + R.half_step(x.dtype) * want.abs()
    assert ((got["dx"][rows].double() - want).abs() <= off).all()
