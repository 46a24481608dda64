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
