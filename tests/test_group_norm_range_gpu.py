"""Group norm of values up to the type's largest and of means far from zero: every
form of the kernel gives what the 64-bit form gives."""
import pytest

torch = pytest.importorskip("torch")

import seq_ref as R  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"
# groups in lanes of a wave; a workgroup a group, of 256 and 1024 threads; whole rows
# in one workgroup of 256 and 1024 threads; two passes
SHAPES = [((6, 64), 4), ((3, 2048), 2), ((2, 5, 3, 30), 3), ((1, 320, 48), 8), ((20, 300, 40), 5),
          ((20, 300, 12), 12), ((10, 300, 24), 24), ((1, 64, 1000), 8), ((1, 20000, 64), 4), ((2, 9000, 60), 4)]


def answer(x, groups, w, b, eps, terms):
    """In 64 bits, and the error that is allowed: sums of `terms` additions in 64
    bits; hi and lo (2^-48 of the mean); the variance by a difference of means of
    squares; then seven fp32 roundings of the two summands and their sum.  The
    kernels round two numbers, 2^-16 x - hi and lo, to fp32, whose values are 2^-149
    apart at least: each is off by up to 2^-150, or 2^-134 of x, which counts where
    eps is 0 and the spread is below 2^-100."""
    U32, U64 = 2.0 ** -24, 2.0 ** -53
    x64 = x.cpu().double().reshape(x.shape[0], -1, groups, x.shape[-1] // groups)
    mean = x64.mean((1, 3), keepdim=True)
    var = ((x64 - mean) ** 2).mean((1, 3), keepdim=True)
    rstd = 1.0 / torch.sqrt(var + eps)
    size = x64.abs().mean((1, 3), keepdim=True)
    y = (x64 - mean) * rstd
    far = ((terms * U64 + 2.0 ** -48) * size + 2 * 2.0 ** -134) * rstd
    off = far + y.abs() * (5 * U32 + terms * U64 * ((x64 ** 2).mean((1, 3), keepdim=True) * rstd ** 2 + 1.0))
    y, off, low = y.reshape(x.shape), off.reshape(x.shape), (2.0 ** -24 * size * rstd).expand(x64.shape).reshape(x.shape)
    w, b = w.cpu().double(), b.cpu().double()
    off = off * w.abs() + 2 * U32 * ((y * w).abs() + b.abs() + low * w.abs())
    return y * w + b, off


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape,groups", SHAPES, ids=str)
@pytest.mark.parametrize("kind", ["spread", "most", "ends", "far", "far_and_large", "tiny"])
def test_range(dtype, shape, groups, kind):
    t = R.TYPES[dtype]
    top = torch.finfo(t).max
    gen = torch.Generator(device=DEV)
    gen.manual_seed(60)
    x = torch.randn(shape, generator=gen, device=DEV)
    w = 1 + 0.3 * torch.randn(shape[-1], generator=gen, device=DEV)
    b = 0.3 * torch.randn(shape[-1], generator=gen, device=DEV)
    half = 1.0 if dtype != "f16" else 2.0 ** -12      # of 1e20 and 1e36 in fp16's range: 16, 244
    if kind == "spread":
        x = x * (1e20 if half == 1.0 else 1e3)
    elif kind == "most":                               # a plain fp32 sum of 1000 passes the largest value
        x = top / 64 * (1.0 + 0.1 * x.clamp(-3, 3))
    elif kind == "ends":
        x = torch.where(x < 0, -top, top)
    elif kind == "far":                                # what the type holds of a mean 10^6 deviations away
        x = x + (1e6 if dtype == "f32" else 64.0)
    elif kind == "far_and_large":
        x = (x + (1e6 if dtype == "f32" else 64.0)) * (1e25 if half == 1.0 else 100.0)
    else:
        x = x * 1e-30 if half == 1.0 else x * 1e-3
    x, w, b = x.to(t), w.to(t), b.to(t)
    assert torch.isfinite(x).all()
    from ssla_hip import ops
    got = ops.group_norm(x, groups, w, b, eps=1e-5)
    assert torch.isfinite(got).all()
    want, off = answer(x, groups, w, b, 1e-5, 64)
    tol = off + R.half_step(t) * (1 + 2.0 ** -8) * want.abs() + R.tiny(t)
    worst = ((got.cpu().double() - want).abs() / tol).max().item()
    assert worst <= 1.0, f"{worst:.3g} of the tolerance"


@pytest.mark.parametrize("shape,groups", SHAPES, ids=str)
def test_small_spreads_without_eps(shape, groups):
    """eps = 0: the variance of values of 1e-30 is below fp32's smallest."""
    from ssla_hip import ops
    x = torch.randn(shape, generator=torch.Generator().manual_seed(61)).to(DEV) * 1e-30
    w = torch.ones(shape[-1], device=DEV)
    want, off = answer(x, groups, w, 0 * w, 0.0, 64)
    got = ops.group_norm(x, groups, w, eps=0.0)
    assert ((got.cpu().double() - want).abs() / (off + 1e-36)).max() <= 1.0


@pytest.mark.parametrize("shape,groups", SHAPES, ids=str)
def test_an_infinite_eps_leaves_the_bias(shape, groups):
    from ssla_hip import ops
    x, b = torch.randn(shape, device=DEV), torch.randn(shape[-1], device=DEV)
    assert torch.equal(ops.group_norm(x, groups, None, b, eps=float("inf")), b.expand(shape))
