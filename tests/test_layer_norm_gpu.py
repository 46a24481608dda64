"""Layer norm and its gradients against the plain 64-bit form."""
import pytest

torch = pytest.importorskip("torch")

import train_ref as R  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(DEV)


def tensors(rows, c, dtype, residual, affine, wide=False, seed=1):
    t = R.TYPES[dtype]
    x = (normal(seed, rows, c) * 1.7 + normal(seed + 1, c)).to(t)
    res = normal(seed + 2, rows, c).to(t) if residual else None
    wt = torch.float32 if wide else t
    w = (1 + 0.2 * normal(seed + 3, c)).to(wt) if affine else None
    b = (0.2 * normal(seed + 4, c)).to(wt) if affine else None
    return x, res, w, b, normal(seed + 5, rows, c).to(t)


# rows, channels: one value, odd ones, those about a wave's and a workgroup's reach, wide ones
SIZES = [(1, 1), (5, 1), (3, 2), (70, 7), (33, 24), (1, 48), (320, 48), (257, 96), (100, 97), (9, 255), (64, 256),
         (17, 511), (40, 513), (30, 1000), (21, 1024), (12, 1025), (10, 2048), (7, 2049), (6, 4096), (5, 5003),
         (4, 8192), (3, 8200), (3, 16384), (2, 20001), (2, 40000)]


def grads(x, res, w, b, dy, eps=1e-5):
    from ssla_hip import ops
    leaves = {n: t.detach().requires_grad_() for n, t in (("dx", x), ("dres", res), ("dw", w), ("db", b))
              if t is not None}
    y = ops.layer_norm(leaves["dx"], leaves.get("dw"), leaves.get("db"), eps=eps, residual=leaves.get("dres"))
    got = torch.autograd.grad(y, list(leaves.values()), dy)
    return dict(zip(leaves, got), y=y.detach())


def compare(got, val, tol):
    for n in got:
        k = "dx" if n == "dres" else n
        R.check(n, got[n], val[k], tol[k])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,c", SIZES)
@pytest.mark.parametrize("residual", [False, True])
def test_rows(dtype, rows, c, residual):
    from ssla_hip import ops
    wide = (rows + c) % 2 == 0
    x, res, w, b, dy = tensors(rows, c, dtype, residual, rows % 3 != 1, wide)
    val, tol = R.layer_norm(x, res, w, b, 1e-5, dy)
    R.check("y", ops.layer_norm(x, w, b, residual=res), val["y"], tol["y"])
    compare(grads(x, res, w, b, dy), val, tol)


@pytest.mark.parametrize("rows,c", [(5000, 48), (3001, 96), (2100, 130), (1027, 512), (700, 2048), (600, 3000)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_rows(rows, c, dtype):
    """Sums over rows that many workgroups share."""
    x, res, w, b, dy = tensors(rows, c, dtype, True, True)
    val, tol = R.layer_norm(x, res, w, b, 1e-5, dy)
    compare(grads(x, res, w, b, dy), val, tol)


def test_gradients_agree_with_differences():
    """A central difference of a step of 1e-4 of the 64-bit form is off by the third
    derivative's 1e-8."""
    x, res, w, b, dy = tensors(40, 50, "f32", True, True)
    got = grads(x, res, w, b, dy)
    args = [x, res, w, b]
    for i, n in enumerate(("dx", "dres", "dw", "db")):
        d = torch.randn(args[i].shape, generator=torch.Generator().manual_seed(30 + i), dtype=torch.float64)
        f = []
        for e in (1e-4, -1e-4):
            a = [R.f64(t) for t in args]
            a[i] = a[i] + e * d
            f.append((R.layer_norm(*a, 1e-5)[0]["y"] * R.f64(dy)).sum())
        want, along = (f[0] - f[1]).item() / 2e-4, (R.f64(got[n]) * d).sum().item()
        assert abs(along - want) <= 1e-5 * (R.f64(got[n]) * d).abs().sum().item(), n


@pytest.mark.parametrize("c", [24, 96, 1000, 9000])
def test_a_mean_far_from_zero_and_a_spread_of_none(c):
    x = (normal(1, 20, c) + 1e5)
    x[3] = 12345.678
    x[4] = 0.0
    dy = normal(2, 20, c)
    val, tol = R.layer_norm(x, None, None, None, 1e-5, dy)
    got = grads(x, None, None, None, dy)
    compare(got, val, tol)
    assert (got["y"][4] == 0).all()


@pytest.mark.parametrize("c", [48, 1000])
def test_finite_values_of_any_size(c):
    from ssla_hip import ops
    for scale in (1e-30, 1e-15, 1e15, 3e37):
        x = (normal(3, 9, c) * scale).clamp(-3e38, 3e38)
        val, tol = R.layer_norm(x, None, None, None, 0.0)
        R.check("y", ops.layer_norm(x, eps=0.0), val["y"], tol["y"])


def test_infinities_and_nans_stay_in_their_row():
    for c in (24, 96, 700, 5000):
        x, res, w, b, dy = tensors(50, c, "f32", True, True)
        want = grads(x, res, w, b, dy)
        x[7, 3], x[20, c - 1], res[30, 5], dy[41, 0] = float("nan"), float("inf"), float("-inf"), float("nan")
        got = grads(x, res, w, b, dy)
        ok = torch.ones(50, dtype=torch.bool, device=DEV)
        ok[[7, 20, 30]] = False
        assert torch.equal(got["y"][ok], want["y"][ok]) and not torch.isfinite(got["y"][~ok]).any()
        ok[41] = False
        assert torch.equal(got["dx"][ok], want["dx"][ok]) and not torch.isfinite(got["dx"][~ok]).any()


@pytest.mark.parametrize("dtype,c", [("f32", 5), ("f32", 96), ("bf16", 64), ("bf16", 101), ("f16", 999)])
def test_strides_addresses_and_places(dtype, c):
    """Rows at odd strides and addresses; out in x's and in residual's place, in rows of a
    larger tensor whose other columns stay; more dimensions."""
    from ssla_hip import ops
    base = normal(4, 37 * (2 * c + 3) + 1).to(R.TYPES[dtype])
    m = base[1:].view(37, 2 * c + 3)
    was = m.clone()
    x, res = m[:, 1:1 + c], m[:, c + 2:2 * c + 2]
    w, b = (normal(5, c + 1).to(x.dtype)[1:], normal(6, c + 1).to(x.dtype)[1:])
    val, tol = R.layer_norm(x, res, w, b, 1e-3)
    R.check("y", ops.layer_norm(x, w, b, eps=1e-3, residual=res), val["y"], tol["y"])
    ops.layer_norm(x, w, b, x, eps=1e-3, residual=res)
    R.check("y", x, val["y"], tol["y"])
    x.copy_(was[:, 1:1 + c])
    ops.layer_norm(x, w, b, res, eps=1e-3, residual=res)
    R.check("y", res, val["y"], tol["y"])
    res.copy_(was[:, c + 2:2 * c + 2])
    assert torch.equal(m, was)
    y = torch.empty(6, 1, 7, c, device=DEV, dtype=x.dtype)
    x4 = base[:6 * 7 * c].view(6, 1, 7, c)
    ops.layer_norm(x4, w, b, y, eps=1e-3)
    val, tol = R.layer_norm(x4, None, w, b, 1e-3)
    R.check("y", y, val["y"], tol["y"])
    one = base[:c]
    val, tol = R.layer_norm(one[None], None, w, b, 1e-3)
    R.check("y", ops.layer_norm(one, w, b, eps=1e-3)[None], val["y"], tol["y"])


def test_gradients_through_shapes():
    """More dimensions, rows at a stride, one input as x and residual, an expanded
    gradient, a transposed one, a weight that alone wants one."""
    from ssla_hip import ops
    x, _, w, b, _ = tensors(30, 40, "f32", False, True)
    val, tol = R.layer_norm(x, None, w, b, 1e-5, torch.ones(30, 40))
    leaf = x.clone().requires_grad_()
    ops.layer_norm(leaf.view(2, 3, 5, 40), w, b).sum().backward()
    R.check("dx", leaf.grad, val["dx"], tol["dx"])
    dy = normal(9, 40, 30).t()
    val, tol = R.layer_norm(x, None, w, b, 1e-5, dy)
    leaf, lw = x.clone().requires_grad_(), w.clone().requires_grad_()
    ops.layer_norm(leaf, lw, b).backward(dy)
    R.check("dx", leaf.grad, val["dx"], tol["dx"])
    R.check("dw", lw.grad, val["dw"], tol["dw"])
    for i, n in ((1, "dw"), (2, "db")):
        ts = [t.clone().requires_grad_(i == j) for j, t in enumerate((x, w, b))]
        ops.layer_norm(*ts).backward(dy)
        R.check(n, ts[i].grad, val[n], tol[n])
        assert all(t.grad is None for j, t in enumerate(ts) if j != i)
    leaf = x.clone().requires_grad_()
    ops.layer_norm(leaf, w, b, residual=leaf).backward(dy)
    val, tol = R.layer_norm(x, x, w, b, 1e-5, dy)
    R.check("dx", leaf.grad, 2 * val["dx"], 2 * tol["dx"] + 3 * R.U32 * val["dx"].abs())


def test_no_rows_and_no_channels():
    from ssla_hip import ops
    for shape in ((0, 8), (4, 0), (2, 0, 5)):
        x = torch.empty(shape, device=DEV).requires_grad_()
        w = torch.ones(shape[-1], device=DEV).requires_grad_()
        y = ops.layer_norm(x, w)
        assert y.shape == shape
        y.sum().backward()
        assert x.grad.shape == shape and (w.grad == 0).all()


@pytest.mark.parametrize("rows,c", [(5, 40), (4000, 96), (300, 3000), (20, 30000)])
def test_reruns_streams_and_captures(rows, c):
    x, res, w, b, dy = (t.clone() for t in tensors(rows, c, "bf16", True, True))
    first = grads(x, res, w, b, dy)
    again = grads(x, res, w, b, dy)
    assert all(torch.equal(first[n], again[n]) for n in first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = grads(x, res, w, b, dy)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(first[n], other[n]) for n in first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = grads(x, res, w, b, dy)
    for i in range(4):
        x.add_(0.5)
        want = grads(x, res, w, b, dy)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(want[n], got[n]) for n in want), i
