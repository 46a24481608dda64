"""Group norm with an activation, channels last, against its 64-bit form."""
import pytest

torch = pytest.importorskip("torch")

import seq_ref as R  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ops():
    from ssla_hip import ops as o
    return o


def make(shape, dtype, seed=0):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    c = shape[-1]
    x = (rnd(*shape) * (0.5 + rnd(c).abs()) + rnd(c)).to(dtype)
    return x, (1 + 0.3 * rnd(c)).to(dtype), (0.3 * rnd(c)).to(dtype), rnd(*shape).to(dtype)


SHAPES = [((1, 9000, 60), 2), ((2, 24, 606), 1), ((2, 200, 128), 1), ((2, 1500, 9), 1),
          ((130, 30, 256), 4),
          ((600, 100, 24), 1), ((3, 16384), 8), ((40, 65536), 16), ((1, 2000, 24), 3),
          ((40, 320, 48), 8), ((290, 70, 33), 11), ((1, 1, 1), 1), ((3, 7, 24), 4),
          ((2, 5, 3, 24), 24), ((1, 20, 16, 48), 8), ((5, 33), 3), ((700, 96), 2),
          ((129, 2048), 16), ((2, 300, 40), 1), ((2, 1000, 30), 5), ((1, 6000, 48), 16),
          ((4, 2500, 96), 8), ((3, 64, 1000), 8), ((1, 30000, 8), 2), ((2, 4, 4096), 32),
          ((1, 2, 20000), 4), ((20, 1, 7), 7)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape,groups", SHAPES, ids=str)
def test_shapes(dtype, shape, groups):
    t = R.TYPES[dtype]
    x, w, b, gate = make(shape, t, 1)
    R.check_group_norm(ops().group_norm(x, groups, w, b, act="silu"),
                       R.group_norm(x, groups, w, b, 1e-5, "silu"), t)
    R.check_group_norm(ops().group_norm(x, groups, w, b, act="silu", gate=gate),
                       R.group_norm(x, groups, w, b, 1e-5, "silu", gate), t)


@pytest.mark.parametrize("shape,groups", [((5, 96), 4), ((2, 50, 24), 3), ((2, 9000, 24), 3)], ids=str)
@pytest.mark.parametrize("act", ["none", "silu", "sigmoid", "relu", None])
@pytest.mark.parametrize("affine", ["both", "weight", "bias", "no"])
def test_activations_and_affine(shape, groups, act, affine):
    x, w, b, gate = make(shape, torch.float32, 2)
    w, b = (w if affine in ("both", "weight") else None), (b if affine in ("both", "bias") else None)
    for gt in (None, gate):
        R.check_group_norm(ops().group_norm(x, groups, w, b, eps=1e-3, act=act, gate=gt),
                           R.group_norm(x, groups, w, b, 1e-3, act, gt), torch.float32)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape,groups", [((40, 48), 4), ((3, 40, 48), 4), ((2, 9000, 48), 4)], ids=str)
@pytest.mark.parametrize("layout", ["padded", "odd", "item_gap"])
def test_strides(dtype, shape, groups, layout):
    t, c = R.TYPES[dtype], shape[-1]
    x, w, b, gate = make(shape, t, 3)

    def place(v):
        if layout == "item_gap":
            buf = torch.full((shape[0] * 2,) + shape[1:], 9.0, dtype=t, device=DEV)
            y = buf[::2]
        else:
            extra, off = (8, 0) if layout == "padded" else (3, 1)
            buf = torch.full(shape[:-1] + (c + extra,), 9.0, dtype=t, device=DEV)
            y = buf[..., off:off + c]
        y.copy_(v)
        return buf, y

    want = R.group_norm(x, groups, w, b, 1e-5, "silu", gate)
    (_, xs), (_, gs), (ob, os) = place(x), place(gate), place(torch.zeros_like(x))
    mark = torch.ones_like(ob, dtype=torch.bool)
    if layout == "item_gap":
        mark[::2] = False
    else:
        mark[..., (0 if layout == "padded" else 1):][..., :c] = False
    got = ops().group_norm(xs, groups, w, b, os, act="silu", gate=gs)
    assert got is os
    R.check_group_norm(os, want, t)
    assert (ob[mark] == 9).all()


@pytest.mark.parametrize("shape", [(30, 64), (2, 100, 64), (2, 9000, 64)], ids=str)
def test_in_place(shape):
    x, w, b, gate = make(shape, torch.bfloat16, 4)
    want = ops().group_norm(x, 4, w, b, act="silu", gate=gate)
    y = x.clone()
    assert torch.equal(ops().group_norm(y, 4, w, b, y, act="silu", gate=gate), want)
    z = gate.clone()
    assert torch.equal(ops().group_norm(x, 4, w, b, z, act="silu", gate=z), want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(6, 64), (2, 200, 64), (1, 20000, 64)], ids=str)
@pytest.mark.parametrize("kind", ["offset", "outlier", "constant", "tiny", "large"])
def test_values(dtype, shape, kind):
    """Means far from zero, one value far from the others, no spread at all."""
    t = R.TYPES[dtype]
    x, w, b, _ = make(shape, t, 5)
    x = x.float()
    if kind == "offset":
        x = x + 3000.0
    elif kind == "outlier":
        x[0].view(-1)[0] = 1e5
    elif kind == "constant":
        x = torch.full_like(x, 1.7)
    elif kind == "tiny":
        x = x * 1e-12
    elif kind == "large":
        x = x * 1e12
    x = x.to(t)
    R.check_group_norm(ops().group_norm(x, 4, w, b), R.group_norm(x, 4, w, b, 1e-5, "none"), t)


@pytest.mark.parametrize("shape", [(6, 64), (3, 200, 64), (3, 20000, 64)], ids=str)
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_non_finite_values_stay_in_their_group(shape, value):
    x, w, b, _ = make(shape, torch.float32, 6)
    want, off = R.group_norm(x, 4, w, b, 1e-5, "silu")
    x[1].view(-1)[17] = value                    # channel 17 of 64, group 1 of 4
    got = ops().group_norm(x, 4, w, b, act="silu").cpu()
    bad = torch.zeros(shape, dtype=torch.bool)
    bad[1, ..., 16:32] = True
    assert torch.isnan(got[bad]).all()
    R.check_group_norm(torch.where(bad, 0.0, got), (torch.where(bad, 0.0, want), off), torch.float32)


def test_empty():
    for shape in ((0, 5, 8), (3, 0, 8), (0, 8)):
        assert ops().group_norm(torch.empty(shape, device=DEV), 2).shape == shape


def test_offsets_past_32_bits():
    far = 2 ** 31 + 64
    mem = torch.empty(far + 64, dtype=torch.bfloat16, device=DEV)
    x, w, b, _ = make((2, 64), torch.bfloat16, 7)
    y = mem.as_strided((2, 64), (far, 1))
    y.copy_(x)
    R.check_group_norm(ops().group_norm(y, 4, w, b, y, act="silu"),
                       R.group_norm(x, 4, w, b, 1e-5, "silu"), torch.bfloat16)


@pytest.mark.parametrize("shape", [(50, 512), (2, 100, 48), (2, 15000, 48)], ids=str)
def test_graphs_and_reruns(shape):
    x, w, b, _ = make(shape, torch.float32, 8)
    out = torch.empty_like(x)
    ops().group_norm(x, 4, w, b, out, act="silu")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops().group_norm(x, 4, w, b, out, act="silu")
    for i in range(3):
        x.copy_(make(shape, torch.float32, 9 + i)[0])
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops().group_norm(x, 4, w, b, act="silu"))


def test_streams():
    sets = [make((2, 12000, 48), torch.float32, 20 + i) for i in range(2)]
    want = [ops().group_norm(x, 8, w, b) for x, w, b, _ in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        got = []
        for (x, w, b, _), st in zip(sets, streams):
            with torch.cuda.stream(st):
                got.append(ops().group_norm(x, 8, w, b))
        torch.cuda.synchronize()
        for a, c in zip(want, got):
            assert torch.equal(a, c)
