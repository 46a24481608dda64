"""The operators with gradients at their ends: offsets past 32 bits, more rows than a grid
has workgroups for, short sequences about where their kernel changes, two calls at once."""
import pytest

torch = pytest.importorskip("torch")

import train_ref as R  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(DEV)


def far(t, stride):
    """The rows of t, `stride` elements from one another."""
    base = torch.empty((t.shape[0] - 1) * stride + t.shape[1], dtype=t.dtype, device=DEV)
    view = base.as_strided(t.shape, (stride, 1))
    view.copy_(t)
    return view


FAR = (1 << 23) + 5          # 600 rows: five billion elements


def test_recurrence_of_rows_far_apart():
    from ssla_hip import ops
    T, c = 600, 40
    x = [far(normal(i, T, c).bfloat16(), FAR) for i in (1, 2)]
    q, s, dout, dlast = normal(3, T, c).bfloat16(), normal(4, 3, c), far(normal(5, T, c).bfloat16(), FAR), normal(6, 3, c)
    bounds = [(0, 250), (250, 250), (250, 599)]
    cu = torch.tensor([0, 250, 250, 599], dtype=torch.int32, device=DEV)
    val, tol = R.recurrence(x[0], x[1], q, bounds, s, dout, dlast)
    leaves = [t.detach().requires_grad_() for t in (x[0], x[1], q, s)]
    out, last = ops.linear_recurrence(*leaves[:3], cu_seqlens=cu, state_in=leaves[3], return_state=True)
    got = torch.autograd.grad((out, last), leaves, (dout, dlast))
    for n, t in zip(("out", "state", "dgate", "dv", "dq", "dstate_in"), (out.detach(), last.detach()) + got):
        R.check(n, t, val[n], tol[n])
    o = far(torch.full((T, c), 7.0, device=DEV).bfloat16(), FAR)
    ops.linear_recurrence(x[0], x[1], q, o, cu_seqlens=cu, state_in=s)
    R.check("out", o[:599], val["out"][:599], tol["out"][:599])
    assert (o[599] == 7).all()


def test_states_far_apart():
    """Slots of a pool past 32 bits, of sequences and of single tokens."""
    from ssla_hip import ops
    n, c = 600, 24
    pool = far(normal(7, n, c), FAR)
    was = pool.contiguous()
    slots = torch.randperm(n, generator=torch.Generator().manual_seed(8)).to(torch.int32).to(DEV)
    gate, v = normal(9, n, c), normal(10, n, c)
    val, tol = R.recurrence(gate, v, None, [(i, i + 1) for i in range(n)], was[slots.long()])
    R.check("out", ops.linear_recurrence_step(gate, v, pool, slots=slots), val["out"], tol["out"])
    R.check("state", pool[slots.long()], val["state"], tol["state"])
    for t in (1, 40):                                        # in tiles, and without
        pool.copy_(was)
        g, x = normal(11, n * t, c), normal(12, n * t, c)
        val, tol = R.recurrence(g, x, None, [(i * t, i * t + t) for i in range(n)], was[slots.long()])
        out = ops.linear_recurrence(g, x, n_seqs=n, state_in=pool, state_out=pool, slots=slots)
        R.check("out", out, val["out"], tol["out"])
        R.check("state", pool[slots.long()], val["state"], tol["state"])


def test_norm_of_rows_far_apart():
    from ssla_hip import ops
    T, c = 600, 48
    x, res, dy = (far(normal(i, T, c).bfloat16(), FAR) for i in (13, 14, 15))
    w, b = normal(16, c), normal(17, c)
    val, tol = R.layer_norm(x, res, w, b, 1e-5, dy)
    leaves = [t.detach().requires_grad_() for t in (x, res, w, b)]
    y = ops.layer_norm(leaves[0], leaves[2], leaves[3], residual=leaves[1])
    got = torch.autograd.grad(y, leaves, dy)
    R.check("y", y.detach(), val["y"], tol["y"])
    for n, k, t in zip(("dx", "dres", "dw", "db"), ("dx", "dx", "dw", "db"), got):
        R.check(n, t, val[k], tol[k])
    with torch.no_grad():
        assert ops.layer_norm(x, w, b, x, residual=res) is not None
    assert torch.equal(x, y)


@pytest.mark.parametrize("c,dtype", [(4, "f32"), (8, "bf16")])
def test_norm_of_more_rows_than_a_grid_has_workgroups_for(c, dtype):
    """2^32 threads over 256."""
    from ssla_hip import ops
    n = (1 << 24) + 77
    t = R.TYPES[dtype]
    gen = torch.Generator(device=DEV).manual_seed(18)
    x, dy = (torch.randn(n, c, generator=gen, device=DEV).to(t) for _ in range(2))
    w, b = normal(19, c), normal(20, c)
    at = torch.cat([torch.arange(100), torch.arange((1 << 24) - 50, n), torch.randperm(n)[:1000]]).to(DEV)
    val, tol = R.layer_norm(x[at], None, w, b, 1e-5, dy[at])
    leaves = [i.requires_grad_() for i in (x, w, b)]
    y = ops.layer_norm(*leaves)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    R.check("y", y.detach()[at], val["y"], tol["y"])
    R.check("dx", dx[at], val["dx"], tol["dx"])
    # a thread adds up 2^24 / (256 * 512) = 129 rows at most, eight steps join a workgroup's, and
    # parts are joined in 64 bits: 138 roundings, and some 10 of each row's product
    x64, g = x.detach().double(), dy.double()
    x64 = x64 - x64.mean(1, keepdim=True)
    x64 *= torch.rsqrt((x64 * x64).mean(1, keepdim=True) + 1e-5)
    g64, terms = g.abs().sum(0).cpu(), (g * x64).abs().sum(0).cpu()
    R.check("db", db, g.sum(0).cpu(), 160 * R.U32 * g64)
    R.check("dw", dw, (g * x64).sum(0).cpu(), 160 * R.U32 * terms)


@pytest.mark.parametrize("n,t,c,dtype", [(1, 32, 3, "f32"), (1, 33, 3, "f32"), (7, 31, 65, "bf16"), (4096, 2, 5, "f16"),
                                         (4097, 2, 5, "f16"), (2048, 3, 65, "f32"), (2049, 3, 65, "f32"),
                                         (3, 1, 20000, "bf16")])
@pytest.mark.parametrize("read", [False, True])
def test_short_sequences(n, t, c, dtype, read):
    from ssla_hip import ops
    gate, v, q = (normal(21 + i, n * t, c).to(R.TYPES[dtype]) for i in range(3))
    s, dout = normal(24, n, c), normal(25, n * t, c).to(R.TYPES[dtype])
    q = q if read else None
    val, tol = R.recurrence(gate, v, q, [(i * t, i * t + t) for i in range(n)], s, dout)
    out, last = ops.linear_recurrence(gate, v, q, n_seqs=n, state_in=s, return_state=True)
    R.check("out", out, val["out"], tol["out"])
    R.check("state", last, val["state"], tol["state"])
    leaves = [i.requires_grad_() for i in (gate, v, s)]
    out = ops.linear_recurrence(gate, v, q, n_seqs=n, state_in=s)
    for k, d in zip(("dgate", "dv", "dstate_in"), torch.autograd.grad(out, leaves, dout)):
        R.check(k, d, val[k], tol[k])


def test_two_calls_at_once():
    """On two streams, each with its own workspace: to the bits of one after the other."""
    from ssla_hip import ops
    cu = torch.tensor([0, 1, 9000, 9000, 30000], dtype=torch.int32, device=DEV)
    gate, v, q = (normal(26 + i, 30000, 192).bfloat16().requires_grad_() for i in range(3))
    w, b = normal(29, 192), normal(30, 192)
    dout = normal(31, 30000, 192).bfloat16()

    def both():
        x = ops.layer_norm(v, w, b)
        out = ops.linear_recurrence(gate, x, q, cu_seqlens=cu)
        return (out.detach(),) + torch.autograd.grad(out, (gate, v, q), dout)

    want = both()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(both())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


@pytest.mark.parametrize("dtype,c", [("f32", 48), ("bf16", 96), ("f16", 70), ("f32", 3)])
def test_sequences_that_end_where_tiles_do_and_stretches_of_none(dtype, c):
    """Boundaries at powers of two, which tiles end at; before and behind the sequences
    longer stretches of tokens that belong to none, with NaN in all they have."""
    from ssla_hip import ops
    t = R.TYPES[dtype]
    bounds = [(4096, 4608), (4608, 4672), (4672, 6784)]
    cu = torch.tensor([4096, 4608, 4672, 6784], dtype=torch.int32, device=DEV)
    T = 6784 + 4096
    gate, v, q, dout = (normal(40 + i, T, c).to(t) for i in range(4))
    for x in (gate, v, q):
        x[:4096] = float("nan")
        x[6784:] = float("nan")
    s, dlast = normal(44, 3, c), normal(45, 3, c)
    val, tol = R.recurrence(gate, v, q, bounds, s, dout, dlast)
    mine, rest = slice(4096, 6784), [slice(0, 4096), slice(6784, T)]
    kept = torch.full((T, c), 7.0, device=DEV, dtype=t)
    ops.linear_recurrence(gate, v, q, kept, cu_seqlens=cu, state_in=s)
    R.check("out", kept[mine], val["out"][mine], tol["out"][mine])
    assert all((kept[i] == 7).all() for i in rest)
    leaves = [x.requires_grad_() for x in (gate, v, q, s)]
    out, last = ops.linear_recurrence(gate, v, q, cu_seqlens=cu, state_in=s, return_state=True)
    got = torch.autograd.grad((out, last), leaves, (dout, dlast))
    R.check("state", last.detach(), val["state"], tol["state"])
    R.check("dstate_in", got[3], val["dstate_in"], tol["dstate_in"])
    for n, x in zip(("out", "dgate", "dv", "dq"), (out.detach(),) + got[:3]):
        R.check(n, x[mine], val[n][mine], tol[n][mine])
        assert all((x[i] == 0).all() for i in rest), n


@pytest.mark.parametrize("dtype,c,T", [("f32", 48, 1000), ("bf16", 96, 333), ("f16", 70, 4097), ("f32", 3, 1025)])
def test_an_infinity_in_the_last_token(dtype, c, T):
    """What a tile has behind the last token is no token: nothing of that one comes from there."""
    from ssla_hip import ops
    t = R.TYPES[dtype]
    gate, v, q, dout = (normal(50 + i, T, c).to(t) for i in range(4))
    val, tol = R.recurrence(gate, v, q, [(0, T)], None, dout)
    v[-1] = float("inf")
    gate[-1] = float("inf")                                  # an open gate
    leaves = [x.requires_grad_() for x in (gate, v, q)]
    out = ops.linear_recurrence(gate, v, q)
    dg, dv, dq = torch.autograd.grad(out, leaves, dout)
    R.check("out", out.detach()[:-1], val["out"][:-1], tol["out"][:-1])
    R.check("dq", dq[:-1], val["dq"][:-1], tol["dq"][:-1])
    assert (dg[-1] == 0).all() and not torch.isfinite(dq[-1]).any()
    gate, v = gate.detach(), v.detach()
    v[-1] = 0
    val, tol = R.recurrence(gate.double().clamp(max=80), v, q, [(0, T)], None, dout)
    R.check("dv", dv, val["dv"], tol["dv"])
    R.check("dgate", dg[:-1], val["dgate"][:-1], tol["dgate"][:-1])


@pytest.mark.parametrize("n,c,dtype", [(66000, 5, "f32"), (700, 40, "bf16")])
def test_more_sequences_than_a_workgroup_has_threads(n, c, dtype):
    """Boundaries that are searched for in one step more, and two; most sequences are empty."""
    from ssla_hip import ops
    lens = [2 * (i % 6 == 0) + (i % 35 == 34) for i in range(n)]
    first = [0]
    for k in lens:
        first.append(first[-1] + k)
    cu = torch.tensor(first, dtype=torch.int32, device=DEV)
    gate, v, q, dout = (normal(60 + i, first[-1], c).to(R.TYPES[dtype]) for i in range(4))
    s, dlast = normal(64, n, c), normal(65, n, c)
    val, tol = R.recurrence(gate, v, q, list(zip(first[:-1], first[1:])), s, dout, dlast)
    leaves = [x.requires_grad_() for x in (gate, v, q, s)]
    out, last = ops.linear_recurrence(gate, v, q, cu_seqlens=cu, state_in=s, return_state=True)
    got = torch.autograd.grad((out, last), leaves, (dout, dlast))
    for k, x in zip(("out", "state", "dgate", "dv", "dq", "dstate_in"), (out.detach(), last.detach()) + got):
        R.check(k, x, val[k], tol[k])
