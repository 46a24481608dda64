"""The gated linear recurrence, its gradients and its single tokens against the plain
64-bit form."""
import pytest

torch = pytest.importorskip("torch")

import train_ref as R  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rows(n, c, dtype, seed, fused=True, read=True):
    """gate, v, q: parts of one projection's rows, or tensors of their own."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, 3 * c, generator=g)
    x[:, :c] = 1.5 * x[:, :c] + 2.0
    x = x.to(R.TYPES[dtype]).to(DEV)
    parts = x.split(c, 1)
    if not fused:
        parts = [p.contiguous() for p in parts]
    return parts[0], parts[1], parts[2] if read else None


def bounds_of(cu, total):
    cu = [min(max(c, 0), total) for c in cu]
    return list(zip(cu[:-1], cu[1:]))


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(DEV)


def run(gate, v, q, cu, state_in=None, **kw):
    from ssla_hip import ops
    return ops.linear_recurrence(gate, v, q, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=DEV),
                                 state_in=state_in, **kw)


# sequences: one token; a ragged handful with empty ones at both ends and between; many of
# a few tokens; lengths about powers of two; one of several tiles; long and short in turn
LENGTHS = {"one": [1], "ragged": [0, 5, 1, 0, 0, 17, 64, 0, 3, 0], "short": [i % 5 for i in range(150)],
           "powers": [63, 64, 65, 127, 128, 129, 1, 2], "long": [1700], "mixed": [700, 1, 2, 900, 0, 3, 511]}
CASES = [(d, c, name, read) for d in ("f32", "bf16", "f16") for c, name, read in (
    (1, "ragged", True), (3, "mixed", False), (7, "powers", True), (8, "one", True), (24, "long", True),
    (48, "short", True), (96, "ragged", False), (97, "mixed", True), (130, "powers", False), (257, "short", True))]


@pytest.mark.parametrize("dtype,c,name,read", CASES)
@pytest.mark.parametrize("states", [False, True])
def test_sequences(dtype, c, name, read, states):
    lens = LENGTHS[name]
    cu = [sum(lens[:i]) for i in range(len(lens) + 1)]
    gate, v, q = rows(cu[-1], c, dtype, 1, states, read)
    s = normal(2, len(lens), c) if states else None
    val, tol = R.recurrence(gate, v, q, bounds_of(cu, cu[-1]), s)
    out, last = run(gate, v, q, cu, s, return_state=True)
    R.check("out", out, val["out"], tol["out"])
    R.check("state", last, val["state"], tol["state"])


def gradients(gate, v, q, cu, s, dout, dstate):
    leaves = [t.detach().requires_grad_() for t in (gate, v, q, s) if t is not None]
    left = list(leaves)
    a, b = left.pop(0), left.pop(0)
    p = left.pop(0) if q is not None else None
    i = left.pop(0) if s is not None else None
    got = run(a, b, p, cu, i, return_state=True)
    which = [(t, d) for t, d in zip(got, (dout, dstate)) if d is not None]
    grads = torch.autograd.grad([t for t, _ in which], leaves, [d for _, d in which])
    names = ["dgate", "dv"] + ["dq"] * (q is not None) + ["dstate_in"] * (s is not None)
    return dict(zip(names, grads), out=got[0].detach(), state=got[1].detach())


@pytest.mark.parametrize("dtype,c,name,read", CASES)
@pytest.mark.parametrize("which", ["out", "both", "state"])
def test_gradients(dtype, c, name, read, which):
    lens = LENGTHS[name]
    cu = [sum(lens[:i]) for i in range(len(lens) + 1)]
    gate, v, q = rows(cu[-1], c, dtype, 3, which == "both", read)
    s = normal(4, len(lens), c) if which != "out" else None
    dout = normal(5, cu[-1], c).to(v.dtype) if which != "state" else None
    dstate = normal(6, len(lens), c) if which != "out" else None
    val, tol = R.recurrence(gate, v, q, bounds_of(cu, cu[-1]), s, dout, dstate)
    got = gradients(gate, v, q, cu, s, dout, dstate)
    for n in got:
        R.check(n, got[n], val[n], tol[n])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,t", [(1, 1), (1, 300), (6, 50), (64, 3), (5, 64), (3, 200)])
def test_sequences_of_one_length(dtype, n, t):
    from ssla_hip import ops
    gate, v, q = rows(n * t, 40, dtype, 7)
    s = normal(8, n, 40)
    val, tol = R.recurrence(gate, v, q, [(i * t, i * t + t) for i in range(n)], s)
    out, last = ops.linear_recurrence(gate, v, q, n_seqs=n, state_in=s, return_state=True)
    R.check("out", out, val["out"], tol["out"])
    R.check("state", last, val["state"], tol["state"])


def test_gradients_agree_with_differences():
    """The oracle's values differ along a direction as the kernel's gradients say: a
    central difference of a step of 1e-4 is off by the third derivative's 1e-8."""
    lens, c = [90, 0, 33, 140], 20
    cu = [sum(lens[:i]) for i in range(len(lens) + 1)]
    gate, v, q = rows(cu[-1], c, "f32", 9)
    s = normal(10, len(lens), c)
    dout, dstate = normal(11, cu[-1], c), normal(12, len(lens), c)
    got = gradients(gate, v, q, cu, s, dout, dstate)
    for i, (t, n) in enumerate(((gate, "dgate"), (v, "dv"), (q, "dq"), (s, "dstate_in"))):
        d = torch.randn(t.shape, generator=torch.Generator().manual_seed(20 + i), dtype=torch.float64)
        f = []
        for e in (1e-4, -1e-4):
            args = [R.f64(x) for x in (gate, v, q, s)]
            args[i] = args[i] + e * d
            val, _ = R.recurrence(*args[:3], bounds_of(cu, cu[-1]), args[3])
            f.append((val["out"] * R.f64(dout)).sum() + (val["state"] * R.f64(dstate)).sum())
        want = (f[0] - f[1]).item() / 2e-4
        along = (R.f64(got[n]) * d).sum().item()
        size = (R.f64(got[n]) * d).abs().sum().item()
        assert abs(along - want) <= 1e-5 * size, (n, along, want)


@pytest.mark.parametrize("dtype,c", [("f32", 21), ("bf16", 64), ("f16", 130)])
def test_rows_of_no_sequence(dtype, c):
    """Rows before the first sequence and behind the last one stay; with gradients they
    are zeros, and their gradients too."""
    cu, total = [70, 70, 150, 320], 500
    gate, v, q = rows(total, c, dtype, 13)
    for t in (gate, v, q):
        t[:70] = float("nan")
        t[320:] = float("inf")
    out = torch.full((total, c), 7.0, device=DEV, dtype=v.dtype)
    run(gate, v, q, cu, out=out)
    val, tol = R.recurrence(gate, v, q, bounds_of(cu, total))
    R.check("out", out[70:320], val["out"][70:320], tol["out"][70:320])
    assert (out[:70] == 7).all() and (out[320:] == 7).all()
    dout = normal(14, total, c).to(v.dtype)
    dout[:70] = float("nan")
    val, tol = R.recurrence(gate, v, q, bounds_of(cu, total), None, dout)
    got = gradients(gate, v, q, cu, None, dout, None)
    for n in ("out", "dgate", "dv", "dq"):
        R.check(n, got[n][70:320], val[n][70:320], tol[n][70:320])
        assert (got[n][:70] == 0).all() and (got[n][320:] == 0).all(), n


def test_bounds_outside_the_tokens_are_clamped():
    gate, v, q = rows(100, 16, "f32", 15)
    out = run(gate, v, q, [-50, 40, 2_000_000_000])
    val, tol = R.recurrence(gate, v, q, [(0, 40), (40, 100)])
    R.check("out", out, val["out"], tol["out"])


def test_no_tokens_and_no_sequences():
    from ssla_hip import ops
    s = normal(16, 4, 12)
    none = torch.empty(0, 12, device=DEV)
    out, last = run(none, none, None, [0, 0, 0, 0, 0], s, return_state=True)
    assert out.shape == (0, 12) and torch.equal(last, s)
    out, last = run(none, none, none, [0, 0, 0], None, return_state=True)
    assert torch.equal(last, torch.zeros(2, 12, device=DEV))
    assert ops.linear_recurrence(none, none, n_seqs=0).shape == (0, 12)
    x = torch.full((3, 12), 5.0, device=DEV)
    out = torch.full((3, 12), 7.0, device=DEV)
    run(x, x, None, [2], out=out)
    assert (out == 7).all()
    a = none.clone().requires_grad_()
    i = s.clone().requires_grad_()
    out, last = run(a, none, None, [0, 0, 0, 0, 0], i, return_state=True)
    da, di = torch.autograd.grad(last, (a, i), s, allow_unused=True)
    assert torch.equal(di, s) and da.shape == (0, 12)
    b = x.clone().requires_grad_()
    (db,) = torch.autograd.grad(run(b, x, None, [2]).sum(), b)
    assert (db == 0).all()


@pytest.mark.parametrize("dtype,c", [("f32", 33), ("bf16", 96)])
def test_a_pool_in_its_own_place(dtype, c):
    """States of permuted slots read and written in one pool; a padded batch's rows and
    the other slots stay."""
    lens = [3, 0, 200, 1, 90, 2, 64, 5] * 6
    cu = [sum(lens[:i]) for i in range(len(lens) + 1)]
    slots = torch.randperm(70, generator=torch.Generator().manual_seed(1))[:len(lens)]
    slots[4] = -1
    slots[7] = 70 + 3
    gate, v, q = rows(cu[-1], c, dtype, 17)
    pool = normal(18, 70, c)
    first = torch.stack([pool[s] if 0 <= s < 70 else torch.zeros(c, device=DEV) for s in slots.tolist()])
    val, tol = R.recurrence(gate, v, q, bounds_of(cu, cu[-1]), first)
    was = pool.clone()
    out = torch.full((cu[-1], c), 7.0, device=DEV, dtype=v.dtype)
    run(gate, v, q, cu, pool, state_out=pool, slots=slots.to(torch.int32).to(DEV), out=out)
    kept = torch.ones(70, dtype=torch.bool)
    for i, s in enumerate(slots.tolist()):
        t = slice(cu[i], cu[i + 1])
        if 0 <= s < 70:
            kept[s] = False
            R.check("out", out[t], val["out"][t], tol["out"][t])
            R.check("state", pool[s], val["state"][i], tol["state"][i])
        else:
            assert (out[t] == 7).all()
    assert torch.equal(pool[kept.to(DEV)], was[kept.to(DEV)])


def test_pools_side_by_side():
    """Slots of two pools that lie in turn, and a pool whose slots lie apart."""
    both = normal(19, 6, 2, 40)
    was = both.clone()
    gate, v, q = rows(120, 40, "f32", 20)
    cu = [0, 30, 31, 31, 100, 119, 120]
    run(gate, v, q, cu, both[:, 0], state_out=both[:, 1])
    val, tol = R.recurrence(gate, v, q, bounds_of(cu, 120), was[:, 0])
    assert torch.equal(both[:, 0], was[:, 0])
    R.check("state", both[:, 1], val["state"], tol["state"])


def test_infinities_and_nans_stay_with_their_sequence_and_channel():
    lens, c = [80, 200, 5, 400, 70], 24
    cu = [sum(lens[:i]) for i in range(len(lens) + 1)]
    gate, v, q = rows(cu[-1], c, "f32", 21)
    want = run(gate, v, q, cu)
    bad = [(100, 3, v, float("inf")), (100, 7, gate, float("nan")), (350, 11, v, float("nan")), (81, 23, v, -float("inf"))]
    for t, ch, x, value in bad:
        x[t, ch] = value
    out = run(gate, v, q, cu)
    free = torch.ones_like(out, dtype=torch.bool)
    for t, ch, _, _ in bad:
        end = next(e for e in cu if e > t)
        free[t:end, ch] = False
        assert not torch.isfinite(out[t:end, ch]).any()
    assert torch.equal(out[free], want[free])
    dout = normal(22, cu[-1], c)
    got = gradients(gate, v, q, cu, None, dout, None)
    val, tol = R.recurrence(*(torch.where(torch.isfinite(x), x, 0.0) for x in (gate, v, q)), bounds_of(cu, cu[-1]),
                            None, dout)
    hurt = torch.ones(cu[-1], c, dtype=torch.bool)
    for t, ch, _, _ in bad:
        i = max(j for j, e in enumerate(cu) if e <= t)
        hurt[cu[i]:cu[i + 1], ch] = False
    for n in ("dgate", "dv", "dq"):
        R.check(n, got[n].cpu()[hurt], val[n][hurt], tol[n][hurt])


@pytest.mark.parametrize("value", [-200.0, -90.0, -30.0, 0.0, 30.0, 90.0, 200.0, float("inf"), -float("inf")])
def test_gates_at_their_ends(value):
    """Closed gates forget all, open ones nothing; no state is lost to a product with an
    infinity or a difference of like numbers."""
    v = normal(23, 300, 16) * 1e3
    gate = torch.full_like(v, value)
    out = run(gate, v, None, [0, 300])
    a = torch.sigmoid(torch.tensor(value, dtype=torch.float64))
    x, m, want, tol = torch.zeros(16, dtype=torch.float64), 0.0, [], []
    k = (min(abs(value), 110.0) + 16) * R.U32
    e = 0.0
    for t in range(300):
        x = a * x + R.f64(v[t])
        m = a * m + R.f64(v[t]).abs()
        # the gate's complement is off by k of the smaller of the two
        e = a * e + R.U32 * 3 * m + k * min(a, 1 - a) * m
        want.append(x), tol.append(e)
    R.check("out", out, torch.stack(want), torch.stack(tol))


@pytest.mark.parametrize("dtype,c", [("f32", 5), ("bf16", 10), ("bf16", 64), ("f16", 100)])
def test_strides_and_addresses(dtype, c):
    """Rows at odd strides and addresses, a gate that all tokens share, out at a stride of
    its own with its other columns kept."""
    from ssla_hip import ops
    T = 333
    base = normal(24, T * (2 * c + 3) + 1).to(R.TYPES[dtype])
    x = base[1:].view(T, 2 * c + 3)
    v, q = x[:, 1:1 + c], x[:, c + 2:2 * c + 2]
    gate = normal(25, c).to(v.dtype).expand(T, c)
    whole = torch.full((T, c + 5), 7.0, device=DEV, dtype=v.dtype)
    out = ops.linear_recurrence(gate, v, q, whole[:, 3:3 + c], n_seqs=3)
    val, tol = R.recurrence(gate, v, q, [(0, 111), (111, 222), (222, 333)])
    R.check("out", out, val["out"], tol["out"])
    assert (whole[:, :3] == 7).all() and (whole[:, 3 + c:] == 7).all()


def test_gradients_of_a_shared_gate_and_an_expanded_sum():
    """A gate of one row gets the sum over its tokens; out.sum()'s gradient comes
    expanded, with strides of zero."""
    from ssla_hip import ops
    T, c = 200, 30
    _, v, q = rows(T, c, "f32", 26)
    g = normal(27, c).requires_grad_()
    v = v.detach().requires_grad_()
    out = ops.linear_recurrence(g.expand(T, c), v, q, n_seqs=4)
    out.sum().backward()
    val, tol = R.recurrence(g.expand(T, c), v, q, [(i, i + 50) for i in range(0, T, 50)], None,
                            torch.ones(T, c))
    R.check("dv", v.grad, val["dv"], tol["dv"])
    R.check("dgate", g.grad, val["dgate"].sum(0), tol["dgate"].sum(0) + T * R.U32 * val["dgate"].abs().sum(0))


@pytest.mark.parametrize("want", [(0,), (1,), (2,), (3,), (0, 3), (1, 2)])
def test_only_the_wanted_gradients(want):
    lens, c = [40, 3, 90], 18
    cu = [0, 40, 43, 133]
    ts = list(rows(133, c, "f32", 28)) + [normal(29, 3, c)]
    dout = normal(30, 133, c)
    val, tol = R.recurrence(*ts[:3], bounds_of(cu, 133), ts[3], dout)
    xs = [t.detach().requires_grad_(i in want) for i, t in enumerate(ts)]
    run(xs[0], xs[1], xs[2], cu, xs[3]).backward(dout)
    for i, n in enumerate(("dgate", "dv", "dq", "dstate_in")):
        if i in want:
            R.check(n, xs[i].grad, val[n], tol[n])
        else:
            assert xs[i].grad is None


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_one_input_in_several_places(dtype):
    """gate, v and q may be one tensor; its gradient is the sum of the three."""
    x = (0.7 * normal(31, 150, 40)).to(R.TYPES[dtype])
    dout = normal(32, 150, 40).to(x.dtype)
    val, tol = R.recurrence(x, x, x, [(0, 150)], None, dout)
    y = x.clone().requires_grad_()
    run(y, y, y, [0, 150]).backward(dout)
    parts = [val[n] for n in ("dgate", "dv", "dq")]
    # two sums' roundings and three outputs'
    h = R.half_step(x.dtype)
    extra = 2 * h * sum(p.abs() for p in parts) + h * sum(p.abs() for p in parts)
    R.check("dx", y.grad, sum(parts), sum(tol[n] for n in ("dgate", "dv", "dq")) + extra)


def test_reruns_are_bit_identical():
    """Long sequences are scanned by many workgroups; what they find of each other's
    work on the way must not show."""
    lens, c = [9000, 12, 4000, 1, 1, 7000], 200
    cu = [sum(lens[:i]) for i in range(len(lens) + 1)]
    gate, v, q = rows(cu[-1], c, "bf16", 33)
    s, dout, dstate = normal(34, len(lens), c), normal(35, cu[-1], c).bfloat16(), normal(36, len(lens), c)
    first = gradients(gate, v, q, cu, s, dout, dstate)
    for _ in range(4):
        again = gradients(gate, v, q, cu, s, dout, dstate)
        assert all(torch.equal(first[n], again[n]) for n in first)


def test_a_sequence_in_parts():
    """States carried over calls give what one call gives."""
    gate, v, q = rows(1000, 56, "f32", 37)
    val, tol = R.recurrence(gate, v, q, [(0, 1000)])
    s, at = None, 0
    for n in (1, 99, 400, 64, 436):
        t = slice(at, at + n)
        out, s = run(gate[t], v[t], q[t], [0, n], s, return_state=True)
        R.check("out", out, val["out"][t], 2 * tol["out"][t])
        at += n
    R.check("state", s, val["state"], 2 * tol["state"])


@pytest.mark.parametrize("dtype,c", [("f32", 1), ("f32", 96), ("bf16", 40), ("f16", 129)])
@pytest.mark.parametrize("read", [True, False])
@pytest.mark.parametrize("n", [1, 70, 513])
def test_single_tokens(dtype, c, read, n):
    from ssla_hip import ops
    gate, v, q = rows(n, c, dtype, 38, True, read)
    pool = normal(39, n + 5, c + 3)[:, :c]
    was = pool.clone()
    slots = torch.randperm(n + 5, generator=torch.Generator().manual_seed(2))[:n]
    slots[n // 2] = -1 if n > 1 else slots[0]
    val, tol = R.recurrence(gate, v, q, [(i, i + 1) for i in range(n)], was[slots.to(DEV)])
    out = torch.full((n, c), 7.0, device=DEV, dtype=v.dtype)
    ops.linear_recurrence_step(gate, v, pool, q, out, slots=slots.to(torch.int32).to(DEV))
    on = slots >= 0
    R.check("out", out.cpu()[on], val["out"][on], tol["out"][on])
    R.check("state", pool.cpu()[slots[on]], val["state"][on], tol["state"][on])
    kept = torch.ones(n + 5, dtype=torch.bool)
    kept[slots[on]] = False
    assert torch.equal(pool.cpu()[kept], was.cpu()[kept]) and (out.cpu()[~on] == 7).all()


def test_tokens_one_by_one_are_the_sequence():
    from ssla_hip import ops
    gate, v, q = rows(60, 50, "bf16", 40)
    pool = torch.zeros(1, 50, device=DEV)
    outs = [ops.linear_recurrence_step(gate[t:t + 1], v[t:t + 1], pool, q[t:t + 1]) for t in range(60)]
    val, tol = R.recurrence(gate, v, q, [(0, 60)])
    R.check("out", torch.cat(outs), val["out"], tol["out"])
    R.check("state", pool, val["state"], tol["state"])


@pytest.mark.parametrize("lens", [[40], [3000, 1, 0, 900]])
def test_on_another_stream_and_captured(lens):
    """Replays read lengths, slots and rows anew, between the program's own work."""
    from ssla_hip import ops
    c = 72
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=DEV)
    total = int(cu[-1])
    gate, v, q = (t.clone() for t in rows(total, c, "bf16", 41))
    pool = normal(42, len(lens), c)
    start = pool.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = ops.linear_recurrence(gate, v, q, cu_seqlens=cu, state_in=pool, state_out=pool)
    torch.cuda.current_stream().wait_stream(side)
    after = pool.clone()
    val, tol = R.recurrence(gate, v, q, list(zip(cu.tolist()[:-1], cu.tolist()[1:])), start)
    R.check("out", eager, val["out"], tol["out"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.linear_recurrence(gate, v, q, cu_seqlens=cu, state_in=pool, state_out=pool)
    for i in range(4):
        pool.copy_(start)
        if i == 2:
            v.mul_(2.0)
            start2 = pool.clone()
            eager = ops.linear_recurrence(gate, v, q, cu_seqlens=cu, state_in=start2, state_out=start2)
            after = start2
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(pool, after), i


@pytest.mark.parametrize("lens", [[40, 7], [3000, 1, 0, 900]])
def test_a_captured_training_step(lens):
    from ssla_hip import ops
    c = 72
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=DEV)
    xs = [t.clone().requires_grad_() for t in rows(int(cu[-1]), c, "f32", 43)]
    dout = normal(44, int(cu[-1]), c)

    def step():
        out = ops.linear_recurrence(*xs, cu_seqlens=cu)
        return [out.detach()] + list(torch.autograd.grad(out, xs, dout))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        with torch.no_grad():
            xs[1].add_(0.25)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
