"""Operators with gradients under torch's autograd: what it records, what is refused,
several of them together."""
import pytest

torch = pytest.importorskip("torch")

import train_ref as R  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rnd(*s):
    return torch.randn(*s, device=DEV)


def calls():
    """Each operator as a function of its tensors by name."""
    from ssla_hip import ops
    T, C = 6, 8
    return [(ops.linear_recurrence, dict(gate=rnd(T, C), v=rnd(T, C), q=rnd(T, C), state_in=rnd(1, C))),
            (ops.layer_norm, dict(x=rnd(T, C), weight=rnd(C), bias=rnd(C), residual=rnd(T, C)))]


def writes():
    """Calls that write to tensors of the user's, and which those are."""
    from ssla_hip import ops
    T, C = 6, 8
    return [(ops.linear_recurrence, dict(gate=rnd(T, C), v=rnd(T, C), q=rnd(T, C), state_in=rnd(1, C),
                                         state_out=rnd(1, C), out=rnd(T, C)), ("out", "state_out")),
            (ops.linear_recurrence_step, dict(gate=rnd(T, C), v=rnd(T, C), q=rnd(T, C), state=rnd(T, C),
                                              out=rnd(T, C)), ("out", "state")),
            (ops.layer_norm, dict(x=rnd(T, C), weight=rnd(C), bias=rnd(C), residual=rnd(T, C), out=rnd(T, C)), ("out",))]


NAMES = ["sequences", "step", "norm"]


@pytest.mark.parametrize("i", range(3), ids=NAMES)
def test_forward_gradients_are_refused(i):
    import torch.autograd.forward_ad as fw
    f, kw, _ = writes()[i]
    for name in kw:
        with fw.dual_level():
            dual = fw.make_dual(kw[name], torch.ones_like(kw[name]))
            with pytest.raises(ValueError, match=name + " carries a forward gradient"):
                f(**dict(kw, **{name: dual}))


@pytest.mark.parametrize("i", range(3), ids=NAMES)
def test_function_transforms_raise(i):
    f, kw, _ = writes()[i]
    first = next(iter(kw))
    for out in ({}, {"out": None}):
        kw = dict(kw, **out)
        with pytest.raises((ValueError, RuntimeError)):
            torch.func.jvp(lambda x: f(**dict(kw, **{first: x})), (kw[first],), (torch.ones_like(kw[first]),))
        with pytest.raises((ValueError, RuntimeError)):
            torch.func.grad(lambda x: f(**dict(kw, **{first: x})).sum())(kw[first])
        with pytest.raises((ValueError, RuntimeError)):
            torch.func.vmap(lambda x: f(**dict(kw, **{first: x})))(kw[first][None])


@pytest.mark.parametrize("i", range(3), ids=NAMES)
def test_tensors_that_are_written_get_a_version(i):
    f, kw, written = writes()[i]
    before = {n: t._version for n, t in kw.items()}
    f(**kw)
    for n in kw:
        assert (kw[n]._version > before[n]) == (n in written), n


@pytest.mark.parametrize("i", range(2), ids=["sequences", "norm"])
def test_a_saved_input_that_changes_is_noticed(i):
    f, kw = calls()[i]
    for name in kw:
        if name in ("bias",):
            continue                                   # its values are not needed
        other = next(n for n in kw if n != name)
        ts = {n: t.clone().requires_grad_(n == other) for n, t in kw.items()}
        y = f(**ts)
        ts[name].mul_(2.0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


@pytest.mark.parametrize("i", range(2), ids=["sequences", "norm"])
def test_second_derivatives_are_refused(i):
    f, kw = calls()[i]
    for name in kw:
        x = kw[name].clone().requires_grad_()
        y = f(**dict(kw, **{name: x}))
        with pytest.raises(RuntimeError, match="second derivatives"):
            torch.autograd.grad(y.sum(), x, create_graph=True)


def test_what_has_no_gradient_is_refused_while_torch_records():
    from ssla_hip import ops
    x = rnd(6, 8).requires_grad_()
    y, s = rnd(6, 8), rnd(6, 8)
    slots = torch.zeros(1, dtype=torch.int32, device=DEV)
    bad = [lambda: ops.linear_recurrence(x, y, out=rnd(6, 8)), lambda: ops.linear_recurrence(y, x, state_out=rnd(1, 8)),
           lambda: ops.linear_recurrence(x, y, state_in=s, slots=slots), lambda: ops.linear_recurrence(x, y, state_in=s),
           lambda: ops.linear_recurrence(y, y, state_in=s[:1], state_out=rnd(1, 8), return_state=True),
           lambda: ops.linear_recurrence(y, y, state_in=s, slots=slots, return_state=True),
           lambda: ops.linear_recurrence(y, y, out=x), lambda: ops.linear_recurrence(y, y, state_out=x[:1]),
           lambda: ops.linear_recurrence_step(x, y, s), lambda: ops.linear_recurrence_step(y, y, x),
           lambda: ops.layer_norm(x, out=rnd(6, 8)), lambda: ops.layer_norm(y, out=x)]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was taken")
    with torch.no_grad():
        assert not ops.linear_recurrence(x, y, out=rnd(6, 8)).requires_grad
        assert not ops.layer_norm(x, out=rnd(6, 8)).requires_grad


def test_wrong_tensors_are_refused():
    from ssla_hip import lib, ops
    lr, st, ln = ops.linear_recurrence, ops.linear_recurrence_step, ops.layer_norm
    x, w, s = rnd(6, 8), rnd(8), rnd(6, 8)
    cu = torch.tensor([0, 6], dtype=torch.int32, device=DEV)
    bad = [lambda: lr(x.double(), x.double()), lambda: lr(x, x.half()), lambda: lr(x, x[:5]), lambda: lr(x, x, x[:, :7]),
           lambda: lr(x[0], x[0]), lambda: lr(x, x.cpu()), lambda: lr(x.t(), x.t()), lambda: lr(x[:, :0], x[:, :0]),
           lambda: lr(x, x, n_seqs=4), lambda: lr(x, x, n_seqs=0), lambda: lr(x, x, n_seqs=-1),
           lambda: lr(x, x, cu_seqlens=cu.long()), lambda: lr(x, x, cu_seqlens=cu.cpu()), lambda: lr(x, x, cu_seqlens=cu[:0]),
           lambda: lr(x, x, state_in=s.half()), lambda: lr(x, x, state_in=s[:, :4]), lambda: lr(x, x, state_in=s[0]),
           lambda: lr(x, x, n_seqs=2, state_in=s[:1]), lambda: lr(x, x, state_in=s, state_out=s[:5]),
           lambda: lr(x, x, state_in=s, slots=cu), lambda: lr(x, x, state_in=s, slots=cu[:1].long()),
           lambda: lr(x, x, out=rnd(6, 9)), lambda: lr(x, x, out=rnd(8, 6).t()), lambda: lr(x, x, out=rnd(6, 8).half()),
           lambda: lr(x.to_sparse(), x), lambda: lr(x, x, return_state="yes"),
           lambda: st(x, x, s[:5]), lambda: st(x, x, s.half()), lambda: st(x, x, s, slots=cu), lambda: st(x, x, s, rnd(6, 9)),
           lambda: ln(x.double()), lambda: ln(x.t()), lambda: ln(x, w.half()), lambda: ln(x.half(), w.bfloat16()),
           lambda: ln(x.half(), w, w.half()), lambda: ln(x, w[:7]), lambda: ln(x, rnd(16)[::2]), lambda: ln(x, residual=x[:5]),
           lambda: ln(x, residual=x.half()), lambda: ln(x, out=x[:5]), lambda: ln(x[0, 0]), lambda: ln(x, eps="1"),
           lambda: ln(rnd(4, 5, 6, 8).transpose(1, 2)), lambda: ln(x.to_sparse())]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was taken")
    with pytest.raises(lib.SslaHipError, match="out"):
        lr(x, x, out=x)
    with pytest.raises(lib.SslaHipError, match="overlap"):
        lr(x, x, out=torch.empty(1, 8, device=DEV).expand(6, 8))
    with pytest.raises(lib.SslaHipError, match="overlap"):
        big = rnd(7, 8)
        lr(x, x, n_seqs=6, state_in=big[:6], state_out=big[1:])
    with pytest.raises(lib.SslaHipError, match="eps"):
        ln(x, eps=-1.0)


def test_a_capture_with_an_older_graph_of_its_leaves_is_refused():
    """Autograd would add up their gradients on the default stream, from within the
    capture, which ends the process."""
    from ssla_hip import ops
    for i in range(2):
        f, kw = calls()[i]
        for name in kw:
            x = kw[name].clone().requires_grad_()
            older = f(**dict(kw, **{name: x}))
            graph = torch.cuda.CUDAGraph()
            with pytest.raises(ValueError, match=name + " has a graph"):
                with torch.cuda.graph(graph):
                    ops.group_norm(kw[next(iter(kw))], 2)
                    f(**dict(kw, **{name: x}))
            del older
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                got = torch.autograd.grad(f(**dict(kw, **{name: x})).sum(), x)
            for _ in range(3):
                graph.replay()
                torch.cuda.synchronize()
                want = torch.autograd.grad(f(**dict(kw, **{name: x})).sum(), x)
                assert torch.equal(got[0], want[0])


def layer(x, w_in, w_out, gamma, beta, cu, plain):
    """An SSLA layer over records sorted by cell: q, v, g from one projection, the
    recurrence, the contraction, layer norm with the residual."""
    from ssla_hip import ops
    c = x.shape[1]
    p = x @ w_in
    if plain:
        q, v, g = p.split(c, 1)
        h, outs = None, []
        ends = cu.tolist()
        for t in range(x.shape[0]):
            h = v[t] if t in ends else torch.sigmoid(g[t]) * h + v[t]
            outs.append(q[t] * h)
        s = torch.stack(outs) @ w_out + x
        d = s - s.mean(1, keepdim=True)
        return d / torch.sqrt((d * d).mean(1, keepdim=True) + 1e-5) * gamma + beta
    q, v, g = p.split(c, 1)
    y = ops.linear_recurrence(g, v, q, cu_seqlens=cu)
    return ops.layer_norm(y @ w_out, gamma, beta, residual=x)


def test_two_layers_together():
    """The values and all gradients of two layers, one behind the other.  Their products
    are torch's, in fp32: a relative error of 1e-4 of each tensor's size is a thousand
    roundings."""
    gen = torch.Generator().manual_seed(5)
    lens = [9, 0, 30, 1, 44, 16]
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    c, T = 48, sum(lens)
    mk = lambda *s, scale=1.0: (torch.randn(*s, generator=gen, dtype=torch.float64) * scale)  # noqa: E731
    x = mk(T, c)
    params = [(mk(c, 3 * c, scale=c ** -0.5), mk(c, c, scale=c ** -0.5), 1 + 0.2 * mk(c), 0.2 * mk(c)) for _ in range(2)]
    dy = mk(T, c)

    def whole(dev, dtype, plain):
        leaves = [t.to(dev, dtype).requires_grad_() for t in [x] + [t for p in params for t in p]]
        y = leaves[0]
        for i in range(2):
            y = layer(y, *leaves[1 + 4 * i:5 + 4 * i], cu.to(dev), plain)
        return [y.detach()] + list(torch.autograd.grad(y, leaves, dy.to(dev, dtype)))

    want, got = whole("cpu", torch.float64, True), whole(DEV, torch.float32, False)
    for i, (a, b) in enumerate(zip(got, want)):
        assert (a.cpu().double() - b).abs().max() <= 1e-4 * b.abs().max(), i


def test_a_drain_s_features_normed_and_read_as_sequences(stub_dir):
    """Output slots (98 words, features behind two flags) as rows of both operators."""
    from test_ops_on_drain_buffers_gpu import Words
    from ssla_hip import abi, events, hybrid, ops
    rec = events.blob_records(900, seed=4)
    with hybrid.Drain.from_weights_dir(stub_dir) as d:
        d.load_rings([events.to_records(rec)])
        d._outs[0].zero()
        d.run()
        slots = torch.as_tensor(Words(d._outs[0].ptr, 900, abi.OUTPUT_DTYPE.itemsize // 4), device="cuda")
        feat = slots[:, 2:]
        was = feat.clone()
        val, tol = R.recurrence(was, was, was, [(0, 900)])
        R.check("out", ops.linear_recurrence(feat, feat, feat), val["out"], tol["out"])
        val, tol = R.layer_norm(was, None, None, None, 1e-5)
        ops.layer_norm(feat, out=feat)
        R.check("y", feat, val["y"], tol["y"])
