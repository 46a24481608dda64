"""Sequence operators and torch's gradients, which they have none of: nothing is
dropped in silence."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
DEV = "cuda"


def calls():
    """Each operator as a function of its tensors by name."""
    from ssla_hip import ops
    T, H, D = 6, 2, 8
    rnd = lambda *s: torch.randn(*s, device=DEV)  # noqa: E731
    seq = dict(q=rnd(T, H, D), k=rnd(T, H, D), v=rnd(T, H, D), log_decay=-rnd(T, H).abs())
    return [
        (ops.linear_attention, dict(seq, state_in=rnd(1, H, D, D), state_out=rnd(1, H, D, D), out=rnd(T, H, D))),
        (ops.linear_attention_step, dict(seq, state=rnd(T, H, D, D), out=rnd(T, H, D))),
        (lambda **kw: ops.group_norm(groups=2, **kw),
         dict(x=rnd(T, 8), weight=rnd(8), bias=rnd(8), gate=rnd(T, 8), out=rnd(T, 8))),
    ]


@pytest.mark.parametrize("i", range(3), ids=["sequences", "step", "norm"])
def test_forward_gradients_are_refused(i):
    import torch.autograd.forward_ad as fw
    f, kw = calls()[i]
    want = f(**{n: t.clone() for n, t in kw.items()})
    for name in kw:
        with fw.dual_level():
            dual = fw.make_dual(kw[name], torch.ones_like(kw[name]))
            with pytest.raises(ValueError, match=name + " carries a forward gradient"):
                f(**dict(kw, **{name: dual}))
            # the primal is taken
            f(**{n: fw.unpack_dual(dual).primal.clone() if n == name else t.clone() for n, t in kw.items()})
    assert torch.equal(f(**kw), want)


@pytest.mark.parametrize("i", range(3), ids=["sequences", "step", "norm"])
def test_function_transforms_raise(i):
    f, kw = calls()[i]
    first = next(iter(kw))
    with pytest.raises((ValueError, RuntimeError)):
        torch.func.jvp(lambda x: f(**dict(kw, **{first: x})), (kw[first],), (torch.ones_like(kw[first]),))
    with pytest.raises((ValueError, RuntimeError)):
        torch.func.grad(lambda x: f(**dict(kw, **{first: x})).sum())(kw[first])
    with pytest.raises((ValueError, RuntimeError)):
        torch.func.vmap(lambda x: f(**dict(kw, **{first: x})))(kw[first][None])


@pytest.mark.parametrize("i,name", [(0, "out"), (0, "state_out"), (1, "out"), (1, "state"), (2, "out")])
def test_a_saved_tensor_that_a_call_overwrites_is_noticed(i, name):
    f, kw = calls()[i]
    x = torch.randn_like(kw[name]).requires_grad_()
    y = (x * kw[name]).sum()                   # keeps kw[name] for x's gradient
    before = kw[name]._version
    f(**kw)
    assert kw[name]._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.parametrize("i", range(3), ids=["sequences", "step", "norm"])
def test_tensors_that_are_only_read_keep_their_version(i):
    f, kw = calls()[i]
    before = {n: t._version for n, t in kw.items()}
    f(**kw)
    for n in kw:
        assert (kw[n]._version == before[n]) == (n not in ("out", "state", "state_out")), n


@pytest.mark.parametrize("i", range(3), ids=["sequences", "step", "norm"])
def test_inference_tensors_are_taken(i):
    with torch.inference_mode():
        f, kw = calls()[i]
        f(**kw)
    assert kw["out"].is_inference()
    want = f(**{n: t.clone() for n, t in kw.items()})
    assert torch.equal(f(**kw), want)
