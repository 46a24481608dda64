"""Operators with gradients without a GPU: descriptors and what the C ABI refuses
(before any device call)."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from ssla_hip import abi, lib, ops  # noqa: E402

P = 1 << 20          # an aligned address; refused calls never follow it


def fill(d, kw):
    for n, v in kw.items():
        setattr(d, n, v)
    return d


def linrec(**kw):
    d = abi.SslaHipLinRec()
    d.dtype, d.channels, d.n_seqs, d.n_slots, d.n_tokens = abi.SSLA_BF16, 32, 2, 2, 20
    for i, n in enumerate(("gate", "v", "q", "out", "state_in", "state_out", "carries")):
        setattr(d, n, P + (i << 24))
    for n in ("gate", "v", "q", "out", "state_in", "state_out"):
        setattr(d, n + "_stride", 32)
    return fill(d, kw)


def linrec_grad(**kw):
    g = abi.SslaHipLinRecGrad()
    for i, n in enumerate(("dout", "dstate_out", "dgate", "dv", "dq", "dstate_in")):
        setattr(g, n, P + ((16 + i) << 24))
        setattr(g, n + "_stride", 32)
    return fill(g, kw)


def norm(**kw):
    d = abi.SslaHipLayerNorm()
    d.dtype, d.weight_dtype, d.rows, d.channels, d.eps = abi.SSLA_BF16, abi.SSLA_F32, 10, 48, 1e-5
    for i, n in enumerate(("x", "residual", "weight", "bias", "out", "stats")):
        setattr(d, n, P + (i << 24))
    d.x_stride = d.residual_stride = d.out_stride = 48
    return fill(d, kw)


def norm_grad(**kw):
    g = abi.SslaHipLayerNormGrad()
    for i, n in enumerate(("dout", "dx", "dweight", "dbias")):
        setattr(g, n, P + ((16 + i) << 24))
    g.dout_stride = g.dx_stride = 48
    return fill(g, kw)


def at(d):
    return ctypes.addressof(d)


def test_descriptor_layouts():
    out = (ctypes.c_longlong * 4)()
    lib.check(lib.load().ssla_hip_train_layout(out, 4))
    assert list(out) == [ctypes.sizeof(t) for t in (abi.SslaHipLinRec, abi.SslaHipLinRecGrad,
                                                    abi.SslaHipLayerNorm, abi.SslaHipLayerNormGrad)]
    assert lib.load().ssla_hip_train_layout(out, 3) == abi.SSLA_ERR_ARG


BAD = [dict(dtype=3), dict(dtype=-1), dict(channels=0), dict(channels=0x7fff0001), dict(n_seqs=-1),
       dict(n_slots=-1), dict(n_seqs=0x7fff0001), dict(gate_stride=-1), dict(v_stride=(1 << 40) + 1), dict(q_stride=-1),
       dict(gate=None), dict(v=None), dict(gate=P + 1), dict(v=P + 1), dict(q=P + 1),
       dict(state_in=P + 2), dict(state_in_stride=31)]
BAD_OUT = [dict(out=None), dict(out=P + 1), dict(out_stride=31), dict(out_stride=-1), dict(out=P),
           dict(out=P + (1 << 24)), dict(out=P + (2 << 24)), dict(slots=P + 2), dict(state_out=P + 2),
           dict(state_out_stride=31), dict(n_slots=1), dict(state_out=P + (4 << 24) + 4),
           dict(state_out=P + (4 << 24), state_out_stride=33)]
BAD_TOKENS = [dict(n_tokens=-1), dict(n_tokens=0x7fff0001), dict(n_tokens=21), dict(n_seqs=0), dict(cu_seqlens=P + 1),
              dict(carries=P + 2)]


@pytest.mark.parametrize("bad", BAD + BAD_OUT + BAD_TOKENS, ids=str)
def test_linrec_refuses(bad):
    L, n = lib.load(), ctypes.c_size_t(7)
    d = linrec(**bad)
    assert L.ssla_hip_linrec(at(d), P, 1 << 40, None) == abi.SSLA_ERR_ARG
    assert b"ssla_hip_linrec" in L.ssla_hip_last_error()
    if bad not in BAD_OUT:
        assert L.ssla_hip_linrec_workspace(at(d), ctypes.byref(n)) == abi.SSLA_ERR_ARG
        assert L.ssla_hip_linrec_carries(at(d), ctypes.byref(n)) == abi.SSLA_ERR_ARG
    if bad not in BAD_TOKENS:
        assert L.ssla_hip_linrec_step(at(d), None) == abi.SSLA_ERR_ARG
    if bad not in BAD_OUT:
        assert L.ssla_hip_linrec_backward(at(d), at(linrec_grad()), P, 1 << 40, None) == abi.SSLA_ERR_ARG


@pytest.mark.parametrize("bad", [
    dict(dout=P + (16 << 24) + 1), dict(dgate=P + 1), dict(dv=P + 1), dict(dq=P + 1), dict(dstate_in=P + 2),
    dict(dstate_out=P + 2), dict(dout_stride=-1), dict(dgate_stride=31), dict(dv_stride=-1), dict(dq_stride=1 << 41),
    dict(dstate_in_stride=31), dict(dstate_out_stride=-1), dict(dgate=P), dict(dv=P + (16 << 24)),
    dict(dstate_in=P + (17 << 24)), dict(dstate_in=P + (4 << 24))], ids=str)
def test_linrec_backward_refuses(bad):
    L = lib.load()
    assert L.ssla_hip_linrec_backward(at(linrec()), at(linrec_grad(**bad)), P, 1 << 40, None) == abi.SSLA_ERR_ARG
    assert b"ssla_hip_linrec_backward" in L.ssla_hip_last_error()


def test_linrec_refuses_nulls_and_what_is_missing():
    L, n = lib.load(), ctypes.c_size_t()
    assert L.ssla_hip_linrec(None, None, 0, None) == abi.SSLA_ERR_ARG
    assert L.ssla_hip_linrec_step(None, None) == abi.SSLA_ERR_ARG
    assert L.ssla_hip_linrec_workspace(None, ctypes.byref(n)) == abi.SSLA_ERR_ARG
    assert L.ssla_hip_linrec_workspace(at(linrec()), None) == abi.SSLA_ERR_ARG
    assert L.ssla_hip_linrec_carries(at(linrec()), None) == abi.SSLA_ERR_ARG
    assert L.ssla_hip_linrec_backward(at(linrec()), None, P, 1 << 40, None) == abi.SSLA_ERR_ARG
    for d, g in ((linrec(slots=P), linrec_grad()), (linrec(carries=None), linrec_grad()),
                 (linrec(q=None), linrec_grad())):
        assert L.ssla_hip_linrec_backward(at(d), at(g), P, 1 << 40, None) == abi.SSLA_ERR_ARG
    for bad in (dict(state_in=None), dict(state_out=None)):
        assert L.ssla_hip_linrec_step(at(linrec(**bad)), None) == abi.SSLA_ERR_ARG


def test_linrec_workspace():
    """What the sizes depend on; a workspace that is missing, too small or misaligned is
    refused where one is needed."""
    L, n, m = lib.load(), ctypes.c_size_t(7), ctypes.c_size_t(7)
    assert L.ssla_hip_linrec_workspace(at(linrec(n_tokens=0)), ctypes.byref(n)) == 0 and n.value == 0
    big = dict(n_tokens=1_000_000, n_seqs=2, out=P + (1 << 40), gate=P + (2 << 40), v=P + (3 << 40), q=P + (4 << 40))
    assert L.ssla_hip_linrec_workspace(at(linrec(**big)), ctypes.byref(n)) == 0
    assert L.ssla_hip_linrec_carries(at(linrec(**big)), ctypes.byref(m)) == 0 and m.value > 0
    if n.value:
        for ws, size in ((None, n.value), (P, n.value - 1), (P + 8, n.value)):
            assert L.ssla_hip_linrec(at(linrec(**big)), ws, size, None) == abi.SSLA_ERR_ARG
            assert b"workspace" in L.ssla_hip_last_error()
            assert L.ssla_hip_linrec_backward(at(linrec(**big)), at(linrec_grad()), ws, size, None) == abi.SSLA_ERR_ARG
            assert b"workspace" in L.ssla_hip_last_error()


def test_grids_that_cannot_be_launched_are_refused():
    L, big = lib.load(), 0x7fff0000
    wide = dict(gate_stride=1 << 32, v_stride=1 << 32, q_stride=1 << 32, out_stride=1 << 32, state_in_stride=1 << 32,
                state_out_stride=1 << 32, state_in=None, state_out=None)
    for d in (linrec(n_tokens=big, n_seqs=1, channels=big, **wide),):
        assert L.ssla_hip_linrec(at(d), P, 1 << 62, None) == abi.SSLA_ERR_ARG
        assert b"too many" in L.ssla_hip_last_error()
        g = linrec_grad(**{n + "_stride": 1 << 32 for n in ("dout", "dgate", "dv", "dq", "dstate_in", "dstate_out")})
        assert L.ssla_hip_linrec_backward(at(d), at(g), P, 1 << 62, None) == abi.SSLA_ERR_ARG
        assert b"too many" in L.ssla_hip_last_error()
    assert L.ssla_hip_linrec(at(linrec(wait_us=1000001)), P, 1 << 40, None) == abi.SSLA_ERR_ARG
    d = linrec(n_seqs=big, n_slots=big, channels=1 << 20, gate_stride=1 << 20, v_stride=1 << 20, q_stride=1 << 20,
               out_stride=1 << 20, state_in_stride=1 << 20, state_out_stride=1 << 20, state_out=P + (4 << 24))
    assert L.ssla_hip_linrec_step(at(d), None) == abi.SSLA_ERR_ARG
    assert b"too many" in L.ssla_hip_last_error()


BAD_NORM = [dict(dtype=3), dict(weight_dtype=abi.SSLA_F16), dict(weight_dtype=-1), dict(rows=-1), dict(channels=-1),
            dict(rows=0x7fff0001), dict(channels=0x7fff0001), dict(eps=-1.0), dict(eps=float("nan")), dict(x=None),
            dict(x=P + 1), dict(residual=P + 1), dict(weight=P + 2), dict(stats=P + 2), dict(x_stride=-1),
            dict(residual_stride=1 << 41)]
BAD_NORM_OUT = [dict(out=None), dict(out=P + 1), dict(out_stride=47), dict(bias=P + 2), dict(out=P, x_stride=50),
                dict(out=P + (1 << 24), residual_stride=96)]


@pytest.mark.parametrize("bad", BAD_NORM + BAD_NORM_OUT, ids=str)
def test_layer_norm_refuses(bad):
    L, n = lib.load(), ctypes.c_size_t(7)
    assert L.ssla_hip_layer_norm(at(norm(**bad)), None) == abi.SSLA_ERR_ARG
    assert b"ssla_hip_layer_norm" in L.ssla_hip_last_error()
    if bad in BAD_NORM:
        d, g = norm(**bad), norm_grad()
        assert L.ssla_hip_layer_norm_backward(at(d), at(g), P, 1 << 40, None) == abi.SSLA_ERR_ARG
        assert L.ssla_hip_layer_norm_backward_workspace(at(d), at(g), ctypes.byref(n)) == abi.SSLA_ERR_ARG


@pytest.mark.parametrize("bad", [dict(dout=None), dict(dout=P + 1), dict(dx=P + 1), dict(dweight=P + 2),
                                 dict(dbias=P + 2), dict(dout_stride=-1), dict(dx_stride=47), dict(dx_stride=1 << 41),
                                 dict(dx=P), dict(dx=P + (16 << 24)), dict(dweight=P + (2 << 24))], ids=str)
def test_layer_norm_backward_refuses(bad):
    L, n = lib.load(), ctypes.c_size_t(7)
    d, g = norm(), norm_grad(**bad)
    assert L.ssla_hip_layer_norm_backward(at(d), at(g), P, 1 << 40, None) == abi.SSLA_ERR_ARG
    assert b"ssla_hip_layer_norm_backward" in L.ssla_hip_last_error()
    assert L.ssla_hip_layer_norm_backward_workspace(at(d), at(g), ctypes.byref(n)) == abi.SSLA_ERR_ARG


def test_layer_norm_refuses_nulls_and_a_missing_workspace():
    L, n = lib.load(), ctypes.c_size_t()
    assert L.ssla_hip_layer_norm(None, None) == abi.SSLA_ERR_ARG
    assert L.ssla_hip_layer_norm_backward(None, at(norm_grad()), P, 1, None) == abi.SSLA_ERR_ARG
    assert L.ssla_hip_layer_norm_backward(at(norm()), None, P, 1, None) == abi.SSLA_ERR_ARG
    assert L.ssla_hip_layer_norm_backward(at(norm(stats=None)), at(norm_grad()), P, 1, None) == abi.SSLA_ERR_ARG
    assert L.ssla_hip_layer_norm_backward_workspace(at(norm()), at(norm_grad()), None) == abi.SSLA_ERR_ARG
    assert L.ssla_hip_layer_norm_backward_workspace(at(norm()), at(norm_grad()), ctypes.byref(n)) == 0 and n.value
    for ws, size in ((None, n.value), (P, n.value - 1), (P + 4, n.value)):
        assert L.ssla_hip_layer_norm_backward(at(norm()), at(norm_grad()), ws, size, None) == abi.SSLA_ERR_ARG
        assert b"workspace" in L.ssla_hip_last_error()
    g = norm_grad(dweight=None, dbias=None)
    assert L.ssla_hip_layer_norm_backward_workspace(at(norm()), at(g), ctypes.byref(n)) == 0 and n.value == 0


def test_nothing_to_do_is_no_error():
    L = lib.load()
    assert L.ssla_hip_linrec(at(linrec(n_seqs=0, n_tokens=0)), None, 0, None) == 0
    assert L.ssla_hip_linrec_step(at(linrec(n_seqs=0)), None) == 0
    assert L.ssla_hip_layer_norm(at(norm(rows=0)), None) == 0
    assert L.ssla_hip_layer_norm(at(norm(channels=0)), None) == 0


def test_python_refuses_tensors_off_the_gpu_and_what_is_no_argument():
    q = torch.zeros(5, 8)
    for f in (lambda: ops.linear_recurrence(q, q), lambda: ops.linear_recurrence_step(q, q, q), lambda: ops.layer_norm(q)):
        with pytest.raises(ValueError, match="GPU"):
            f()
    for f in (lambda: ops.linear_recurrence(q.numpy(), q), lambda: ops.linear_recurrence(q, None),
              lambda: ops.linear_recurrence_step(q, q, None), lambda: ops.layer_norm(None),
              lambda: ops.layer_norm(q, eps="1"), lambda: ops._ops.layer_norm(q)):
        with pytest.raises(ValueError):
            f()


def test_carries_and_sums_that_cannot_be_are_refused():
    L, big = lib.load(), 0x7fff0000
    assert L.ssla_hip_linrec(at(linrec(slots=P)), None, 0, None) == abi.SSLA_ERR_ARG
    assert b"slots" in L.ssla_hip_last_error()
    wide = norm(rows=1, channels=big, weight=None, bias=None)
    assert L.ssla_hip_layer_norm_backward(at(wide), at(norm_grad()), P, 1 << 62, None) == abi.SSLA_ERR_ARG
    assert b"too many" in L.ssla_hip_last_error()
