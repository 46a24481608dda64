"""Sequence operators without a GPU: descriptors, what the C ABI refuses (before
any device call), and what the Python entry points refuse."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from ssla_hip import abi, lib, ops  # noqa: E402

P = 1 << 20          # an aligned address; refused calls never follow it


def linattn(**kw):
    d = abi.SslaHipLinAttn()
    d.dtype, d.heads, d.qk_heads, d.dk, d.dv = abi.SSLA_BF16, 4, 2, 32, 64
    d.n_seqs, d.max_len, d.n_slots, d.n_tokens = 2, 10, 2, 20
    for i, n in enumerate(("q", "k", "v", "log_decay", "out", "state_in", "state_out")):
        setattr(d, n, P + (i << 24))
    for n, w in (("q", 2 * 32), ("k", 2 * 32), ("v", 4 * 64), ("out", 4 * 64)):
        getattr(d, n + "_stride")[:] = [w, w // (2 if n in "qk" else 4)]
    d.decay_stride[:] = [4, 1]
    d.state_stride = 4 * 32 * 64
    for n, v in kw.items():
        if n.endswith("_stride") and n != "state_stride":
            getattr(d, n)[:] = v
        else:
            setattr(d, n, v)
    return d


def norm(**kw):
    d = abi.SslaHipGroupNorm()
    d.dtype, d.n, d.rows, d.channels, d.groups, d.act = abi.SSLA_F32, 2, 10, 48, 4, abi.SSLA_ACT_SILU
    d.x, d.gate, d.weight, d.bias, d.out = P, P + 8192, 0, 0, P + 16384
    for s in (d.x_stride, d.gate_stride, d.out_stride):
        s[:] = [480, 48]
    d.eps = 1e-5
    for n, v in kw.items():
        if n.endswith("_stride"):
            getattr(d, n)[:] = v
        else:
            setattr(d, n, v)
    return d


def test_descriptor_layouts():
    out = (ctypes.c_longlong * 2)()
    lib.check(lib.load().ssla_hip_ops_layout(out, 2))
    assert list(out) == [ctypes.sizeof(abi.SslaHipLinAttn), ctypes.sizeof(abi.SslaHipGroupNorm)]
    assert lib.load().ssla_hip_ops_layout(out, 1) == abi.SSLA_ERR_ARG


BAD_BOTH = [dict(dtype=3), dict(dtype=-1), dict(heads=0), dict(qk_heads=0), dict(qk_heads=3),
            dict(dk=0), dict(dk=257), dict(dv=0), dict(dv=257), dict(n_seqs=-1), dict(n_slots=-1),
            dict(q_stride=[-1, 32]), dict(v_stride=[256, -64]), dict(out_stride=[1 << 41, 64]),
            dict(q=None), dict(k=None), dict(v=None), dict(log_decay=None), dict(out=None),
            dict(q=P + 1), dict(out=P + 1), dict(log_decay=P + 2), dict(slots=P + 2),
            dict(state_out=P + 3), dict(state_stride=4 * 32 * 64 - 1), dict(n_slots=1),
            dict(out_stride=[0, 64]), dict(out_stride=[256, 0]), dict(out_stride=[200, 64]),
            dict(state_out=P + (5 << 24) + 4), dict(out=P), dict(out=P + (2 << 24))]
BAD_PROMPT = [dict(n_tokens=-1), dict(n_tokens=1 << 31, cu_seqlens=P), dict(max_len=-1),
              dict(n_tokens=21), dict(cu_seqlens=P + 1),
              dict(n_tokens=(1 << 31) - (1 << 16) + 1, cu_seqlens=P),
              dict(n_tokens=(1 << 31) - (1 << 16), max_len=1 << 30, cu_seqlens=P, n_seqs=(1 << 31) - 1,
                   state_in=None, state_out=None, heads=1, qk_heads=1)]


@pytest.mark.parametrize("bad", BAD_BOTH + BAD_PROMPT, ids=str)
def test_linattn_refuses(bad):
    L, d, n = lib.load(), linattn(**bad), ctypes.c_size_t(7)
    assert L.ssla_hip_linattn(ctypes.addressof(d), None, 0, None) == abi.SSLA_ERR_ARG
    assert b"ssla_hip_linattn" in L.ssla_hip_last_error()
    assert L.ssla_hip_linattn_workspace(ctypes.addressof(d), ctypes.byref(n)) == abi.SSLA_ERR_ARG
    if bad in BAD_BOTH:
        assert L.ssla_hip_linattn_step(ctypes.addressof(d), None) == abi.SSLA_ERR_ARG


def test_linattn_refuses_nulls_and_missing_states():
    L = lib.load()
    n = ctypes.c_size_t()
    assert L.ssla_hip_linattn(None, None, 0, None) == abi.SSLA_ERR_ARG
    assert L.ssla_hip_linattn_step(None, None) == abi.SSLA_ERR_ARG
    assert L.ssla_hip_linattn_workspace(None, ctypes.byref(n)) == abi.SSLA_ERR_ARG
    assert L.ssla_hip_linattn_workspace(ctypes.addressof(linattn()), None) == abi.SSLA_ERR_ARG
    for bad in (dict(state_in=None), dict(state_out=None)):
        assert L.ssla_hip_linattn_step(ctypes.addressof(linattn(**bad)), None) == abi.SSLA_ERR_ARG


def test_grids_that_cannot_be_launched_are_refused():
    L, n = lib.load(), (1 << 31) - 1
    for heads in (1, n):
        d = linattn(n_seqs=n, heads=heads, qk_heads=1, n_tokens=0, max_len=0, n_slots=n, state_in=None,
                    state_out=None)
        assert L.ssla_hip_linattn(ctypes.addressof(d), None, 0, None) == abi.SSLA_ERR_ARG
        assert b"too many" in L.ssla_hip_last_error()
    d = linattn(n_seqs=1 << 24, n_slots=1 << 24, heads=1, qk_heads=1, state_out=P + (5 << 24))
    assert L.ssla_hip_linattn_step(ctypes.addressof(d), None) == abi.SSLA_ERR_ARG
    assert b"too many" in L.ssla_hip_last_error()
    d = norm(n=1 << 24, rows=100, channels=64, groups=1, x_stride=[6400, 64], gate_stride=[6400, 64],
             out_stride=[6400, 64], out=P + (1 << 45))
    assert L.ssla_hip_group_norm(ctypes.addressof(d), None, 0, None) == abi.SSLA_ERR_ARG
    assert b"too many" in L.ssla_hip_last_error()


def test_linattn_workspace():
    """None for short sequences; a state for each piece of cut ones, refused when
    missing, too small or misaligned."""
    L, n = lib.load(), ctypes.c_size_t(7)
    d = linattn()
    assert L.ssla_hip_linattn_workspace(ctypes.addressof(d), ctypes.byref(n)) == 0 and n.value == 0
    d = linattn(max_len=4000, n_tokens=8000)
    assert L.ssla_hip_linattn_workspace(ctypes.addressof(d), ctypes.byref(n)) == 0
    assert n.value >= 2 * 2 * 4 * 32 * 64 * 4
    for ws, size in ((None, n.value), (P, n.value - 1), (P + 8, n.value)):
        assert L.ssla_hip_linattn(ctypes.addressof(d), ws, size, None) == abi.SSLA_ERR_ARG
        assert b"workspace" in L.ssla_hip_last_error()
    d = linattn(max_len=1 << 30, n_tokens=(1 << 31) - 1, cu_seqlens=P, heads=512, qk_heads=512)
    assert L.ssla_hip_linattn_workspace(ctypes.addressof(d), ctypes.byref(n)) in (0, abi.SSLA_ERR_ARG)


@pytest.mark.parametrize("bad", [
    dict(dtype=3), dict(n=-1), dict(rows=-1), dict(channels=-48), dict(groups=0), dict(groups=5),
    dict(act=4), dict(act=-1), dict(rows=0x7fff0001), dict(channels=0x7fff0001, groups=1), dict(eps=-1.0), dict(eps=float("nan")), dict(x=None), dict(out=None),
    dict(x=P + 2), dict(gate=P + 1), dict(weight=P + 1), dict(bias=P + 3), dict(out=P + 1),
    dict(x_stride=[-1, 48]), dict(gate_stride=[480, -1]), dict(out_stride=[480, 1 << 41]),
    dict(out_stride=[0, 48]), dict(out_stride=[480, 47]), dict(out_stride=[479, 48]),
    dict(out=P, x_stride=[960, 96]), dict(out=P + 8192, gate_stride=[960, 96])], ids=str)
def test_group_norm_refuses(bad):
    L, d, n = lib.load(), norm(**bad), ctypes.c_size_t(7)
    assert L.ssla_hip_group_norm(ctypes.addressof(d), P, 1 << 30, None) == abi.SSLA_ERR_ARG
    assert b"ssla_hip_group_norm" in L.ssla_hip_last_error()
    assert L.ssla_hip_group_norm_workspace(ctypes.addressof(d), ctypes.byref(n)) == abi.SSLA_ERR_ARG


def test_group_norm_refuses_nulls_and_a_missing_workspace():
    L, n = lib.load(), ctypes.c_size_t()
    assert L.ssla_hip_group_norm(None, None, 0, None) == abi.SSLA_ERR_ARG
    assert L.ssla_hip_group_norm_workspace(None, ctypes.byref(n)) == abi.SSLA_ERR_ARG
    d = norm(rows=200_000, x_stride=[9_600_000, 48], gate_stride=[9_600_000, 48],
             out_stride=[9_600_000, 48], out=P + (1 << 40))
    assert L.ssla_hip_group_norm_workspace(ctypes.addressof(d), ctypes.byref(n)) == 0 and n.value
    for ws, size in ((None, n.value), (P, n.value - 1), (P + 4, n.value)):
        assert L.ssla_hip_group_norm(ctypes.addressof(d), ws, size, None) == abi.SSLA_ERR_ARG
        assert b"workspace" in L.ssla_hip_last_error()


def test_nothing_to_do_is_no_error():
    L = lib.load()
    assert L.ssla_hip_linattn(ctypes.addressof(linattn(n_seqs=0, n_tokens=0)), None, 0, None) == 0
    assert L.ssla_hip_linattn_step(ctypes.addressof(linattn(n_seqs=0)), None) == 0
    for z in (dict(n=0), dict(rows=0), dict(channels=0)):
        assert L.ssla_hip_group_norm(ctypes.addressof(norm(**z)), None, 0, None) == 0


def test_python_refuses_tensors_off_the_gpu():
    q = torch.zeros(5, 2, 8)
    with pytest.raises(ValueError, match="GPU"):
        ops.linear_attention(q, q, q, torch.zeros(2))
    with pytest.raises(ValueError, match="GPU"):
        ops.linear_attention_step(q, q, q, torch.zeros(2), torch.zeros(5, 2, 8, 8))
    with pytest.raises(ValueError, match="GPU"):
        ops.group_norm(q, 2)


def test_python_refuses_what_is_no_argument():
    q = torch.zeros(5, 2, 8)
    for f in (lambda: ops.linear_attention(q.numpy(), q, q, q), lambda: ops.group_norm(None, 2),
              lambda: ops.linear_attention_step(q, q, q, q, None),
              lambda: ops.group_norm(q, 2, act="gelu")):
        with pytest.raises(ValueError):
            f()
    with pytest.raises(ValueError):            # the module itself
        ops._ops.group_norm(q)


@pytest.mark.gpu
def test_python_refuses_wrong_tensors():
    D = "cuda"
    q, v = torch.zeros(6, 2, 8, device=D), torch.zeros(6, 4, 8, device=D)
    g, s = torch.zeros(4, device=D), torch.zeros(6, 4, 8, 8, device=D)
    cu = torch.tensor([0, 6], dtype=torch.int32, device=D)
    la, st, gn = ops.linear_attention, ops.linear_attention_step, ops.group_norm
    bad = [lambda: la(q.double(), q.double(), v.double(), g), lambda: la(q, q.half(), v, g),
           lambda: la(q, q[:5], v, g), lambda: la(q, q, v[:, :3], g), lambda: la(q[0], q, v, g),
           lambda: la(q, q[:, :, :4], v, g), lambda: la(q, q, v, g.double()),
           lambda: la(q, q, v, g[:3]), lambda: la(q, q, v, g.cpu()),
           lambda: la(q, q, v, torch.zeros(5, 4, device=D)),
           lambda: la(q, q, v, g, torch.zeros(5, 4, 8, device=D)),
           lambda: la(q, q, v, g, torch.zeros(6, 4, 8, device=D).half()),
           lambda: la(q, q, v, g, n_seqs=4), lambda: la(q, q, v, g, n_seqs=0),
           lambda: la(q, q, v, g, max_len=3), lambda: la(q, q, v, g, cu_seqlens=cu.long()),
           lambda: la(q, q, v, g, cu_seqlens=cu.cpu()), lambda: la(q, q, v, g, cu_seqlens=cu[:0]),
           lambda: la(q, q, v, g, state_in=s.half()), lambda: la(q, q, v, g, state_in=s[:, :2]),
           lambda: la(q, q, v, g, state_in=s.transpose(2, 3)),
           lambda: la(q, q, v, g, n_seqs=6, state_in=s, state_out=s[:5]),
           lambda: la(q, q, v, g, n_seqs=3, state_out=s[:2]),
           lambda: la(q, q, v, g, state_out=s, slots=cu),
           lambda: la(q.transpose(1, 2).contiguous().transpose(1, 2), q, v, g),
           lambda: la(torch.zeros(6, 2, 257, device=D), torch.zeros(6, 2, 257, device=D), v, g),
           lambda: st(q, q, v, g, s[:5]), lambda: st(q, q, v, g, s, slots=cu[:1]),
           lambda: gn(q, 3), lambda: gn(q, 0), lambda: gn(q, 2, act="tanh"), lambda: gn(q.double(), 2),
           lambda: gn(q, 2, g), lambda: gn(q, 2, torch.zeros(8, device=D).half()),
           lambda: gn(q, 2, gate=v), lambda: gn(q, 2, out=v), lambda: gn(q.transpose(1, 2), 2),
           lambda: gn(torch.zeros(4, 5, 6, 8, device=D).transpose(1, 2), 2)]
    grad = q.clone().requires_grad_()
    bad += [lambda: la(grad, q, v, g), lambda: gn(grad, 2), lambda: la(q, q, v, g, n_seqs=1.5),
            lambda: la(q, q, v, g, scale="1"), lambda: la(q, q, v, g, cu_seqlens=cu, max_len=-1),
            lambda: la(q, q, v, g.to_sparse()), lambda: gn(q.to_sparse(), 2), lambda: st(q, q, v, g, s.to_sparse())]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was taken")
    with pytest.raises(lib.SslaHipError, match="out"):
        la(q, q, q, g[:2], q)
    with torch.no_grad():
        assert gn(grad, 2).shape == q.shape
