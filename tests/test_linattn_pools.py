"""State pools that lie in one another: slots of both in turn."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

import seq_ref as R  # noqa: E402
import test_ops as T  # noqa: E402
from ssla_hip import abi, lib  # noqa: E402

STATE = 4 * 32 * 64


@pytest.mark.parametrize("apart,stride,ok", [
    (STATE, 2 * STATE, True), (-STATE, 2 * STATE, True), (STATE + 8, 2 * STATE + 8, True),
    (3 * STATE, 2 * STATE, True), (2 * STATE, 2 * STATE, False), (STATE - 1, 2 * STATE, False),
    (STATE + 1, 2 * STATE, False), (1, STATE, False), (STATE, STATE, False), (-1, 2 * STATE, False),
    (STATE, 2 * STATE - 1, False), (8 * STATE, STATE, True), (-8 * STATE, STATE, True)], ids=str)
def test_which_pools_overlap(apart, stride, ok):
    d = T.linattn(n_slots=8, n_seqs=2, state_stride=stride)
    d.state_out = d.state_in + 4 * apart
    n = ctypes.c_size_t()
    rc = lib.load().ssla_hip_linattn_workspace(ctypes.addressof(d), ctypes.byref(n))
    assert rc == (abi.SSLA_OK if ok else abi.SSLA_ERR_ARG)
    if not ok:
        assert b"overlap" in lib.load().ssla_hip_last_error()


@pytest.mark.gpu
def test_slots_of_two_pools_in_turn():
    from ssla_hip import ops
    dev, lens, H, dk, dv = "cuda", [300, 40, 70], 2, 24, 40
    gen = torch.Generator(device=dev)
    gen.manual_seed(80)
    rnd = lambda *s: torch.randn(*s, generator=gen, device=dev)  # noqa: E731
    n = sum(lens)
    q, k, v, g = rnd(n, H, dk), rnd(n, H, dk), rnd(n, H, dv), -rnd(n, H).abs()
    cu = torch.tensor([0, 300, 340, 410], dtype=torch.int32, device=dev)
    both = rnd(3, 2, H, dk, dv)
    was = both.clone()
    out = ops.linear_attention(q, k, v, g, cu_seqlens=cu, state_in=both[:, 0], state_out=both[:, 1])
    R.check_linear_attention(out, both[:, 1], R.linear_attention(q, k, v, g, lens, 1.0, was[:, 0]), torch.float32,
                             dk, 300)
    assert torch.equal(both[:, 0], was[:, 0])
