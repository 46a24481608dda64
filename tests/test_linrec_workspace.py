"""The recurrence's workspace: there is one for every call of more than one tile, and a
call without it is refused."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from ssla_hip import abi, lib  # noqa: E402
from test_ops_train import P, at, linrec, linrec_grad  # noqa: E402

FAR = dict(out=P + (1 << 40), gate=P + (2 << 40), v=P + (3 << 40), q=P + (4 << 40))


@pytest.mark.parametrize("tokens,channels,dtype", [(1_000_000, 32, abi.SSLA_BF16), (4097, 1, abi.SSLA_F32),
                                                   (200, 512, abi.SSLA_F16), (300, 2048, abi.SSLA_F32)])
def test_calls_of_more_than_one_tile_need_one(tokens, channels, dtype):
    L, n = lib.load(), ctypes.c_size_t(7)
    d = linrec(n_tokens=tokens, n_seqs=1, channels=channels, dtype=dtype, **FAR,
               **{k + "_stride": channels for k in ("gate", "v", "q", "out", "state_in", "state_out")})
    g = linrec_grad(**{k + "_stride": channels for k in ("dout", "dgate", "dv", "dq", "dstate_in", "dstate_out")})
    assert L.ssla_hip_linrec_workspace(at(d), ctypes.byref(n)) == 0 and n.value > 0
    for ws, size in ((None, n.value), (P, n.value - 1), (P + 8, n.value)):
        assert L.ssla_hip_linrec(at(d), ws, size, None) == abi.SSLA_ERR_ARG
        assert b"workspace" in L.ssla_hip_last_error()
        assert L.ssla_hip_linrec_backward(at(d), at(g), ws, size, None) == abi.SSLA_ERR_ARG
        assert b"workspace" in L.ssla_hip_last_error()
