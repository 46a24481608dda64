"""The recurrence's tiles without one another: a call whose workgroups do not wait
makes the missing maps itself, and gives the same bits."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from ssla_hip import abi, lib  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"f32": (torch.float32, abi.SSLA_F32), "bf16": (torch.bfloat16, abi.SSLA_BF16),
         "f16": (torch.float16, abi.SSLA_F16)}


def both(wait, gate, v, q, cu, n_seqs, s_in, s_out, dout, dstate, slots=None):
    """Forward and backward pass over the C ABI; slots: forward in the place of s_in."""
    L = lib.load()
    T, C = v.shape
    d, g = abi.SslaHipLinRec(), abi.SslaHipLinRecGrad()
    d.dtype = {t: n for t, n in TYPES.values()}[v.dtype]
    d.channels, d.n_seqs, d.n_tokens, d.wait_us = C, n_seqs, T, wait
    d.n_slots = n_seqs if s_in is None else s_in.shape[0]
    out = torch.zeros_like(v)
    keep = [out]
    for n, t in (("gate", gate), ("v", v), ("q", q), ("out", out)):
        if t is not None:
            setattr(d, n, t.data_ptr())
            setattr(d, n + "_stride", t.stride(0))
    for n, t in (("state_in", s_in), ("state_out", s_out)):
        if t is not None:
            setattr(d, n, t.data_ptr())
            setattr(d, n + "_stride", t.stride(0))
    if cu is not None:
        d.cu_seqlens = cu.data_ptr()
    if slots is not None:
        d.slots = slots.data_ptr()
    n = ctypes.c_size_t()

    def room(f):
        lib.check(f(ctypes.addressof(d), ctypes.byref(n)))
        keep.append(torch.empty(max(1, n.value), dtype=torch.uint8, device=DEV))
        return keep[-1].data_ptr(), n.value

    grads = []
    if slots is None:
        d.carries = room(L.ssla_hip_linrec_carries)[0]
    stream = torch.cuda.current_stream().cuda_stream
    lib.check(L.ssla_hip_linrec(ctypes.addressof(d), *room(L.ssla_hip_linrec_workspace), stream), "linrec")
    if slots is None:
        grads = [torch.zeros_like(v) for _ in range(3)] + [torch.zeros(n_seqs, C, device=DEV)]
        names = ["dgate", "dv", "dq", "dstate_in"]
        for name, t in list(zip(names, grads)) + [("dout", dout), ("dstate_out", dstate)]:
            if t is None or (name == "dq" and q is None):
                continue
            setattr(g, name, t.data_ptr())
            setattr(g, name + "_stride", t.stride(0))
        lib.check(L.ssla_hip_linrec_backward(ctypes.addressof(d), ctypes.addressof(g),
                                             *room(L.ssla_hip_linrec_workspace), stream), "linrec_backward")
    torch.cuda.synchronize()
    return [out] + grads


def inputs(dtype, c, total, n_seqs, seed):
    gen = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    t = TYPES[dtype][0]
    x = [(1.5 * rnd(total, c) + 2.0).to(t).to(DEV), rnd(total, c).to(t).to(DEV), rnd(total, c).to(t).to(DEV)]
    return x, rnd(n_seqs, c).to(DEV), rnd(total, c).to(t).to(DEV), rnd(n_seqs, c).to(DEV)


LENGTHS = {"one": [1500], "ragged": [700, 1, 0, 2, 900, 3, 511, 128, 64, 5], "gap": [40, 900, 300]}


@pytest.mark.parametrize("dtype,c", [("f32", 24), ("f32", 70), ("bf16", 64), ("bf16", 37), ("f16", 130), ("f32", 2)])
@pytest.mark.parametrize("name", list(LENGTHS) + ["even"])
@pytest.mark.parametrize("read", [True, False])
def test_same_bits(dtype, c, name, read):
    cu, n = None, 3
    total = 1800
    if name != "even":
        lens = LENGTHS[name]
        n = len(lens)
        first = 33 if name == "gap" else 0
        cu = torch.tensor([first + sum(lens[:i]) for i in range(n + 1)], dtype=torch.int32, device=DEV)
        total = int(cu[-1]) + (200 if name == "gap" else 0)
    (gate, v, q), s, dout, dstate = inputs(dtype, c, total, n, 3)
    args = (gate, v, q if read else None, cu, n, s)
    last = [torch.zeros_like(s) for _ in range(3)]
    want = both(0, *args, last[0], dout, dstate)
    for i, wait in enumerate((-1, 1)):
        got = both(wait, *args, last[1 + i], dout, dstate)
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(last[1 + i], last[0]), wait


@pytest.mark.parametrize("dtype,c", [("f32", 70), ("bf16", 64)])
def test_same_bits_in_one_pool(dtype, c):
    """States read and written in one pool, sequences within a tile and over several."""
    lens = LENGTHS["ragged"] * 2
    n = len(lens)
    cu = torch.tensor([sum(lens[:i]) for i in range(n + 1)], dtype=torch.int32, device=DEV)
    (gate, v, q), pool, _, _ = inputs(dtype, c, int(cu[-1]), n + 4, 5)
    slots = torch.randperm(n + 4, generator=torch.Generator().manual_seed(6))[:n].to(torch.int32)
    slots[3] = -1
    slots = slots.to(DEV)
    pools = [pool.clone() for _ in range(3)]
    want = both(0, gate, v, q, cu, n, pools[0], pools[0], None, None, slots)
    for i, wait in enumerate((-1, 1)):
        got = both(wait, gate, v, q, cu, n, pools[1 + i], pools[1 + i], None, None, slots)
        assert torch.equal(got[0], want[0]) and torch.equal(pools[1 + i], pools[0]), wait
