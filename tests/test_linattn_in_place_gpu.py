"""Whole sequences whose states are read from and written to the same pool."""
import pytest

torch = pytest.importorskip("torch")

import seq_ref as R  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ops():
    from ssla_hip import ops as o
    return o


def make(lens, H, dk, dv, dtype, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    T = sum(lens)
    q, k, v = rnd(T, H, dk).to(dtype), rnd(T, H, dk).to(dtype), rnd(T, H, dv).to(dtype)
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=DEV)
    return q, k, v, torch.nn.functional.logsigmoid(2.0 + 1.5 * rnd(T, H)), cu, \
        rnd(len(lens), H, dk, dv)


@pytest.mark.parametrize("busy", [False, True], ids=["alone", "beside_another_stream"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("H,dk,dv", [(3, 64, 64), (16, 24, 130), (1, 200, 72)])
def test_one_pool_gives_what_two_pools_give(dtype, H, dk, dv, busy):
    """Sequences cut into segments of 64 tokens, the last of one token, beside
    sequences of one segment: the same bits, and the 64-bit form's values."""
    lens, t = [641, 0, 321, 65, 64, 1], R.TYPES[dtype]
    q, k, v, g, cu, s0 = make(lens, H, dk, dv, t, 50)
    two = torch.full_like(s0, 7.0)
    want = ops().linear_attention(q, k, v, g, scale=0.2, cu_seqlens=cu, state_in=s0, state_out=two)
    R.check_linear_attention(want, two, R.linear_attention(q, k, v, g, lens, 0.2, s0), t, dk, max(lens))
    other, a = torch.cuda.Stream(), torch.randn(2048, 2048, device=DEV)
    torch.cuda.synchronize()
    for _ in range(5):
        if busy:
            with torch.cuda.stream(other):
                for _ in range(4):
                    a @ a
        pool = s0.clone()
        got = ops().linear_attention(q, k, v, g, scale=0.2, cu_seqlens=cu, state_in=pool, state_out=pool)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(pool, two)


def test_one_pool_without_cu_seqlens():
    """Equal lengths, cut: the same through the other way of finding segments."""
    lens = [321, 321]
    q, k, v, g, _, s0 = make(lens, 3, 48, 40, torch.bfloat16, 51)
    two, pool = torch.empty_like(s0), s0.clone()
    want = ops().linear_attention(q, k, v, g, n_seqs=2, state_in=s0, state_out=two)
    R.check_linear_attention(want, two, R.linear_attention(q, k, v, g, lens, 1.0, s0), torch.bfloat16, 48, 321)
    got = ops().linear_attention(q, k, v, g, n_seqs=2, state_in=pool, state_out=pool)
    assert torch.equal(got, want) and torch.equal(pool, two)
