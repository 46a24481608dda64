"""Linear attention with heads of more than 128 in whole and cut sequences, eager
and captured."""
import pytest

torch = pytest.importorskip("torch")

import seq_ref as R  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(lens, H, HQ, dk, dv, dtype, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    T = sum(lens)
    q, k, v = rnd(T, HQ, dk).to(dtype), rnd(T, HQ, dk).to(dtype), rnd(T, H, dv).to(dtype)
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=DEV)
    return q, k, v, torch.nn.functional.logsigmoid(2.0 + 1.5 * rnd(T, H)), cu, rnd(len(lens), H, dk, dv)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lens", [[700, 0, 321, 1], [200, 150, 33]], ids=["cut", "whole"])
@pytest.mark.parametrize("dk,dv", [(256, 256), (200, 136), (255, 129)])
def test_wide_heads(dtype, lens, dk, dv):
    from ssla_hip import ops
    t = R.TYPES[dtype]
    q, k, v, g, cu, s = make(lens, 2, 1, dk, dv, t, 90)
    want = R.linear_attention(q, k, v, g, lens, dk ** -0.5, s)
    out = ops.linear_attention(q, k, v, g, scale=dk ** -0.5, cu_seqlens=cu, max_len=max(lens), state_in=s,
                               state_out=s)
    R.check_linear_attention(out, s, want, t, dk, max(lens))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_graph_of_cut_wide_heads(dtype):
    """States updated in place by replays, with eager work between them."""
    from ssla_hip import ops
    t, lens = R.TYPES[dtype], [450, 321]
    q, k, v, g, cu, s = make(lens, 2, 2, 256, 256, t, 91)
    pool, out = s.clone(), torch.zeros_like(v)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.linear_attention(q, k, v, g, out, scale=0.0625, cu_seqlens=cu, state_in=pool, state_out=pool)
    eager = s.clone()
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        want = ops.linear_attention(q, k, v, g, scale=0.0625, cu_seqlens=cu, state_in=eager, state_out=eager)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(pool, eager)
        q.copy_(q.roll(1, 0))


def test_two_calls_at_once_with_states():
    """Cut calls on two streams, each with its own pool, updated in place."""
    from ssla_hip import ops
    sets = [make([500, 65, 300], 3, 3, 40, 72, torch.bfloat16, 92 + i) for i in range(2)]
    want = []
    for q, k, v, g, cu, s in sets:
        pool = s.clone()
        want.append((ops.linear_attention(q, k, v, g, cu_seqlens=cu, state_in=pool, state_out=pool), pool))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        pools = [x[5].clone() for x in sets]
        torch.cuda.synchronize()
        got = []
        for (q, k, v, g, cu, _), pool, st in zip(sets, pools, streams):
            with torch.cuda.stream(st):
                got.append(ops.linear_attention(q, k, v, g, cu_seqlens=cu, state_in=pool, state_out=pool))
        torch.cuda.synchronize()
        for (o, p), a, b in zip(want, got, pools):
            assert torch.equal(o, a) and torch.equal(p, b)
