"""The recurrence with first and last states in one pool: the same bits as with two,
whatever order its tiles come in."""
import pytest

torch = pytest.importorskip("torch")

from ssla_hip import abi  # noqa: E402
from test_linrec_alone_gpu import DEV, both, inputs  # noqa: E402

pytestmark = pytest.mark.gpu


def one_and_two(dtype, c, cu, n, total, waits, seed, slots=None, read=True):
    """A call with two pools, then with one for each of `waits`."""
    (gate, v, q), pool, _, _ = inputs(dtype, c, total, n + 4, seed)
    if slots is None:
        slots = torch.randperm(n + 4, generator=torch.Generator().manual_seed(seed))[:n].to(torch.int32).to(DEV)
    q = q if read else None
    last = pool.clone()
    want = both(0, gate, v, q, cu, n, pool, last, None, None, slots)[0]
    for wait in waits:
        place = pool.clone()
        got = both(wait, gate, v, q, cu, n, place, place, None, None, slots)[0]
        assert torch.equal(got, want), wait
        assert torch.equal(place, last), wait


@pytest.mark.parametrize("dtype,c,tile", [("f32", 1024, 128), ("bf16", 1024, 128), ("f16", 1021, 128)])
def test_last_tiles_end_before_first_ones_begin(dtype, c, tile):
    """More workgroups (4000) than a card of 256 compute units holds at three or four each,
    the last tile's first: they store the sequence's last state, made without the others,
    before the first tile is there to read its first one."""
    one_and_two(dtype, c, None, 1, 250 * tile - 5, (abi.SSLA_LINREC_ALONE,), 21)


@pytest.mark.parametrize("dtype,c", [("f32", 2), ("f32", 70), ("bf16", 37), ("bf16", 64), ("f16", 130), ("bf16", 1024)])
@pytest.mark.parametrize("name", ["ends", "ragged", "gap", "even", "empty at tiles' ends"])
def test_one_pool(dtype, c, name):
    lens = {"ends": [64, 63, 1, 129, 127, 255, 257, 128, 513, 511, 1, 1500, 548, 2048],
            "ragged": [700, 1, 0, 2, 900, 3, 511, 128, 64, 5], "gap": [40, 900, 1300],
            "empty at tiles' ends": [0, 2048, 0, 0, 1024, 0, 128, 0, 0, 64, 3000, 0], "even": [683] * 3}[name]
    cu, n, first = None, len(lens), 33 if name == "gap" else 0
    if name != "even":
        cu = torch.tensor([first + sum(lens[:i]) for i in range(n + 1)], dtype=torch.int32, device=DEV)
    total = first + sum(lens) + (200 if name == "gap" else 0)
    one_and_two(dtype, c, cu, n, total, (0, -1, abi.SSLA_LINREC_ALONE), 22, read=c % 2 == 0)


def test_many_sequences():
    """More than a wave looks through at once, most of them within a tile, some over many."""
    n = 20000
    lens = [0 if i % 7 == 3 else 6000 if i % 6000 == 5 else i % 5 for i in range(n)]
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(DEV)
    one_and_two("bf16", 48, cu, n, int(cu[-1]), (0, -1), 23)
    # passed over, so that there is no first state to keep; and a first boundary behind tiles' ends
    slots = torch.arange(n, dtype=torch.int32, device=DEV)
    slots[5::6000] = -1
    slots[6005] = 1 << 30
    one_and_two("f32", 48, cu, n, int(cu[-1]) + 3000, (0, -1), 24, slots)
    one_and_two("f32", 48, (cu + 2500).contiguous(), n, int(cu[-1]) + 3000, (0, -1), 25, slots)


def test_captured():
    """A call in one pool in a graph: every replay goes on from the states of the last one."""
    from ssla_hip import ops
    (gate, v, q), pool, _, _ = inputs("bf16", 200, 3000, 3, 26)
    cu = torch.tensor([0, 1700, 1700, 3000], dtype=torch.int32, device=DEV)
    place, out = pool.clone(), torch.empty_like(v)
    call = lambda a, b, o: ops.linear_recurrence(gate, v, q, o, cu_seqlens=cu, state_in=a, state_out=b)  # noqa: E731
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad():
        with torch.cuda.graph(graph):
            call(place, place, out)
        for i in range(4):
            v.add_(0.25)
            last = pool.clone()
            want = call(pool, last, None)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(place, last), i
            pool.copy_(last)


def test_calls_at_once():
    """Four streams, each with a call in one pool that fills the card by itself."""
    from ssla_hip import ops
    cu = torch.tensor([0, 9000, 9000, 9001, 20000], dtype=torch.int32, device=DEV)
    calls = []
    for i in range(4):
        (gate, v, q), pool, _, _ = inputs("bf16", 1024, 20000, 4, 30 + i)
        last = pool.clone()
        with torch.no_grad():
            want = ops.linear_recurrence(gate, v, q, cu_seqlens=cu, state_in=pool, state_out=last)
        calls.append((gate, v, q, pool, torch.empty_like(want), want, last, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for turn in range(5):
        places = [c[3].clone() for c in calls]
        torch.cuda.synchronize()
        for (gate, v, q, _, out, _, _, stream), place in zip(calls, places):
            with torch.cuda.stream(stream), torch.no_grad():
                ops.linear_recurrence(gate, v, q, out, cu_seqlens=cu, state_in=place, state_out=place)
        torch.cuda.synchronize()
        for (_, _, _, _, out, want, last, _), place in zip(calls, places):
            assert torch.equal(out, want) and torch.equal(place, last), turn
