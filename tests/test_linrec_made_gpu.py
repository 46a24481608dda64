"""The recurrence's maps as a tile makes them for another: with SSLA_LINREC_ALONE no
workgroup publishes its own, so every map that a state goes through comes from there."""
import pytest

torch = pytest.importorskip("torch")

from ssla_hip import abi  # noqa: E402
from test_linrec_alone_gpu import DEV, both, inputs  # noqa: E402

pytestmark = pytest.mark.gpu

# tiles have 32 to 2048 tokens: sequences that end with a tile, a token before and behind
# its end, in its last thread; a last tile of one token, of all but one
LENGTHS = {"ends": [64, 63, 1, 129, 127, 255, 257, 128, 513, 511, 1], "last": [1025], "short of one": [2047],
           "ragged": [700, 1, 0, 2, 900, 3, 511, 128, 64, 5], "gap": [40, 900, 300]}


@pytest.mark.parametrize("dtype,c", [("f32", 2), ("f32", 24), ("f32", 70), ("bf16", 37), ("bf16", 64), ("f16", 130)])
@pytest.mark.parametrize("name", list(LENGTHS) + ["even"])
@pytest.mark.parametrize("read", [True, False])
def test_made_maps_give_the_same_bits(dtype, c, name, read):
    cu, n, total = None, 3, 3 * 683
    if name != "even":
        lens = LENGTHS[name]
        n, first = len(lens), 33 if name == "gap" else 0
        cu = torch.tensor([first + sum(lens[:i]) for i in range(n + 1)], dtype=torch.int32, device=DEV)
        total = int(cu[-1]) + (200 if name == "gap" else 0)
    (gate, v, q), s, dout, dstate = inputs(dtype, c, total, n, 13)
    last = [torch.zeros_like(s) for _ in range(2)]
    args = (gate, v, q if read else None, cu, n, s)
    want = both(0, *args, last[0], dout, dstate)
    got = both(abi.SSLA_LINREC_ALONE, *args, last[1], dout, dstate)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(last[1], last[0])
