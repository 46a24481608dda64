"""The recurrence at counts near the largest: what the host compiler evaluates, and a call of
more than 2^30 tokens."""
import shutil
import subprocess
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

import train_ref as R  # noqa: E402

ROOT = Path(__file__).resolve().parent.parent
MOST = (1 << 31) - (1 << 16)


def test_sequences_begun_before_a_token(tmp_path):
    """Evaluated by the compiler, to which an overflow is an error."""
    cxx = shutil.which("g++")
    if not cxx:
        pytest.skip("no compiler")
    at = {(0, 1), (0, MOST), (1, 1), (1, MOST), (1 << 30, 1_100_000_000), (MOST - 1, MOST), (MOST, MOST), (MOST, 1),
          (MOST, MOST // 2), (MOST // 2 + 1, MOST // 2), (MOST // 2, MOST // 2)}
    at |= {(t, n) for t in range(0, 70, 3) for n in (1, 2, 7, 16, 33)}
    lines = [f"static_assert(ssla::linrec_begun({t}, {n}) == {-(-t // n)});" for t, n in sorted(at)]
    src = tmp_path / "begun.cpp"
    src.write_text('#include "linrec.h"\n' + "\n".join(lines) + "\n")
    r = subprocess.run([cxx, "-std=c++17", "-fsyntax-only", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                        f"-I{ROOT}/include", f"-I{ROOT}/ssla-rt_amd/csrc", str(src)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[:2000]


@pytest.mark.gpu
@pytest.mark.parametrize("n_seqs,length", [(1, (1 << 30) + 100_001), (2, (1 << 29) + 70_001)])
def test_more_tokens_than_2_to_the_30(n_seqs, length):
    """One channel.  The gates forget: after 20000 tokens of sigmoid(1.25) = 0.777 or less
    nothing is left of a state, so tokens are as in a short call on those about them, to
    both calls' errors.  A step's is (1.25 + 16) 2^-24 of at most 16 / (1 - 0.777) = 72, and
    4.5 steps' add up: 3.3e-4, in two calls less than 2^-10.  A gate's gradient is a product of
    dh (at most 4.5, error 4.5 * 4.5 * 2 * 17.25 * 2^-24 = 4.2e-5), the state before and 1/4: 1/4 (72 *
    4.2e-5 + 4.5 * 3.3e-4 + 2 * 17.25 * 2^-24 * 4.5 * 72) = 1.3e-3, in two calls less than 2^-8."""
    from ssla_hip import ops
    total, tail, warm = n_seqs * length, 50_000, 20_000
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    gen = torch.Generator(device="cuda").manual_seed(31)
    gate = torch.empty(total, 1, dtype=torch.float16, device="cuda").uniform_(-1.25, 1.25, generator=gen)
    v = torch.empty(total, 1, dtype=torch.float16, device="cuda").uniform_(-16, 16, generator=gen)
    state = torch.full((n_seqs, 1), 3.0, device="cuda")
    out, last = ops.linear_recurrence(gate, v, n_seqs=n_seqs, state_in=state, return_state=True)

    def near(got, want, rel=2 * R.half_step(torch.float16), off=2.0 ** -10):
        assert ((got.double() - want.double()).abs() <= off + rel * want.double().abs()).all()

    for s in range(n_seqs):
        a, b = s * length, (s + 1) * length
        x, h = ops.linear_recurrence(gate[b - tail:b], v[b - tail:b], return_state=True)
        near(out[b - tail + warm:b], x[warm:])
        near(last[s], h[0], 0.0)
        x = ops.linear_recurrence(gate[a:a + tail], v[a:a + tail], state_in=state[s:s + 1])
        near(out[a:a + tail], x)
    # and at some tokens between
    for t in range(warm, total - tail, total // 7):
        if (t - warm) // length == (t + tail - 1) // length:
            x = ops.linear_recurrence(gate[t - warm:t + tail], v[t - warm:t + tail])
            near(out[t:t + tail], x[warm:])
    del out, x
    ga = gate.requires_grad_()
    dout = torch.ones(1, 1, dtype=torch.float16, device="cuda").expand(total, 1)
    y = ops.linear_recurrence(ga, v, n_seqs=n_seqs, state_in=state)
    (dg,) = torch.autograd.grad(y, ga, dout)
    del y
    # nothing comes to the last token from behind, in either call
    gb = gate[total - tail:].detach().requires_grad_()
    (want,) = torch.autograd.grad(ops.linear_recurrence(gb, v[total - tail:]), gb, dout[total - tail:])
    near(dg[total - tail + warm:], want[warm:], off=2.0 ** -8)
