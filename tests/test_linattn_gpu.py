"""Linear attention (whole sequences and single tokens) against a 64-bit
recurrence, at the sizes, layouts and values where it can go wrong."""
import pytest

torch = pytest.importorskip("torch")

import seq_ref as R  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ops():
    from ssla_hip import ops as o
    return o


def make(T, H, HQ, dk, dv, dtype, seed=0, decay="token"):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    q, k, v = rnd(T, HQ, dk).to(dtype), rnd(T, HQ, dk).to(dtype), rnd(T, H, dv).to(dtype)
    g = torch.nn.functional.logsigmoid(2.0 + 1.5 * rnd(T, H)) if decay == "token" \
        else -torch.exp2(-1.0 - 6.0 * torch.rand(H, generator=gen, device=DEV))
    return q, k, v, g


def cu_of(lens):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=DEV)


SIZES = [(4, 2, 24, 24), (1, 1, 1, 1), (2, 1, 48, 33), (3, 3, 96, 96), (2, 2, 128, 128),
         (2, 1, 33, 200), (1, 1, 256, 256), (4, 4, 64, 72), (2, 2, 17, 64), (1, 1, 130, 8)]
LENGTHS = [[1], [17], [64], [65, 0, 1, 31, 32, 33], [0, 130, 0], [700, 3, 300], [513]]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lens", LENGTHS, ids=str)
@pytest.mark.parametrize("size", [SIZES[0], SIZES[3]], ids=str)
def test_lengths(dtype, lens, size):
    H, HQ, dk, dv = size
    t, T = R.TYPES[dtype], sum(lens)
    q, k, v, g = make(T, H, HQ, dk, dv, t, 1)
    s0 = torch.randn(len(lens), H, dk, dv, device=DEV)
    s1 = torch.full_like(s0, 7.0)
    out = ops().linear_attention(q, k, v, g, scale=dk ** -0.5, cu_seqlens=cu_of(lens), state_in=s0,
                                 state_out=s1)
    R.check_linear_attention(out, s1, R.linear_attention(q, k, v, g, lens, dk ** -0.5, s0), t, dk,
                             max(lens))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("decay", ["head", "token"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_sizes(dtype, decay, size):
    H, HQ, dk, dv = size
    lens, t = [70, 5, 300], R.TYPES[dtype]
    q, k, v, g = make(sum(lens), H, HQ, dk, dv, t, 2, decay)
    s1 = torch.full((3, H, dk, dv), 7.0, device=DEV)
    out = ops().linear_attention(q, k, v, g, cu_seqlens=cu_of(lens), max_len=300, state_out=s1)
    R.check_linear_attention(out, s1, R.linear_attention(q, k, v, g, lens, 1.0), t, dk, 300)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,length", [(3, 20), (2, 600), (5, 64)])
def test_equal_lengths_without_cu(dtype, n, length):
    t = R.TYPES[dtype]
    q, k, v, g = make(n * length, 2, 2, 48, 40, t, 3)
    s0 = torch.randn(n, 2, 48, 40, device=DEV)
    want = R.linear_attention(q, k, v, g, [length] * n, 0.5, s0)
    out = ops().linear_attention(q, k, v, g, scale=0.5, n_seqs=n, state_in=s0, state_out=s0)
    R.check_linear_attention(out, s0, want, t, 48, length)


def test_many_sequences_are_found():
    """More sequences than one round of the search holds, some empty."""
    lens = [(7 * i) % 5 for i in range(4100)]
    q, k, v, g = make(sum(lens), 1, 1, 8, 8, torch.float32, 4)
    s1 = torch.zeros(len(lens), 1, 8, 8, device=DEV)
    out = ops().linear_attention(q, k, v, g, cu_seqlens=cu_of(lens), max_len=4, state_out=s1)
    R.check_linear_attention(out, s1, R.linear_attention(q, k, v, g, lens, 1.0), torch.float32, 8, 4)
    # the same where sequences may be cut (an unknown longest length)
    out2 = ops().linear_attention(q, k, v, g, cu_seqlens=cu_of(lens))
    assert torch.equal(out, out2)


@pytest.mark.parametrize("n", [17, 24, 41, 64])
def test_sequences_of_unlike_lengths(n):
    """Short sequences in rounds of 16 (16 heads; the last round whole, partial,
    in either direction), some empty, with states in other slots."""
    lens = [(37 * i) % 61 for i in range(n)]
    q, k, v, g = make(sum(lens), 16, 16, 16, 72, torch.bfloat16, 41)
    slots = torch.arange(n - 1, -1, -1, dtype=torch.int32, device=DEV)
    s0 = torch.randn(n, 16, 16, 72, device=DEV)
    want = R.linear_attention(q, k, v, g, lens, 1.0, s0.flip(0))
    out = ops().linear_attention(q, k, v, g, cu_seqlens=cu_of(lens), max_len=60, state_in=s0, state_out=s0,
                                 slots=slots)
    R.check_linear_attention(out, s0.flip(0), want, torch.bfloat16, 16, 60)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lens", [[700, 300], [300], [30, 40, 10, 20]], ids=str)
def test_shared_heads_and_slices(dtype, lens):
    """Heads that share q and k, columns in four slices, segments and heads that
    do not fill eights: cut sequences and whole ones."""
    t = R.TYPES[dtype]
    q, k, v, g = make(sum(lens), 9, 3, 130, 200, t, 42)
    s1 = torch.full((len(lens), 9, 130, 200), 7.0, device=DEV)
    out = ops().linear_attention(q, k, v, g, scale=0.1, cu_seqlens=cu_of(lens), max_len=max(lens), state_out=s1)
    R.check_linear_attention(out, s1, R.linear_attention(q, k, v, g, lens, 0.1), t, 130, max(lens))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("layout", ["fused", "heads_first", "odd_offset", "padded_rows"])
def test_strides(dtype, layout):
    t, T, H, dk, dv = R.TYPES[dtype], 150, 3, 40, 24
    q, k, v, g = make(T, H, H, dk, dv, t, 5)
    out = None
    if layout == "fused":
        buf = torch.cat([q.flatten(1), k.flatten(1), v.flatten(1)], 1)
        q, k, v = (x.unflatten(1, (H, -1)) for x in buf.split([H * dk, H * dk, H * dv], 1))
    elif layout == "heads_first":
        q, k, v = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v))
        g = g.t().contiguous().t()
        out = torch.empty(H, T, dv, dtype=t, device=DEV).transpose(0, 1)
    else:
        def shifted(x):
            w = x.shape[1] * x.shape[2]
            buf = torch.empty(T, w + (3 if layout == "odd_offset" else 16), dtype=t, device=DEV)
            y = buf[:, 1:1 + w] if layout == "odd_offset" else buf[:, :w]
            y.copy_(x.flatten(1))
            return y.unflatten(1, x.shape[1:])
        q, k, v = shifted(q), shifted(k), shifted(v)
        out = shifted(torch.zeros_like(v))
    got = ops().linear_attention(q, k, v, g, out, cu_seqlens=cu_of([T]))
    assert out is None or got is out
    R.check_linear_attention(got, None, R.linear_attention(q, k, v, g, [T], 1.0), t, dk, T)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dk,dv", [(9, 15), (63, 65), (7, 97), (130, 5), (31, 2)])
def test_odd_sizes_read_and_write_their_columns_only(dtype, dk, dv):
    """Rows that are no whole pieces, in wider rows of NaN, and out in wider rows
    that keep what lies beside it."""
    t, T, H, lens = R.TYPES[dtype], 139, 2, [70, 69]
    q, k, v, g = make(T, H, H, dk, dv, t, 44)

    def wide(x):
        buf = torch.full((T, H, x.shape[2] + 3), float("nan"), dtype=t, device=DEV)
        buf[:, :, 1:-2] = x
        return buf[:, :, 1:-2]
    buf = torch.full((T, H, dv + 5), 5.0, dtype=t, device=DEV)
    s1 = torch.zeros(2, H, dk, dv, device=DEV)
    ops().linear_attention(wide(q), wide(k), wide(v), g, buf[:, :, 3:-2], cu_seqlens=cu_of(lens), max_len=70,
                           state_out=s1)
    R.check_linear_attention(buf[:, :, 3:-2], s1, R.linear_attention(q, k, v, g, lens, 1.0), t, dk, 70)
    assert (buf[:, :, :3] == 5).all() and (buf[:, :, -2:] == 5).all()


def test_rows_of_no_sequence_stay():
    T, H = 200, 2
    q, k, v, g = make(T, H, H, 32, 32, torch.bfloat16, 6)
    buf = torch.full((T, H, 40), 5.0, dtype=torch.bfloat16, device=DEV)
    cu = torch.tensor([10, 40, 40, 150], dtype=torch.int32, device=DEV)
    ops().linear_attention(q, k, v, g, buf[:, :, :32], cu_seqlens=cu)
    assert (buf[:, :, 32:] == 5).all() and (buf[:10] == 5).all() and (buf[150:] == 5).all()
    want = R.linear_attention(q[10:150], k[10:150], v[10:150], g[10:150], [30, 0, 110], 1.0)
    R.check_linear_attention(buf[10:150, :, :32], None, want, torch.bfloat16, 32, 110)


def test_max_len_cuts_longer_sequences():
    q, k, v, g = make(90, 1, 1, 16, 16, torch.float32, 7)
    out = torch.full((90, 1, 16), 5.0, device=DEV)
    ops().linear_attention(q, k, v, g, out, cu_seqlens=cu_of([60, 30]), max_len=40)
    assert (out[40:60] == 5).all()
    want = R.linear_attention(q, k, v, g, [60, 30], 1.0)
    ref = [w[:40] for w in want[:2]] + [None, None]
    R.check_linear_attention(out[:40], None, ref, torch.float32, 16, 40)


@pytest.mark.parametrize("cu", [[0, 500, 20], [-7, 30, 5000], [90, 50, 10], [60, 60, 2 ** 31 - 1],
                                [-2 ** 31, -5, -1]], ids=str)
def test_wrong_cu_stays_in_bounds(cu):
    """Values outside the tokens or falling ones: nothing past the rows is
    touched, and the call ends."""
    T, H, G = 100, 2, 64
    q, k, v, g = make(T, H, H, 16, 16, torch.bfloat16, 8)
    buf = torch.full((T + 2 * G, H, 16), 5.0, dtype=torch.bfloat16, device=DEV)
    pool = torch.full((4, H, 16, 16), 3.0, device=DEV)
    ops().linear_attention(q, k, v, g, buf[G:G + T],
                           cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=DEV),
                           state_out=pool[1:3])
    assert (buf[:G] == 5).all() and (buf[G + T:] == 5).all()
    assert (pool[0] == 3).all() and (pool[3] == 3).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind", ["none", "strong", "reset", "mixed", "growth"])
def test_decays(dtype, kind):
    t, lens, H, dk = R.TYPES[dtype], [150, 300], 2, 32
    T = sum(lens)
    q, k, v, _ = make(T, H, H, dk, 32, t, 9)
    gen = torch.Generator().manual_seed(9)
    g = torch.zeros(T, H)
    if kind == "strong":
        g = -20.0 * torch.rand(T, H, generator=gen)
    elif kind == "reset":
        g = torch.where(torch.rand(T, H, generator=gen) < 0.05, -torch.inf, -0.01)
    elif kind == "mixed":      # large steps whose sum must not blur the small ones
        g = torch.where(torch.rand(T, H, generator=gen) < 0.1, -3000.0, -0.02)
    elif kind == "growth":
        g = torch.full((T, H), 0.01)
    g = g.to(DEV)
    s0 = torch.randn(2, H, dk, 32, device=DEV)
    want = R.linear_attention(q, k, v, g, lens, 1.0, s0)
    out = ops().linear_attention(q, k, v, g, cu_seqlens=cu_of(lens), state_in=s0, state_out=s0)
    R.check_linear_attention(out, s0, want, t, dk, 300)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("what", ["q", "k", "v"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_non_finite_values_reach_no_earlier_token(dtype, what, value):
    t, lens, H, dk, dv, at = R.TYPES[dtype], [40, 600, 50], 2, 32, 48, 40 + 333
    q, k, v, g = make(sum(lens), H, H, dk, dv, t, 10)
    clean = R.linear_attention(q, k, v, g, lens, 1.0)
    {"q": q, "k": k, "v": v}[what][at, 1, 3] = value
    s1 = torch.zeros(3, H, dk, dv, device=DEV)
    out = ops().linear_attention(q, k, v, g, cu_seqlens=cu_of(lens), state_out=s1)
    bad = torch.zeros(sum(lens), H, dv, dtype=torch.bool)
    if what == "q":
        bad[at, 1] = True
    elif what == "k":
        bad[at:640, 1] = True
    else:
        bad[at:640, 1, 3] = True
    o = out.cpu()
    assert not torch.isfinite(o[bad]).any()
    ref = [torch.where(bad, 0.0, x) for x in clean[:2]] + [None, None]
    R.check_linear_attention(torch.where(bad, 0.0, o), None, ref, t, dk, 600)
    sbad = torch.zeros(3, H, dk, dv, dtype=torch.bool)
    if what == "k":
        sbad[1, 1, 3] = True
    elif what == "v":
        sbad[1, 1, :, 3] = True
    s = s1.cpu()
    assert not torch.isfinite(s[sbad]).any() and torch.isfinite(s[~sbad]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_nan_decay_reaches_no_earlier_token(dtype):
    t, lens, at = R.TYPES[dtype], [20, 600, 30], 20 + 333
    q, k, v, g = make(sum(lens), 2, 2, 32, 48, t, 43)
    want = R.linear_attention(q, k, v, g, lens, 1.0)
    g[at, 1] = float("nan")
    s1 = torch.zeros(3, 2, 32, 48, device=DEV)
    out = ops().linear_attention(q, k, v, g, cu_seqlens=cu_of(lens), state_out=s1).cpu()
    bad = torch.zeros(sum(lens), 2, 48, dtype=torch.bool)
    bad[at:620, 1] = True
    assert not torch.isfinite(out[bad]).any() and torch.isnan(s1[1, 1]).all()
    ref = [torch.where(bad, 0.0, x) for x in want[:2]] + [None, None]
    R.check_linear_attention(torch.where(bad, 0.0, out), None, ref, t, 32, 600)
    assert torch.isfinite(s1[[0, 2]]).all() and torch.isfinite(s1[1, 0]).all()


def test_values_behind_a_sequence_are_not_read_into_it():
    """Rows of the next sequence share the last tile: NaN there stays there."""
    q, k, v, g = make(100, 1, 1, 32, 32, torch.bfloat16, 11)
    want = R.linear_attention(q[:50], k[:50], v[:50], g[:50], [50], 1.0)
    for x in (q, k, v, g):
        x[50:] = float("nan")
    s = torch.zeros(1, 1, 32, 32, device=DEV)
    out = ops().linear_attention(q, k, v, g, cu_seqlens=cu_of([50]), state_out=s)
    R.check_linear_attention(out[:50], s, (want[0], want[1], want[2], want[3]), torch.bfloat16, 32, 50)


@pytest.mark.parametrize("lens", [[30, 50, 20], [300, 700, 1]], ids=str)
def test_slots(lens):
    H, dk, dv = 2, 24, 40
    q, k, v, g = make(sum(lens), H, H, dk, dv, torch.bfloat16, 12)
    base = torch.randn(6, H, dk * dv + 8, device=DEV)
    pool = base.flatten()[:6 * H * dk * dv].view(6, H, dk, dv).clone()
    was = pool.clone()
    slots = torch.tensor([4, -1, 1], dtype=torch.int32, device=DEV)
    out = torch.full((sum(lens), H, dv), 5.0, dtype=torch.bfloat16, device=DEV)
    ops().linear_attention(q, k, v, g, out, cu_seqlens=cu_of(lens), state_in=pool, state_out=pool,
                           slots=slots)
    a, b = lens[0], lens[0] + lens[1]
    assert (out[a:b] == 5).all()
    for s in (0, 2, 3, 5):
        assert torch.equal(pool[s], was[s])
    for lo, hi, s in ((0, a, 4), (b, sum(lens), 1)):
        want = R.linear_attention(q[lo:hi], k[lo:hi], v[lo:hi], g[lo:hi], [hi - lo], 1.0, was[s:s + 1])
        R.check_linear_attention(out[lo:hi], pool[s:s + 1], want, torch.bfloat16, dk, hi - lo)
    ops().linear_attention(q, k, v, g, out, cu_seqlens=cu_of(lens), state_in=pool, state_out=pool,
                           slots=torch.tensor([6, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=DEV))


def test_no_tokens_keeps_the_states():
    e = lambda *s: torch.empty(*s, device=DEV)  # noqa: E731
    s0, s1 = torch.randn(3, 2, 8, 8, device=DEV), torch.zeros(3, 2, 8, 8, device=DEV)
    cu = torch.zeros(4, dtype=torch.int32, device=DEV)
    out = ops().linear_attention(e(0, 2, 8), e(0, 2, 8), e(0, 2, 8), e(0, 2), cu_seqlens=cu,
                                 state_in=s0, state_out=s1)
    assert out.shape == (0, 2, 8) and torch.equal(s0, s1)
    ops().linear_attention(e(0, 2, 8), e(0, 2, 8), e(0, 2, 8), e(0, 2), cu_seqlens=cu, state_out=s1)
    assert (s1 == 0).all()
    out = ops().linear_attention(e(0, 2, 8), e(0, 2, 8), e(0, 2, 8), e(0, 2), n_seqs=0)
    assert out.numel() == 0
    s = torch.empty(0, 2, 8, 8, device=DEV)
    assert ops().linear_attention_step(e(0, 2, 8), e(0, 2, 8), e(0, 2, 8), e(0, 2), s).numel() == 0


# ---- single tokens ---------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B", [1, 7, 300])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_step(dtype, B, size):
    H, HQ, dk, dv = size
    if B * H * dk * dv > 10_000_000:
        B = 40
    t = R.TYPES[dtype]
    q, k, v, g = make(B, H, HQ, dk, dv, t, 13, "token" if B != 7 else "head")
    pool = torch.randn(B, H, dk, dv, device=DEV)
    want = R.linear_attention(q, k, v, g, [1] * B, 0.3, pool)
    out = ops().linear_attention_step(q, k, v, g, pool, scale=0.3)
    R.check_linear_attention(out, pool, want, t, dk, 1)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_step_slots_and_layout(dtype):
    t, B, H, dk, dv = R.TYPES[dtype], 5, 3, 24, 37
    q, k, v, g = make(B, H, H, dk, dv, t, 14)
    buf = torch.cat([q.flatten(1), k.flatten(1), v.flatten(1)], 1)
    q, k, v = (x.unflatten(1, (H, -1)) for x in buf.split([H * dk, H * dk, H * dv], 1))
    wide = torch.randn(9, H * dk * dv + 5, device=DEV)
    pool = wide[:, :H * dk * dv].unflatten(1, (H, dk, dv))
    was = wide.clone()
    slots = [8, -1, 0, 9, 3]
    out = torch.full((B, H, dv), 5.0, dtype=t, device=DEV)
    ops().linear_attention_step(q, k, v, g, pool, out,
                                slots=torch.tensor(slots, dtype=torch.int32, device=DEV))
    used = [0, 2, 4]
    idx = [slots[i] for i in used]
    before = was[:, :H * dk * dv].unflatten(1, (H, dk, dv))
    want = R.linear_attention(q[used], k[used], v[used], g[used], [1] * 3, 1.0, before[idx])
    R.check_linear_attention(out[used], pool[idx], want, t, dk, 1)
    assert (out[[1, 3]] == 5).all()
    assert torch.equal(wide[:, H * dk * dv:], was[:, H * dk * dv:])
    for s in (1, 2, 4, 5, 6, 7):
        assert torch.equal(wide[s], was[s])


def test_step_non_finite_values_stay_with_their_row():
    B, H, dk, dv = 4, 2, 16, 24
    q, k, v, g = make(B, H, H, dk, dv, torch.float32, 15)
    g[2] = -torch.inf
    pool = torch.randn(B, H, dk, dv, device=DEV)
    was = pool.clone()
    want = R.linear_attention(q, k, v, g, [1] * B, 1.0, was)
    v[1, 0, 5] = float("nan")
    out = ops().linear_attention_step(q, k, v, g, pool)
    bad = torch.zeros(B, H, dv, dtype=torch.bool)
    bad[1, 0, 5] = True
    o = out.cpu()
    assert torch.isnan(o[bad]).all()
    ref = [torch.where(bad, 0.0, x) for x in want[:2]] + [None, None]
    R.check_linear_attention(torch.where(bad, 0.0, o), None, ref, torch.float32, dk, 1)


# ---- places, streams, graphs -------------------------------------------------------

def test_offsets_past_32_bits():
    """A pool whose last slot and rows whose last token lie past 2^31 elements."""
    H, dk, dv = 1, 16, 16
    far = 2 ** 31 + 4096
    mem = torch.empty(far + 4096, device=DEV)
    pool = mem.as_strided((2, H, dk, dv), (far, dk * dv, dv, 1))
    pool.copy_(torch.randn(2, H, dk, dv, device=DEV))
    q, k, v, g = make(2, H, H, dk, dv, torch.float32, 16)
    want = R.linear_attention(q, k, v, g, [1, 1], 1.0, pool)
    out = ops().linear_attention_step(q, k, v, g, pool)
    R.check_linear_attention(out, pool, want, torch.float32, dk, 1)

    T, step = 65, 2 ** 25
    rows = mem.as_strided((T, 1, 64), (step, 64, 1))
    q, k, v, g = make(T, 1, 1, 16, 16, torch.float32, 17)
    rows[:, :, :16], rows[:, :, 16:32], rows[:, :, 32:48] = q, k, v
    out = rows[:, :, 48:]
    want = R.linear_attention(q, k, v, g, [T], 1.0)
    ops().linear_attention(rows[:, :, :16], rows[:, :, 16:32], rows[:, :, 32:48], g, out,
                           cu_seqlens=cu_of([T]))
    R.check_linear_attention(out, None, want, torch.float32, 16, T)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_reruns_are_equal(dtype):
    q, k, v, g = make(2000, 4, 2, 64, 64, R.TYPES[dtype], 18)
    cu = cu_of([1200, 800])
    a = ops().linear_attention(q, k, v, g, cu_seqlens=cu)
    for _ in range(3):
        assert torch.equal(a, ops().linear_attention(q, k, v, g, cu_seqlens=cu))


def test_streams():
    """Two calls at once on two streams, each with its own workspace."""
    sets = [make(3000, 2, 2, 64, 64, torch.bfloat16, 19 + i) for i in range(2)]
    want = [ops().linear_attention(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        got = []
        for s, st in zip(sets, streams):
            with torch.cuda.stream(st):
                got.append(ops().linear_attention(*s))
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert torch.equal(a, b)


def test_graphs():
    """Two captured graphs (a cut prompt; tokens behind it), replayed in turn with
    eager work between, with other inputs, lengths and slots in place."""
    o = ops()
    H, dk, dv, T, B = 2, 32, 48, 900, 3
    q, k, v, g = make(T, H, H, dk, dv, torch.bfloat16, 21)
    cu = cu_of([500, 100, 300])
    slots = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    pool = torch.zeros(4, H, dk, dv, device=DEV)
    out, tok = torch.zeros(T, H, dv, dtype=torch.bfloat16, device=DEV), None
    qs, ks, vs, gs = make(B, H, H, dk, dv, torch.bfloat16, 22)

    def prompt():
        o.linear_attention(q, k, v, g, out, cu_seqlens=cu, state_out=pool, slots=slots)

    prompt()
    tok = o.linear_attention_step(qs, ks, vs, gs, pool, slots=slots)
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        prompt()
    with torch.cuda.graph(g2):
        o.linear_attention_step(qs, ks, vs, gs, pool, tok, slots=slots)
    for i, (lens, sl) in enumerate((([500, 100, 300], [0, 1, 2]), ([0, 899, 1], [3, 0, 1]),
                                    ([300, 300, 300], [2, -1, 0]))):
        nq, nk, nv, ng = make(T, H, H, dk, dv, torch.bfloat16, 30 + i)
        for a, b in ((q, nq), (k, nk), (v, nv), (g, ng)):
            a.copy_(b)
        cu.copy_(cu_of(lens))
        slots.copy_(torch.tensor(sl, dtype=torch.int32))
        out.zero_(), pool.zero_(), tok.zero_()
        g1.replay()
        g2.replay()
        g2.replay()
        torch.cuda.synchronize()
        got = out.clone(), pool.clone(), tok.clone()
        out.zero_(), pool.zero_(), tok.zero_()
        prompt()
        for _ in range(2):
            o.linear_attention_step(qs, ks, vs, gs, pool, tok, slots=slots)
        torch.cuda.synchronize()
        for a, b in zip(got, (out, pool, tok)):
            assert torch.equal(a, b)


# ---- together ------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_prompt_then_tokens_then_norm(dtype):
    """A prompt fills the pool, tokens follow one at a time; heads are normalised
    and gated: the same as one long call, and as the 64-bit form."""
    o, t = ops(), R.TYPES[dtype]
    H, dk, dv, lens, more = 4, 48, 64, [65, 290], 6
    full = [n + more for n in lens]
    T = sum(full)
    q, k, v, g = make(T, H, 2, dk, dv, t, 40)
    gate = torch.randn(T, H * dv, device=DEV).to(t)
    w = torch.randn(H * dv, device=DEV).to(t)
    starts = [0, full[0]]
    head = torch.cat([torch.arange(s, s + n) for s, n in zip(starts, lens)]).to(DEV)
    pool = torch.zeros(2, H, dk, dv, device=DEV)
    att = torch.empty(T, H, dv, dtype=t, device=DEV)
    att[head] = o.linear_attention(q[head], k[head], v[head], g[head], scale=dk ** -0.5,
                                   cu_seqlens=cu_of(lens), state_in=pool, state_out=pool)
    for i in range(more):
        at = torch.tensor([s + n + i for s, n in zip(starts, lens)], device=DEV)
        att[at] = o.linear_attention_step(q[at], k[at], v[at], g[at], pool, scale=dk ** -0.5)
    ref = R.linear_attention(q, k, v, g, full, dk ** -0.5)
    R.check_linear_attention(att, pool, ref, t, dk, max(full))
    y = o.group_norm(att.flatten(1), H, w, gate=gate, act="silu")
    R.check_group_norm(y, R.group_norm(att.flatten(1), H, w, None, 1e-5, "silu", gate), t)


def test_tokens_from_a_drain(stub_dir):
    """Feature rows of a drain's output slots (98 words a slot, features at the
    second word) as tokens, read where the drain left them."""
    from ssla_hip import abi, events, hybrid
    rec = events.blob_records(1500, seed=3)
    with hybrid.Drain.from_weights_dir(stub_dir) as d:
        (out,) = d.drain([events.to_records(rec)])[0]
    slots = torch.from_numpy(out.view("<i4").reshape(len(out), -1).copy()).to(DEV)
    feat = slots[:, 2:].view(torch.float32).unflatten(1, (2, 48))
    assert feat.stride() == (98, 48, 1) and abi.C3 == 96
    g = torch.full((2,), -0.05, device=DEV)
    got = ops().linear_attention(feat, feat, feat, g, scale=48 ** -0.5)
    R.check_linear_attention(got, None, R.linear_attention(feat, feat, feat, g, [1500], 48 ** -0.5),
                             torch.float32, 48, 1500)
    y = ops().group_norm(slots[:, 2:].view(torch.float32), 2, act="silu")
    R.check_group_norm(y, R.group_norm(feat.flatten(1), 2, None, None, 1e-5, "silu"), torch.float32)
