"""The workspace of cut sequences: its size whatever the number of sequences, and
sequences of all places and lengths in it."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

import seq_ref as R  # noqa: E402
from ssla_hip import abi, lib  # noqa: E402

DEV = "cuda"


def size(n_tokens, n_seqs, max_len, heads=16, dk=128, dv=128, dtype=abi.SSLA_BF16):
    d = abi.SslaHipLinAttn()
    d.dtype, d.heads, d.qk_heads, d.dk, d.dv = dtype, heads, heads, dk, dv
    d.n_seqs, d.max_len, d.n_tokens = n_seqs, max_len, n_tokens
    d.q = d.k = d.v = d.log_decay = d.cu_seqlens = 1 << 20
    d.out = 1 << 24
    for n, w in (("q", dk), ("k", dk), ("v", dv), ("out", dv)):
        getattr(d, n + "_stride")[:] = [heads * w, w]
    d.decay_stride[:] = [heads, 1]
    n = ctypes.c_size_t(7)
    lib.check(lib.load().ssla_hip_linattn_workspace(ctypes.addressof(d), ctypes.byref(n)))
    return n.value


@pytest.mark.parametrize("n", [1, 10, 511, 5000])
def test_short_sequences_beside_a_long_one_take_no_states(n):
    """Segments have 64 tokens at least, and two states for each 64 tokens are enough."""
    state = 16 * (128 * 128 + 1) * 4
    assert 16 * state <= size(4000 + n, n + 1, 4000) <= 2 * ((4000 + n) // 64) * state


def test_a_serving_batch():
    """511 single tokens and a prompt of 4000: segments of 256, 17 whole ones."""
    assert size(4511, 512, 4000) == 2 * 17 * 16 * (128 * 128 + 1) * 4
    # one sequence alone: a state a segment (64 tokens) and one for its odd beginning
    assert size(2000, 1, 2000, heads=4) == (2000 // 64 + 1) * 4 * (128 * 128 + 1) * 4


def test_sizes_at_the_largest_counts():
    """The size at the largest number of tokens, and its refusal beyond."""
    most = (1 << 31) - (1 << 16)
    # one sequence of one head: 127 whole segments of 2^24 tokens and the rest
    assert size(most, 1, most, heads=1) == 128 * (128 * 128 + 1) * 4
    assert size(most, 1_000_000, most, heads=1) == 2 * 127 * (128 * 128 + 1) * 4
    # 128 sequences of 2^24 tokens: nothing is cut
    assert size(most, 128, 1 << 24) == 0
    with pytest.raises(lib.SslaHipError, match="n_tokens"):
        size(most + 1, 1, most, heads=1)
    with pytest.raises(lib.SslaHipError, match="n_tokens"):      # the limit comes before the cut
        size((1 << 31) - 1, 2, 1 << 30, heads=512)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("pool", ["one", "two"])
def test_cut_sequences_among_many_short_ones(dtype, pool):
    """Cut sequences at every kind of place between pieces of 64 tokens, next to one
    another and among sequences of one token and of none."""
    from ssla_hip import ops
    lens = [1] * 40 + [700, 65, 66] + [1] * 20 + [0, 128, 129, 65, 0, 321] + [1] * 15 + [64, 65, 63, 257]
    H, dk, dv, t = 3, 24, 40, R.TYPES[dtype]
    gen = torch.Generator(device=DEV)
    gen.manual_seed(70)
    rnd = lambda *s: torch.randn(*s, generator=gen, device=DEV)  # noqa: E731
    T = sum(lens)
    q, k, v = rnd(T, H, dk).to(t), rnd(T, H, dk).to(t), rnd(T, H, dv).to(t)
    g = torch.nn.functional.logsigmoid(2.0 + 1.5 * rnd(T, H))
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=DEV)
    s0 = rnd(len(lens), H, dk, dv)
    s1 = s0.clone() if pool == "one" else torch.full_like(s0, 7.0)
    # more segments' places than twice the whole ones
    assert (T >> 6) + len(lens) > 2 * (T >> 6)
    want = R.linear_attention(q, k, v, g, lens, 0.3, s0)
    out = ops.linear_attention(q, k, v, g, scale=0.3, cu_seqlens=cu, state_in=s1 if pool == "one" else s0, state_out=s1)
    R.check_linear_attention(out, s1, want, t, dk, max(lens))


@pytest.mark.gpu
@pytest.mark.parametrize("cu", [[0, 500, 20, 400, 90, 300], [-7, 30, 5000, 2, 900, 0], [600] * 6,
                                [600, 0, 600, 0, 600, 0]], ids=str)
def test_wrong_cu_stays_in_the_workspace(cu):
    """Many sequences of garbage lengths: the states' places stay within it (shown
    beside linattn_states), and what lies around it is not touched."""
    L, T, H = lib.load(), 600, 2
    n = 20
    cu = torch.tensor((cu * 4)[:n + 1], dtype=torch.int32, device=DEV)
    x = torch.randn(T, H, 16, device=DEV).bfloat16()
    out = torch.full((T + 128, H, 16), 5.0, device=DEV).bfloat16()
    g = torch.zeros(H, device=DEV)
    d = abi.SslaHipLinAttn()
    d.dtype, d.heads, d.qk_heads, d.dk, d.dv = abi.SSLA_BF16, H, H, 16, 16
    d.n_seqs, d.max_len, d.n_tokens, d.scale = n, T, T, 1.0
    d.q = d.k = d.v = x.data_ptr()
    d.log_decay, d.cu_seqlens, d.out = g.data_ptr(), cu.data_ptr(), out[64:].data_ptr()
    for s in (d.q_stride, d.k_stride, d.v_stride, d.out_stride):
        s[:] = [H * 16, 16]
    d.decay_stride[:] = [0, 1]
    b = ctypes.c_size_t()
    lib.check(L.ssla_hip_linattn_workspace(ctypes.addressof(d), ctypes.byref(b)))
    assert b.value == 2 * (T >> 6) * H * (16 * 16 + 1) * 4
    ws = torch.full((b.value // 4 + 8192,), 3.0, device=DEV)
    lib.check(L.ssla_hip_linattn(ctypes.addressof(d), ws[4096:].data_ptr(), b.value,
                                 torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert (ws[:4096] == 3).all() and (ws[4096 + b.value // 4:] == 3).all()
    assert (out[:64] == 5).all() and (out[-64:] == 5).all()
