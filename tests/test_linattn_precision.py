"""How many bits linear attention's operands keep, at inputs whose answers have
few roundings, so that a term of an operand that is left out shows: one product
chain an output, or two that nearly cancel.  The checks themselves are tested on
the CPU, where an emulation with a term too few has to fail them.

Log decays are 0 (factors of exactly 1), scale is 1.  A sum on the matrix cores may
cut its bits off: two half steps (U) an addition."""
import pytest

torch = pytest.importorskip("torch")

DEV = "cuda"
U = 2.0 ** -24
CHUNK = 32
# Out of one chain: six products of terms for q.k, in two sums that are added (7
# additions), six for P.v; or six for the state and six for it times q.  Three terms
# of an operand, the first of them cut off, leave 2^-26 of it, U / 4 (four operands);
# of a product's terms the ones left out are 2^-8 2^-17 twice, 1 U (two products).
OUT_ROUNDINGS = 2 * 7 + 2 * 6 + 4 / 4 + 2
# The state: six products of terms, two operands, one product.
STATE_ROUNDINGS = 2 * 6 + 2 / 4 + 1
# A difference of two P v: four products and their sums a P, three terms of each P
# times v.
PAIR_ROUNDINGS = 2 * 4 + 2 * 6 + 1


def terms(x, n):
    """x (64 bits) as the sum of n bf16 values."""
    y, left = torch.zeros_like(x), x.clone()
    for _ in range(n):
        t = left.to(torch.bfloat16).double()
        y, left = y + t, left - t
    return y


def f32(x):
    return x.float().double()


# ---- one chain an output -----------------------------------------------------------

def chains(T, H, dk, dv, seed):
    """Token j < dk has its key in dimension j alone, later ones have none; every
    query asks for one dimension: out_t = a_t b_j v_j."""
    gen = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    j = (torch.rand(T, H, generator=gen) * torch.arange(1, T + 1).clamp(max=dk)[:, None]).long()
    a, b, v = rnd(T, H), rnd(T, H), rnd(T, H, dv)
    n = min(T, dk)
    q = torch.zeros(T, H, dk).scatter_(2, j[..., None], a[..., None])
    k = torch.zeros(T, H, dk)
    k[torch.arange(n), :, torch.arange(n)] = b[:n]
    return q, k, v, (a.double(), torch.gather(b.double(), 0, j), j)


def chain_answers(v, abj, dk):
    a, b, j = abj
    T, H, dv = v.shape
    vj = torch.gather(v.double(), 0, j[..., None].expand(T, H, dv))
    return a[..., None] * b[..., None] * vj, vj


def state_answer(k, v):
    return torch.matmul(k.double().permute(1, 2, 0), v.double().transpose(0, 1))


def chain_error(out, want, roundings):
    """Largest error in units of what is allowed."""
    return ((out.detach().cpu().double() - want).abs() / (roundings * U * want.abs() + 1e-36)).max().item()


def emulate_chains(k, v, abj, n):
    """Out and state with operands in n[...] terms."""
    a, b, j = abj
    t = torch.arange(v.shape[0])[:, None]
    _, vj = chain_answers(v, abj, k.shape[2])
    p = f32(terms(a, n["q"]) * terms(b, n["k"]))
    inside = f32(terms(p, n["p"])[..., None] * terms(vj, n["v"]))
    s = f32(terms(b, n["k"])[..., None] * terms(vj, n["v"]))
    before = f32(terms(s, n["s"]) * terms(a, n["q"])[..., None])
    out = torch.where((t // CHUNK == j // CHUNK)[..., None], inside, before)
    return out, torch.matmul(terms(k.double(), n["k"]).permute(1, 2, 0), terms(v.double(), n["v"]).transpose(0, 1))


THREE = dict(q=3, k=3, v=3, p=3, s=3)


@pytest.mark.parametrize("less", [None, "q", "k", "v", "p", "s"])
def test_the_check_of_one_chain_sees_a_term_too_few(less):
    q, k, v, abj = chains(700, 2, 96, 24, 1)
    n = dict(THREE, **({less: 2} if less else {}))
    out, state = emulate_chains(k, v, abj, n)
    worst = chain_error(out, chain_answers(v, abj, 96)[0], OUT_ROUNDINGS)
    assert worst <= 0.2 if less is None else worst > 1.2, worst
    worst = chain_error(state, state_answer(k, v), STATE_ROUNDINGS)
    assert worst > 1.2 if less in ("k", "v") else worst <= 0.2, worst


@pytest.mark.gpu
@pytest.mark.parametrize("T", [30, 200, 700])
@pytest.mark.parametrize("dk,dv", [(32, 24), (96, 72), (130, 40), (1, 1)])
def test_fp32_keeps_three_terms(T, dk, dv):
    """Within a chunk, behind it, whole sequences and cut ones."""
    from ssla_hip import ops
    q, k, v, abj = chains(T, 2, dk, dv, 2)
    s = torch.full((1, 2, dk, dv), 7.0, device=DEV)
    out = ops.linear_attention(q.to(DEV), k.to(DEV), v.to(DEV), torch.zeros(2, device=DEV), state_out=s)
    assert chain_error(out, chain_answers(v, abj, dk)[0], OUT_ROUNDINGS) <= 1.0
    assert chain_error(s[0], state_answer(k, v), STATE_ROUNDINGS) <= 1.0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [30, 700])
def test_states_of_16_bit_tokens_are_exact_products(dtype, T):
    """A product of two such values has at most 22 bits."""
    from ssla_hip import ops
    q, k, v, _ = (x.to(dtype) if torch.is_tensor(x) else x for x in chains(T, 2, 64, 40, 3))
    s = torch.full((1, 2, 64, 40), 7.0, device=DEV)
    ops.linear_attention(q.to(DEV), k.to(DEV), v.to(DEV), torch.zeros(2, device=DEV), state_out=s)
    # bf16: one product; fp16: two terms by two, the lowest three of the sums cut off
    assert chain_error(s[0], state_answer(k, v), 0.5 if dtype == torch.bfloat16 else 8) <= 1.0


# ---- two that nearly cancel ----------------------------------------------------------

def pairs(n, dk, dv, seed):
    """n sequences of one chunk: tokens 0 and 1 have nearly the same key and
    opposite values, the others none; queries have four dimensions:
    out_t = (q_t.k_0 - q_t.k_1) v_0 for t > 0, some 2^-14 of each of the two."""
    gen = torch.Generator().manual_seed(seed)
    pos = lambda *s: 1.0 + torch.rand(*s, generator=gen)  # noqa: E731
    q = torch.zeros(n, CHUNK, 1, dk)
    q[..., :4] = pos(n, CHUNK, 1, 4) * torch.tensor([1.0, 0.3, 0.04, 2.0 ** -6])
    q = q.bfloat16()
    k = torch.zeros(n, CHUNK, 1, dk).bfloat16()
    k[:, 0, 0, :4] = k[:, 1, 0, :4] = pos(n, 4).bfloat16()
    k[:, 1, 0, 3] += 2.0 ** -6
    v = torch.zeros(n, CHUNK, 1, dv).bfloat16()
    v[:, 0, 0] = torch.randn(n, dv, generator=gen).bfloat16()
    v[:, 1, 0] = -v[:, 0, 0]
    return q, k, v


def pair_error(out, q, k, v):
    p = torch.matmul(q[:, :, 0].double(), k[:, :2, 0].double().transpose(1, 2))      # (n, CHUNK, 2)
    v0 = v[:, 0].double()
    want = (p[..., :1] - p[..., 1:]) * v0
    tol = PAIR_ROUNDINGS * U * p.sum(2, keepdim=True) * v0.abs() + 2.0 ** -9 * 1.01 * want.abs() + 1e-36
    return ((out.detach().cpu().double() - want).abs() / tol)[:, 1:].max().item()


@pytest.mark.parametrize("n_terms", [2, 3])
def test_the_check_of_pairs_sees_a_term_too_few(n_terms):
    q, k, v = pairs(40, 16, 24, 4)
    p = terms(f32(torch.matmul(q[:, :, 0].double(), k[:, :2, 0].double().transpose(1, 2))), n_terms)
    out = ((p[..., :1] - p[..., 1:]) * v[:, 0].double()).bfloat16()
    worst = pair_error(out, q, k, v)
    assert worst > 1.2 if n_terms == 2 else worst <= 0.3, worst


@pytest.mark.gpu
@pytest.mark.parametrize("dk,dv", [(16, 24), (128, 128), (256, 40)])
def test_products_within_a_chunk_of_bf16_tokens_keep_three_terms(dk, dv):
    from ssla_hip import ops
    q, k, v = pairs(40, dk, dv, 5)
    out = ops.linear_attention(*(x.flatten(0, 1).to(DEV) for x in (q, k, v)), torch.zeros(1, device=DEV), n_seqs=40)
    assert pair_error(out.view(40, CHUNK, dv), q, k, v) <= 1.0


# ---- the largest values ----------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("T", [90, 600])
@pytest.mark.parametrize("what", ["q", "k", "v"])
@pytest.mark.parametrize("value", [torch.finfo(torch.float32).max, -3.396e38])
def test_the_largest_fp32_values_are_finite(T, what, value):
    """They are beyond bf16's largest; other values keep the answers in range."""
    import seq_ref as R
    from ssla_hip import ops
    gen = torch.Generator().manual_seed(6)
    q, k, v = (1e-10 * torch.randn(T, 2, n, generator=gen) for n in (32, 32, 48))
    {"q": q, "k": k, "v": v}[what][T // 2 + 5, 1, 3] = value
    g = torch.full((2,), -0.02)
    want = R.linear_attention(q, k, v, g, [T], 1.0)
    s = torch.zeros(1, 2, 32, 48, device=DEV)
    out = ops.linear_attention(q.to(DEV), k.to(DEV), v.to(DEV), g.to(DEV), state_out=s)
    R.check_linear_attention(out, s, want, torch.float32, 32, T)
