"""decoder.gated_delta_rule against its definition token by token in float64.

Bounds. Products are exact or to 2^-24 and summed in fp32 over at most dk + 64 places, of what a
token adds to the state and of the state itself at every chunk; with unit keys the state does not grow
beyond what is added. 2^-24 * 64 is room for the square root of a thousand such sums: a head's state is
within 4e-6 of its norm, and an fp32 output row within 4e-6 of the norms that it is a product of
(scale |q| |S| summed, which a row's own norm may be far below). A 16-bit output adds its rounding, 2^-9 or 2^-12 of a value, and the 2^-16 to which the
chunked form's output products are kept. Needs an MI355X."""

import pytest
import torch

from _gpu import graph_replays_equal, poison_allocator

pytestmark = pytest.mark.gpu

TOL = 4e-6


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    assert torch.cuda.is_available(), "GPU tests need an MI355X"


@pytest.fixture(scope="module")
def dec():
    from vllm_gguf_plugin import decoder

    return decoder


def _cu(lens):
    return torch.tensor([0] + list(lens), device="cuda").cumsum(0).to(torch.int32)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _ref(q, k, v, g, beta, states, news, scale, l2norm):
    """(out, last states, the state after every token, a bound of the norms of an output row), float64."""
    q, k, v, g, beta = (x.double().cpu() for x in (q, k, v, g, beta))
    rep = v.shape[1] // q.shape[1]
    if l2norm:
        q, k = (x / torch.sqrt((x * x).sum(-1, keepdim=True) + 1e-6) for x in (q, k))
    q, k = q.repeat_interleave(rep, 1), k.repeat_interleave(rep, 1)
    out, size, every, row = torch.zeros_like(v), torch.zeros(v.shape[:2], dtype=torch.float64), [], 0
    last = []
    for s, n in enumerate(news):
        m, seen = states[s].double().cpu(), []
        for i in range(row, row + n):
            m = m * torch.exp(g[i])[:, None, None]
            u = beta[i][:, None] * (v[i] - (m @ k[i][..., None])[..., 0])
            m = m + u[..., None] * k[i][:, None, :]
            out[i] = scale * (m @ q[i][..., None])[..., 0]
            size[i] = scale * q[i].norm(dim=-1) * m.flatten(1).norm(dim=-1)
            seen.append(m)
        last.append(m)
        every.append(seen)
        row += n
    return out, last, every, size


def _inputs(news, hk, hv, dk, dv, dtype, seed, slots=None, gates=(0.001, 3.0)):
    gen = torch.Generator().manual_seed(seed)
    t = sum(news)

    def normal(*s):
        return torch.randn(*s, generator=gen)

    x = normal(t, 2 * hk * dk + hv * dv).to(dtype).cuda()
    q, k = x[:, :hk * dk].view(t, hk, dk), x[:, hk * dk:2 * hk * dk].view(t, hk, dk)
    v = x[:, 2 * hk * dk:].view(t, hv, dv)
    lo, hi = (torch.tensor(r).log() for r in gates)
    rate = torch.exp(lo + (hi - lo) * torch.rand(hv, generator=gen))
    g = (-rate * torch.nn.functional.softplus(normal(t, hv))).cuda()
    beta = torch.sigmoid(normal(t, hv)).cuda()
    state = (0.3 * normal(slots or len(news), hv, dv, dk)).cuda()
    return q, k, v, g, beta, state


def _check(y, ref, size, dtype, chunked_bits=2.0 ** -16):
    err = (y.double().cpu() - ref).norm(dim=-1)
    bound = TOL * size
    if dtype != torch.float32:
        # each element's rounding, twice for room, and the kept bits of the chunked form's output products
        bound = bound + ref.norm(dim=-1) * (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11) + 4 * chunked_bits * size
    assert (err <= bound + 1e-30).all(), float((err / bound.clamp_min(1e-30)).max())


def _check_state(got, want):
    for h in range(got.shape[0]):
        err = (got[h].double().cpu() - want[h]).norm()
        assert err <= TOL * want[h].norm() + 1e-30, float(err / want[h].norm())


def _run(dec, news, hk, hv, dk, dv, dtype, seed, l2norm=True, max_new=None, change=None):
    q, k, v, g, beta, state = _inputs(news, hk, hv, dk, dv, dtype, seed)
    if change:
        change(q, k, v, g, beta, state)
    first = state.clone()
    scale = dk ** -0.5 if l2norm else 0.02
    if not l2norm:
        k.mul_(dk ** -0.5)
    poison_allocator()
    y = dec.gated_delta_rule(q, k, v, g, beta, state, _i32(list(range(len(news)))), _cu(news), max_new or max(news),
                             scale=scale, l2norm=l2norm)
    out, last, _, size = _ref(q, k, v, g, beta, first, news, scale, l2norm)
    assert y.shape == v.shape and y.dtype == dtype
    _check(y, out, size, dtype)
    for s in range(len(news)):
        _check_state(state[s], last[s])
    return y, state


DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("hk,hv,dk,dv", [(2, 6, 128, 128), (2, 2, 64, 128), (1, 2, 128, 48), (1, 3, 64, 16), (1, 1, 128, 208)])
def test_few_tokens(dec, dtype, hk, hv, dk, dv):
    """The recurrent form; a sequence of no tokens keeps its state."""
    _run(dec, (1, 4, 0, 2), hk, hv, dk, dv, dtype, 31)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("hk,hv,dk,dv", [(2, 6, 128, 128), (2, 2, 64, 128), (1, 2, 128, 48), (1, 3, 64, 16), (1, 1, 128, 208)])
def test_prompts(dec, dtype, hk, hv, dk, dv):
    """Lengths around the chunk's, beside sequences that the recurrent form takes."""
    _run(dec, (33, 1, 64, 65, 0, 200, 32, 127), hk, hv, dk, dv, dtype, 32)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("news", [(3,), (130,)], ids=str)
def test_without_norm(dec, dtype, news):
    _run(dec, news, 1, 2, 128, 64, dtype, 33, l2norm=False)


@pytest.mark.parametrize("max_new", [1, 10000])
def test_hint_only_sizes_the_launch(dec, max_new):
    _run(dec, (70, 2, 130), 1, 2, 128, 32, torch.bfloat16, 34, max_new=max_new)


@pytest.mark.parametrize("news", [(5,), (150,)], ids=str)
@pytest.mark.parametrize("case", ["forget", "keep", "strong", "closed", "same keys", "no keys"])
def test_gates_and_keys_at_their_ends(dec, news, case):
    """Decays of 0 and 1 and far below, beta 0 and 1, a prompt of one key (the worst condition of the
    chunk's system), keys of zeros."""
    def change(q, k, v, g, beta, state):
        if case == "forget":
            g[::7] = -float("inf")
            g[3::11] = -1e30
        elif case == "keep":
            g.zero_()
            beta.fill_(1.0)
        elif case == "strong":
            g.mul_(100)
        elif case == "closed":
            beta[::2] = 0.0
        elif case == "same keys":
            k.copy_(k[:1].clone().expand_as(k))
            g.mul_(1e-3)
            beta.fill_(1.0)
        else:
            k[::3] = 0.0

    _run(dec, news, 1, 2, 128, 64, torch.bfloat16, 35, change=change)


def test_long_prompt_stays_exact(dec):
    """Two thousand tokens through slow heads: the state carries through all of the chunks."""
    _run(dec, (2050,), 1, 2, 128, 32, torch.bfloat16, 36, change=lambda q, k, v, g, beta, s: g.mul_(0.01))


@pytest.mark.parametrize("news", [(1, 4, 3), (1, 90, 3)], ids=str)
def test_slots(dec, news):
    """States from and to other slots; -1 and a slot past the pool: from zero, kept nowhere; a sequence
    of no tokens copies its state."""
    news = news + (0,)
    q, k, v, g, beta, state = _inputs(news, 1, 2, 128, 64, torch.bfloat16, 37, slots=9)
    first = state.clone()
    src, dst = [4, -1, 9, 2], [7, 8, -1, 5]
    y = dec.gated_delta_rule(q, k, v, g, beta, state, _i32(src), _cu(news), max(news), out_slots=_i32(dst))
    zero = torch.zeros_like(first[0])
    out, last, _, size = _ref(q, k, v, g, beta, [first[4], zero, zero, first[2]], news, 128 ** -0.5, True)
    _check(y, out, size, torch.bfloat16)
    for s in (0, 1):
        _check_state(state[dst[s]], last[s])
    assert torch.equal(state[5], first[2])
    for s in (0, 1, 2, 3, 4, 6):
        assert torch.equal(state[s], first[s])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("news", [(4, 1, 0, 6), (40, 2, 0, 6)], ids=str)
def test_every_tokens_state(dec, dtype, news):
    """out_slots [seqs, m]: the states after the first m tokens of each sequence, as far as it has them."""
    m = 4
    q, k, v, g, beta, state = _inputs(news, 1, 2, 64, 32, dtype, 38, slots=4 + 16)
    first = state.clone()
    dst = 4 + torch.arange(16).view(4, m)
    dst[0, 2] = -1
    y = dec.gated_delta_rule(q, k, v, g, beta, state, _i32([0, 1, 2, 3]), _cu(news), max(news), out_slots=dst.to(torch.int32).cuda())
    out, _, every, size = _ref(q, k, v, g, beta, first, news, 64 ** -0.5, True)
    _check(y, out, size, dtype)
    assert torch.equal(state[:4], first[:4])
    for s, n in enumerate(news):
        for i in range(m):
            if i < n and dst[s, i] >= 0:
                _check_state(state[dst[s, i]], every[s][i])
            elif dst[s, i] >= 0:
                assert torch.equal(state[dst[s, i]], first[dst[s, i]])
    assert torch.equal(state[6], first[6])


@pytest.mark.parametrize("news", [(1, 2), (100, 40)], ids=str)
def test_other_stream_and_graph(dec, news):
    q, k, v, g, beta, state = _inputs(news, 2, 4, 128, 128, torch.bfloat16, 39, slots=4)
    cu, to = _cu(news), _i32([2, 3])
    src = _i32([0, 1])
    def call():
        return dec.gated_delta_rule(q, k, v, g, beta, state, src, cu, max(news), out_slots=to)

    y = call()
    kept = state[2:].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, z) and torch.equal(kept, state[2:])
    graph_replays_equal(call, y)
    assert torch.equal(kept, state[2:])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("what", ["q", "k", "v", "g", "beta"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("at", [3, 84, 149])
@pytest.mark.parametrize("max_new", [1, 150], ids=["recurrent", "chunks"])
def test_a_token_that_is_not_finite(dec, dtype, what, bad, at, max_new):
    """Outputs of earlier tokens, of other heads and (for a value) of other columns are as ever; from the token on nothing
    that it reaches is finite (of a query, its own output alone)."""
    news, hk, hv, dk, dv = (150, 40), 2, 4, 128, 48
    q, k, v, g, beta, state = _inputs(news, hk, hv, dk, dv, dtype, 40)
    out, last, _, size = _ref(q, k, v, g, beta, state, news, dk ** -0.5, True)
    {"q": q[at, 1], "k": k[at, 1], "v": v[at, 3], "g": g[at, 3:], "beta": beta[at, 3:]}[what][:1 if what in "g beta" else 6] = bad
    y = dec.gated_delta_rule(q, k, v, g, beta, state, _i32([0, 1]), _cu(news), max_new)
    hit = torch.zeros(y.shape, dtype=torch.bool)
    heads = [2, 3] if what in ("q", "k") else [3]
    for h in heads:
        hit[at:(at + 1 if what == "q" else news[0]), h, :6 if what == "v" else dv] = True
    assert not y.cpu()[hit].isfinite().any()
    y = torch.where(hit.cuda(), 0, y)
    out = torch.where(hit, 0, out)
    _check(y, out, size, dtype)
    _check_state(state[1], last[1])
    fine = torch.ones(hv, dv, dtype=torch.bool)
    if what != "q":
        fine = ~hit[-41]
        assert not state[0].cpu()[~fine].isfinite().any()
    for h in range(hv):
        if fine[h].any():
            _check_state(state[0, h:h + 1, fine[h]], [last[0][h, fine[h]]])
