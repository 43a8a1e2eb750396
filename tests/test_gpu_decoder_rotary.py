"""The position rotation on the way into the 8-bit cache (decoder.kv8_rotary_append) against its formula in 64 bits.

Bounds. fp32 arithmetic: a norm's sum of up to 256 squares is off by at most 2^-17 relative (16 in a lane, then 4 steps, half of
it in the root), the root, weight and rotation by some 2^-22 of |x_i| + |x_j|: 2^-16 (|x_i| + |x_j|) is allowed. A query is rounded
once more, by half a step: eps / 2 of itself, or of the type's smallest normal (2^-14 for fp16) where it is below that. A scale is then off by 2^-16 * 2, a code by at most half a step and 127 * 2^-15 < 2^-8
of one: |code - x / scale| <= 0.5 + 2^-8. Values, which nothing turns, are compared bit for bit with kv8_append's. Needs an MI355X."""

import pytest
import torch

from _gpu import graph_replays_equal, poison_allocator
from test_gpu_decoder_kv8 import _cu, _i32, _random_cache, _table

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def dec():
    from vllm_gguf_plugin import decoder

    assert torch.cuda.is_available(), "GPU tests need an MI355X"
    return decoder


def _angles(n, rot, base=1e4):
    inv = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    a = torch.arange(n, dtype=torch.float64)[:, None] * inv
    return torch.cat([a.cos(), a.sin()], 1).float().cuda()


def _turned(x, w, cs, at, pairs, eps):
    """(the turned rows in 64 bits, |x_i| + |x_j| of each value's pair)"""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    r = cs.shape[1]
    c, s = cs[at, None, :r // 2].double(), cs[at, None, r // 2:].double()
    i = torch.arange(0, r, 2, device="cuda") if pairs else torch.arange(r // 2, device="cuda")
    j = i + 1 if pairs else i + r // 2
    y, both = x.clone(), x.abs()
    y[..., i] = x[..., i] * c - x[..., j] * s
    y[..., j] = x[..., j] * c + x[..., i] * s
    both[..., i] = both[..., j] = x[..., i].abs() + x[..., j].abs()
    return y, both


class _Call:
    def __init__(self, dec, ends, news, hq, heads, d, page, rot, dtype, seed, pairs=False, norms=(True, True), eps=1e-6, table=None):
        g = torch.Generator().manual_seed(seed)
        self.dec, self.news, self.ends, self.page, self.pairs, self.eps = dec, news, ends, page, pairs, eps
        pages = sum(-(-max(e, 0) // page) for e in ends) + 2
        self.cache = _random_cache(dec, pages, heads, page, d, g)
        self.table = _table(ends, page, pages, g) if table is None else table
        t = sum(news)
        x = torch.randn(t, hq + 2 * heads + 1, d, generator=g) * torch.exp(torch.randn(t, 1, 1, generator=g))
        x[:, hq:hq + heads, ::37] *= 6
        x = x.to(dtype).cuda()
        self.q, self.k, self.v = x[:, :hq], x[:, hq:hq + heads], x[:, hq + heads:hq + 2 * heads]
        self.cs = _angles(max(max(ends), 1) + 5, rot)
        self.at = torch.cat([torch.arange(e - n, e) for e, n in zip(ends, news)]).clamp(min=0).cuda()
        self.qw, self.kw = ((1 + 0.3 * torch.randn(d, generator=g)).cuda() if n else None for n in norms)

    def __call__(self, cache=None, max_new=None):
        poison_allocator()
        return self.dec.kv8_rotary_append(cache or self.cache, self.q, self.k, self.v, self.cs, self.at, self.table, _i32(*self.ends),
                                          _cu(self.news), max(self.news) if max_new is None else max_new, interleaved=self.pairs,
                                          q_weight=self.qw, k_weight=self.kw, eps=self.eps)

    def check(self, max_new=None):
        start = self.dec.Kv8Cache(*(x.clone() for x in self.cache))
        by_append = self.dec.Kv8Cache(*(x.clone() for x in self.cache))
        y = self(max_new=max_new)
        ref, both = _turned(self.q, self.qw, self.cs, self.at, self.pairs, self.eps)
        info = torch.finfo(y.dtype)
        assert y.shape == self.q.shape and y.dtype == self.q.dtype and y.is_contiguous()
        bad = (y.double() - ref).abs() > info.eps / 2 * ref.abs().clamp(min=info.smallest_normal) + 2.0 ** -16 * both
        assert not bad.any(), (int(bad.sum()), bad.nonzero()[:3])
        # values: as kv8_append has them, and its older pages and places
        self.dec.kv8_append(by_append, self.k, self.v, self.table, _i32(*self.ends), _cu(self.news), max(self.news))
        assert torch.equal(self.cache.v, by_append.v) and torch.equal(self.cache.v_scale, by_append.v_scale)
        self.check_keys(start)
        return y

    def check_keys(self, start):
        key, both = _turned(self.k, self.kw, self.cs, self.at, self.pairs, self.eps)
        want, scale, kept, least = (x.clone() for x in (start.k, start.k_scale, start.k, start.k_scale))
        page, room, row = self.page, self.table.shape[1] * self.page, 0
        allowed = torch.zeros(start.k.shape, dtype=torch.float64, device="cuda")  # of the codes
        for s, (end, n) in enumerate(zip(self.ends, self.news)):
            base = end - n
            for p in range(max(base, 0) // page, -(-min(max(end, 0), room) // page)) if n else ():
                pid = int(self.table[s, p])
                if not 0 <= pid < start.k.shape[0]:
                    continue
                lo, hi = max(base, p * page), min(end, p * page + page)
                x = key[row + lo - base:row + hi - base].transpose(0, 1)  # [heads, tokens, d]
                got = self.cache.k_scale[pid].double()
                need = (x.abs().amax((1, 2)) / 127)
                was = start.k_scale[pid].double() if base > p * page else torch.zeros_like(need)
                now = torch.maximum(was, need)
                off = both[row + lo - base:row + hi - base].transpose(0, 1).amax((1, 2)) / 127 * 2.0 ** -16
                assert ((got - now).abs() <= off + 2.0 ** -23 * now).all()
                codes = self.cache.k[pid].double()
                place = slice(lo - p * page, hi - p * page)
                assert ((codes[:, place] - x / got[:, None, None]).abs() <= 0.5 + 2.0 ** -8).all()
                older = slice(0, max(base - p * page, 0))
                old = start.k[pid, :, older].double() * (was / got)[:, None, None]
                assert ((codes[:, older] - old).abs() <= 0.5 + 2.0 ** -15).all()
                kept[pid, :, place], kept[pid, :, older] = self.cache.k[pid, :, place], self.cache.k[pid, :, older]
                least[pid] = self.cache.k_scale[pid]
            row += n
        assert torch.equal(kept, self.cache.k) and torch.equal(least, self.cache.k_scale)  # everything else is as it was


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("hq,heads,d,page,rot", [(6, 2, 256, 64, 64), (3, 1, 128, 16, 128), (4, 4, 64, 144, 32), (1, 2, 192, 32, 96),
                                                 (24, 1, 256, 144, 256), (2, 1, 192, 16, 192), (1, 1, 64, 16, 16)])
@pytest.mark.parametrize("pairs", [False, True])
def test_rotary(dec, dtype, hq, heads, d, page, rot, pairs):
    """Prompts, single tokens and none; partial rotation in halves and pairs; norms on both, one or none."""
    norms = [(True, True), (False, False), (True, False), (False, True)][(rot // 16 + pairs + hq) % 4]
    for seed, (ends, news) in enumerate([((37, 300, 5, 90), (37, 1, 0, 26)), ((1, 150), (1, 150)), ((700,), (333,))]):
        _Call(dec, ends, news, hq, heads, d, page, rot, dtype, seed, pairs, norms).check()


@pytest.mark.parametrize("max_new", [0, 1, 10 ** 6, 2 ** 62])
def test_hint_only_sizes_the_launch(dec, max_new):
    _Call(dec, (300, 40), (290, 3), 4, 2, 128, 16, 64, BF16, 5).check(max_new)


def test_many_sequences(dec):
    """More (sequence, head) pairs than workgroups for every page of each: a workgroup takes several."""
    news = [1 + i % 3 for i in range(700)]
    _Call(dec, tuple(n + i % 50 for i, n in enumerate(news)), tuple(news), 2, 2, 64, 16, 64, BF16, 6).check()


@pytest.mark.parametrize("case", ["negative", "capacity", "length"])
def test_positions_lengths_and_pages_at_the_edges(dec, case):
    """Rows before position 0 and past the table's capacity are dropped from the cache, their queries are turned all the same."""
    c = _Call(dec, (30, 100), (30, 20), 3, 2, 128, 16, 64, BF16, 7)
    if case == "negative":
        c.ends = (-4, 11)
    elif case == "capacity":
        c.table = c.table[:, :5].contiguous()
    else:
        c.ends = (30, 2)
    c.check()


def test_bad_positions_and_pages(dec):
    """A position out of the table turns by NaN: the row's turned dims, its page of K, nothing else. A page out of range takes nothing."""
    c = _Call(dec, (64, 20), (10, 5), 3, 2, 128, 16, 64, BF16, 8)
    ref = c(cache=dec.Kv8Cache(*(x.clone() for x in c.cache)))
    c.at[2], c.at[11] = -1, c.cs.shape[0]
    y = c()
    for row in (2, 11):
        assert torch.isnan(y[row, :, :64]).all() and torch.equal(y[row, :, 64:], ref[row, :, 64:])
    rest = [i for i in range(15) if i not in (2, 11)]
    assert torch.equal(y[rest], ref[rest])
    bad = {int(c.table[0, 56 // 16]), int(c.table[1, 16 // 16])}
    nan = torch.isnan(c.cache.k_scale).any(1)
    assert {i for i in range(len(nan)) if nan[i]} == bad and torch.isnan(c.cache.k_scale[list(bad)]).all()
    assert torch.isfinite(c.cache.v_scale).all()

    c = _Call(dec, (64, 20), (10, 5), 3, 2, 128, 16, 64, BF16, 8)
    start = [x.clone() for x in c.cache]
    c.table[0, 3], c.table[1] = 10 ** 6, -1
    c()
    assert all(torch.equal(x, y) for x, y in zip(start, c.cache))


def test_rows_behind_the_last_sequence(dec):
    c = _Call(dec, (40, 9), (20, 9), 3, 2, 64, 16, 32, F16, 9)
    c.news = (5, 9)
    c.ends = (25, 9)
    c.q, c.k, c.v = c.q[:20], c.k[:20], c.v[:20]
    c.at = c.at[:20].contiguous()
    start = [x.clone() for x in c.cache]
    y = c()
    ref, both = _turned(c.q, c.qw, c.cs, c.at, False, c.eps)
    assert ((y.double() - ref).abs() <= 2.0 ** -11 * ref.abs().clamp(min=2.0 ** -14) + 2.0 ** -16 * both).all()
    touched = {int(p) for s, (e, n) in enumerate(zip(c.ends, c.news)) for p in c.table[s, (e - n) // 16:-(-e // 16)]}
    for x, was in zip(c.cache, start):
        for p in range(x.shape[0]):
            assert p in touched or torch.equal(x[p], was[p])


def test_zero_rows_and_values_that_are_not_finite(dec):
    """Rows of zeros stay so (eps holds the norm); an infinity makes NaN of its own query row and its key's (page, head)."""
    c = _Call(dec, (33,), (17,), 3, 2, 128, 16, 64, BF16, 10)
    c.q[:], c.k[:], c.v[:] = 0, 0, 0
    assert (c() == 0).all()
    c = _Call(dec, (33,), (17,), 3, 2, 128, 16, 64, BF16, 10)
    c.q[4, 1, 3], c.k[5, 0, 100] = float("inf"), float("nan")
    y = c()
    nan = torch.isnan(y).any(-1)
    assert nan[4, 1] and int(nan.sum()) == 1
    assert torch.isnan(c.cache.k_scale).sum() == 1 and torch.isnan(c.cache.k_scale[int(c.table[0, 21 // 16]), 0])


def test_steps_give_what_a_prompt_gives(dec):
    """Token by token, in threes and at once: the queries are the same bits, and the pages' first codes differ by what rescaling rounds."""
    a = _Call(dec, (50,), (50,), 4, 2, 128, 16, 128, BF16, 11)
    whole = a()
    for step in (1, 3, 16):
        b = _Call(dec, (50,), (50,), 4, 2, 128, 16, 128, BF16, 11)
        for i in range(0, 50, step):
            n = min(step, 50 - i)
            y = dec.kv8_rotary_append(b.cache, b.q[i:i + n], b.k[i:i + n], b.v[i:i + n], b.cs, b.at[i:i + n], b.table, _i32(i + n), _cu((n,)),
                                      n, q_weight=b.qw, k_weight=b.kw)
            assert torch.equal(y, whole[i:i + n])
        assert torch.equal(a.cache.k_scale, b.cache.k_scale) and torch.equal(a.cache.v_scale, b.cache.v_scale)
        for x, y in ((a.cache.k, b.cache.k), (a.cache.v, b.cache.v)):  # 16 roundings a page, of at most half a step each
            assert (x.int() - y.int()).abs().max() <= 8


def test_rotary_repeats_and_replays(dec):
    c = _Call(dec, (300, 90), (40, 90), 6, 2, 256, 64, 64, BF16, 12)
    y = c()
    lens, cu = _i32(*c.ends), _cu(c.news)

    def call():
        return dec.kv8_rotary_append(c.cache, c.q, c.k, c.v, c.cs, c.at, c.table, lens, cu, 90, q_weight=c.qw, k_weight=c.kw)

    after = [x.clone() for x in c.cache]
    assert torch.equal(call(), y)
    graph_replays_equal(call, y)
    assert all(torch.equal(x, y) for x, y in zip(after, c.cache))
