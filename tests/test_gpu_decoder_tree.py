"""Attention for trees of drafts (decoder.kv8_tree_attention) against a float64 softmax over the cached values, and keeping a
path of a tree (decoder.kv8_keep) against the same moves on the host, bit for bit.

Attention's bound is that of kv8_attention (test_gpu_decoder_kv8.py derives it): |y - ref| <= 2^-8 |ref| (fp16 2^-11) +
2^-10 max |v| of what the row sees. Needs an MI355X."""

import pytest
import torch

from _gpu import graph_replays_equal, poison_allocator
from test_gpu_decoder_kv8 import _close, _cu, _i32, _random_cache, _table, _values

pytestmark = pytest.mark.gpu
BF16, F16, I64 = torch.bfloat16, torch.float16, torch.int64


@pytest.fixture(scope="module")
def dec():
    from vllm_gguf_plugin import decoder

    assert torch.cuda.is_available(), "GPU tests need an MI355X"
    return decoder


def _bits(mask, n):
    """[rows, n] truth values of an int64 [rows, words] mask; rows past its words are not seen."""
    at = torch.arange(n)
    seen = (mask.cpu()[:, (at // 64).clamp(max=mask.shape[1] - 1)] >> (at % 64) & 1).bool()
    return seen & (at < 64 * mask.shape[1])


def _tree_ref(q, cache, table, mask, ends, news, scale):
    hq, heads = q.shape[1], cache.k.shape[1]
    room = table.shape[1] * cache.k.shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    most = torch.zeros(q.shape[0], hq, 1, dtype=torch.float64, device="cuda")
    row = 0
    for s, (end, n) in enumerate(zip(ends, news)):
        base, have = end - n, min(max(end, 0), room)
        if n and have:
            k, v = (x.repeat_interleave(hq // heads, 0) for x in _values(cache, table, s, have))
            bits = _bits(mask[row:row + n], n)
            for i in range(n):
                pos = torch.arange(have)
                see = ((pos < base) | ((pos >= base) & bits[i, (pos - base).clamp(0, n - 1)])).cuda()
                if see.any():
                    x = (k[:, see] @ q[row + i].double()[..., None])[..., 0] * scale
                    out[row + i] = (torch.softmax(x, -1)[:, None] @ v[:, see])[:, 0]
                    most[row + i] = v[:, see].abs().amax((1, 2))[:, None]
        row += n
    return out, most


def _random_mask(rows, words, g, share=0.4):
    bits = torch.rand(rows, 64 * words, generator=g) < share
    weights = torch.tensor([1 << j if j < 63 else -(1 << 63) for j in range(64)], dtype=I64)
    return (bits.view(rows, words, 64).to(I64) * weights).sum(-1)


def _run(dec, ends, news, hq, heads, d, page, dtype, seed, words=1, mask=None, max_new=None, max_len=None, change=None):
    g = torch.Generator().manual_seed(seed)
    pages = sum(-(-max(e, 0) // page) for e in ends) + 2
    cache = _random_cache(dec, pages, heads, page, d, g)
    table = _table(ends, page, pages, g)
    q = (torch.randn(sum(news), hq, d, generator=g) * 0.3).to(dtype).cuda()
    mask = (_random_mask(sum(news), words, g) if mask is None else mask).cuda()
    if change:
        table = change(cache, table)
    poison_allocator()
    y = dec.kv8_tree_attention(q, cache, mask, table, _i32(*ends), _cu(news), max(news) if max_new is None else max_new,
                               max(ends) if max_len is None else max_len)
    ref, most = _tree_ref(q, cache, table, mask, ends, news, d ** -0.5)
    assert y.shape == q.shape and y.dtype == dtype
    _close(y, ref, most)
    return q, cache, table, mask, y


# max_len hints: the contexts' own, and one that asks for the forms for many rows wherever more than 32 rows share a KV head
HINTS = [None, 1 << 24]


@pytest.mark.parametrize("hint", HINTS)
@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
@pytest.mark.parametrize("hq,heads,d,page", [(6, 1, 256, 16), (8, 2, 128, 32), (4, 4, 64, 144), (5, 1, 192, 64), (16, 2, 256, 144), (3, 1, 192, 16)])
@pytest.mark.parametrize("news", [(1, 1, 1, 1), (1, 3, 0, 7), (2, 9, 8, 5), (5, 40, 2, 17), (64, 63, 1, 30)], ids=str)
def test_tree(dec, dtype, hq, heads, d, page, news, hint):
    """Any bits, a root alone to a whole mask word, behind contexts of none to several splits."""
    _run(dec, (news[0], 65, 200, 777), news, hq, heads, d, page, dtype, 21, max_len=hint)


@pytest.mark.parametrize("hq,heads,d,page,dtype", [(6, 1, 256, 16, BF16), (1, 1, 128, 16, F16), (8, 1, 64, 32, BF16)])
@pytest.mark.parametrize("words", [1, 2, 3])
@pytest.mark.parametrize("hint", HINTS)
def test_masks_of_several_words(dec, hq, heads, d, page, dtype, words, hint):
    """Trees that end inside, at and beyond their masks: rows past them are not seen. Tiles that straddle words."""
    _run(dec, (130, 400, 71 + 64 * words, 191), (130, 100, 64 * words, 191), hq, heads, d, page, dtype, 22, words, max_len=hint)


@pytest.mark.parametrize("base", [0, 1, 15, 16, 31, 33, 63, 64, 65, 100])
@pytest.mark.parametrize("hq,news", [(2, 11), (2, 37)])
@pytest.mark.parametrize("d,hint", [(128, None), (128, 1 << 24), (256, 1 << 24)])
def test_where_the_drafts_begin(dec, base, hq, news, d, hint):
    """The first draft at every place of a chunk, tile and page; ancestors as a tree has them."""
    parents = [[-1] + [(i * 7) % i for i in range(1, news)]]
    _run(dec, (base + news,), (news,), 2 * hq, 2, d, 16, BF16, 23, mask=dec.tree_mask(parents), max_len=hint)


@pytest.mark.parametrize("d,hq", [(256, 6), (192, 3), (128, 6)])
def test_long_contexts(dec, d, hq):
    """Contexts that shares of the work begin and end in, beyond the chunks that are looked up at a time (2048 tokens, and 4096), beside
    short ones and empty sequences; one sequence alone; many short ones in a share."""
    _run(dec, (9000, 40, 5, 2600, 0, 4177), (30, 33, 5, 1, 0, 64), hq, 1, d, 64, BF16, 31, max_len=1 << 24)
    _run(dec, (20011,), (24,), hq, 1, d, 16, BF16, 32, max_len=1 << 24)
    ends = tuple(3 + 17 * i % 150 for i in range(300))
    _run(dec, ends, tuple(min(e, 1 + i % 4) for i, e in enumerate(ends)), 3 * hq, 3, d, 32, F16, 33, max_new=20, max_len=1 << 24)


@pytest.mark.parametrize("scale", [-0.5, 0.0, 3e4, 1e-30])
@pytest.mark.parametrize("hint", HINTS)
def test_scales_and_maxima_that_move(dec, scale, hint):
    """Any scale; scores that rise and fall by hundreds from tile to tile, in one half of a tile and the other."""
    g = torch.Generator().manual_seed(34)
    ends, news, page = (700,), (40,), 16
    cache = _random_cache(dec, 46, 1, page, 256, g)
    cache.k_scale.copy_(torch.exp2(12 * torch.rand(46, 1, generator=g) - 8))
    table = _table(ends, page, 46, g)
    q = (torch.randn(40, 4, 256, generator=g) * (1 if abs(scale) > 1 else 0.3)).to(BF16).cuda()
    mask = _random_mask(40, 1, g).cuda()
    y = dec.kv8_tree_attention(q, cache, mask, table, _i32(*ends), _cu(news), 40, hint or 700, scale)
    ref, most = _tree_ref(q, cache, table, mask, ends, news, scale)
    assert torch.isfinite(y).all()
    if abs(scale) < 1:
        _close(y, ref, most)
    else:  # one token takes all, but where two are within the queries' last bits
        assert ((y.double() - ref).abs() <= 2.0 ** -6 * most).float().mean() > 0.98


@pytest.mark.parametrize("news", [(3, 4, 2, 5), (3, 90, 2, 80)], ids=str)
@pytest.mark.parametrize("d,hint", [(128, None), (128, 1 << 24), (256, 1 << 24)])
def test_rows_that_see_nothing(dec, news, d, hint):
    """No bits and no context, a length below the rows, a negative one: zeros. And no bits over a context."""
    mask = torch.zeros(sum(news), 1, dtype=I64)
    mask[news[0] + 3] = 0b1010
    ends = (news[0], 3, -3, news[3] + 50)
    y = _run(dec, ends, news, 6, 2, d, 16, BF16, 24, mask=mask, max_len=hint)[-1]
    assert (y[:news[0]] == 0).all() and (y[news[0]:news[0] + 3] == 0).all() and (y[-news[3] - news[2]:-news[3]] == 0).all()
    assert (y[-news[3]:] != 0).any(-1).all()


@pytest.mark.parametrize("news", [2, 40])
def test_lower_triangle_is_causal(dec, news):
    q, cache, table, mask, y = _run(dec, (300 + news,), (news,), 6, 2, 256, 64, BF16, 25, mask=dec.tree_mask([list(range(-1, news - 1))]))
    x = dec.kv8_attention(q, cache, table, _i32(300 + news), _cu((news,)), news, 300 + news)
    ref, most = _tree_ref(q, cache, table, mask, (300 + news,), (news,), 256 ** -0.5)
    _close(x, ref, most)


@pytest.mark.parametrize("max_new,max_len", [(1, 1), (0, 0), (1000, 100000), (2 ** 62, 2 ** 62)])
@pytest.mark.parametrize("news", [(1, 2), (70, 3)], ids=str)
def test_hints_only_size_the_launch(dec, news, max_new, max_len):
    _run(dec, (300, 1000), news, 6, 2, 128, 16, BF16, 26, max_new=max_new, max_len=max_len)


@pytest.mark.parametrize("news", [5, 70])
@pytest.mark.parametrize("d,hint", [(64, None), (64, 1 << 24), (192, 1 << 24)])
def test_drafts_past_the_table(dec, news, d, hint):
    """A table that holds some of the drafts, none of them, or not the whole context: what it lacks is not seen."""
    for pages in (1, 3, 6, 7):
        _run(dec, (100 + news,), (news,), 4, 2, d, 16, F16, 27, max_len=hint, change=lambda c, t: t[:, :pages].contiguous())


@pytest.mark.parametrize("news", [4, 50])
@pytest.mark.parametrize("d,hint", [(128, None), (128, 1 << 24), (256, 1 << 24)])
def test_what_a_row_does_not_see_does_not_touch_it(dec, news, d, hint):
    """A draft page that is not finite, far larger, or out of range: NaN for the rows that see one of its rows, and others keep
    their bits."""
    ends, page = (32 + news,), 16
    mask = torch.zeros(news, 1, dtype=I64)
    mask[1::2] = 1  # odd rows see the first draft, in page 2
    q, cache, table, mask, y = _run(dec, ends, (news,), 4, 2, d, page, BF16, 28, mask=mask, max_len=hint)

    def again(t):
        poison_allocator()
        return dec.kv8_tree_attention(q, cache, mask, t, _i32(*ends), _cu((news,)), news, hint or ends[0])

    at = int(table[0, 2])
    was = cache.v_scale[at].clone()
    for bad in (float("nan"), float("inf"), 1e30):
        cache.v_scale[at] = bad
        x = again(table)
        assert torch.equal(x[::2], y[::2])
        assert torch.isnan(x[1::2]).all() if bad != 1e30 else (x[1::2].abs() > 1e20).any()
    cache.v_scale[at] = was
    for pid in (-1, cache.k.shape[0], 2 ** 31 - 1):
        t = table.clone()
        t[0, 2] = pid
        x = again(t)
        assert torch.equal(x[::2], y[::2]) and torch.isnan(x[1::2]).all()


@pytest.mark.parametrize("d,hint", [(128, 70), (128, 1 << 24), (256, 1 << 24)])
def test_rows_behind_the_last_sequence_and_strides(dec, d, hint):
    """A padded batch: rows past the last offset cost nothing and touch nobody; queries and masks are views of wider tensors."""
    g = torch.Generator().manual_seed(29)
    cache = _random_cache(dec, 12, 2, 16, d, g)
    ends, news = (70, 50), (6, 20)
    table = _table(ends, 16, 12, g)
    wide = (torch.randn(40, 9, d, generator=g) * 0.3).to(BF16).cuda()
    q, m = wide[:, 2:8], torch.stack([_random_mask(40, 1, g)[:, 0]] * 3, 1).cuda()[:, 1:2]
    y = dec.kv8_tree_attention(q, cache, m, table, _i32(*ends), _cu(news), 20, hint)
    ref, most = _tree_ref(q[:26], cache, table, m, ends, news, d ** -0.5)
    _close(y[:26], ref, most)
    x = dec.kv8_tree_attention(q[:26], cache, m[:26], table, _i32(*ends), _cu(news), 20, hint)
    assert torch.equal(x, y[:26])


@pytest.mark.parametrize("news", [3, 40])
@pytest.mark.parametrize("d,hint", [(256, 2000), (128, 1 << 24), (256, 1 << 24)])
def test_tree_repeats_and_replays(dec, news, d, hint):
    """The same bits every time, in a graph too; and a graph replayed with other lengths, offsets, masks and pages, which are cut into
    other shares."""
    q, cache, table, mask, y = _run(dec, (900, 2000), (news, news), 12, 2, d, 64, BF16, 30, max_len=hint)
    lens, cu = _i32(900, 2000), _cu((news, news))

    def call():
        return dec.kv8_tree_attention(q, cache, mask, table, lens, cu, news, hint)

    assert torch.equal(call(), y)
    graph_replays_equal(call, y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for ends, at in (((70, 1900), (0, 1, 1 + news)), ((2000, 2000), (0, news, 2 * news)), ((0, 3), (0, 0, news))):
        lens.copy_(_i32(*ends))
        cu.copy_(_i32(*at))
        table.copy_(table.flip(1))
        mask.copy_(mask.flip(0))
        graph.replay()
        torch.cuda.synchronize()
        got = out[:at[-1]].clone()
        assert torch.equal(got.nan_to_num(7), call()[:at[-1]].nan_to_num(7))
        # (a table turned round has pages that are not there: NaN, in the same places)


# ------------------------------------------------------------------------------------------ keep


def _keep_ref(cache, table, path, ends, news):
    """The same moves on the host, row by row: fp32 scales, rounding to even."""
    k, v, ks, vs = (x.cpu().clone() for x in cache)
    pages, heads, page, d = k.shape
    table, path, least = table.cpu(), path.cpu(), 2.0 ** -100
    f32 = torch.float32

    def rounded(c, ratio):
        return torch.nan_to_num(torch.round(c.to(f32) * ratio), nan=0.0).clamp(-127, 127).to(torch.int8)

    room = table.shape[1] * page
    for s, (end, n) in enumerate(zip(ends, news)):
        base, rows = end - n, []
        for r in path[s].tolist():
            if r < 0 or r >= n or (rows and r <= rows[-1]):
                break
            rows.append(r)
        for codes, scales in ((k, ks), (v.transpose(2, 3), vs)):
            dest = sorted({(base + j) // page for j, r in enumerate(rows) if r != j and 0 <= base + j < room})
            for p in dest:
                to = int(table[s, p])
                if not 0 <= to < pages:
                    continue
                js = [j for j, r in enumerate(rows) if r != j and (base + j) // page == p and 0 <= base + j < room]
                where = []
                for j in js:
                    at = base + rows[j]
                    sp = at // page if at < room else -1
                    pid = int(table[s, sp]) if sp >= 0 else -1
                    where.append((sp, pid if 0 <= pid < pages else None, at % page))
                for h in range(heads):
                    was = scales[to, h].clone()
                    need = torch.tensor(0.0)
                    moved = []
                    for sp, pid, off in where:
                        c = codes[pid, h, off].clone() if pid is not None else torch.zeros(d, dtype=torch.int8)
                        sc = scales[pid, h].clone() if pid is not None else torch.tensor(float("nan"))
                        moved.append((sp, pid, off, c, sc))
                        if sp != p:
                            x = (c.abs().max().to(f32) / 127) * sc if sc.isfinite() else sc
                            need = torch.maximum(need, x)  # a NaN stays
                    if need < least:
                        need = torch.tensor(0.0)
                    now = was if need <= was or was.isnan() else need
                    if not now == was:
                        codes[to, h] = rounded(codes[to, h], was / now)
                        scales[to, h] = now
                    for j, (sp, pid, off, c, sc) in zip(js, moved):
                        codes[to, h, (base + j) % page] = codes[to, h, off].clone() if sp == p else rounded(c, sc / now)
    return k, v, ks, vs


def _keep(dec, ends, news, heads, d, page, path, seed, change=None):
    g = torch.Generator().manual_seed(seed)
    pages = sum(-(-max(e, 0) // page) for e in ends) + 2
    cache = _random_cache(dec, pages, heads, page, d, g)
    table = _table(ends, page, pages, g)
    if change:
        table = change(cache, table)
    path = torch.tensor(path, dtype=torch.int32).cuda()
    ref = _keep_ref(cache, table, path, ends, news)
    dec.kv8_keep(cache, path, table, _i32(*ends), _cu(news))
    starts = [max(e - n, 0) for e, n in zip(ends, news)]
    for x, y, name in zip(cache, ref, ("k", "v", "k_scale", "v_scale")):
        x = x.cpu()
        same = torch.equal(torch.nan_to_num(x.float(), nan=-5.0), torch.nan_to_num(y.float(), nan=-5.0))
        d = ((x != y) & ~(x.isnan() & y.isnan())).nonzero()
        assert same, (name, starts, d[:4], [(x[tuple(i)].item(), y[tuple(i)].item()) for i in d[:4]])
    return cache, table


def _path(n, m, g):
    kept = int(torch.randint(1, min(n, m) + 1, (1,), generator=g))
    rows = torch.randperm(n, generator=g)[:kept].sort().values.tolist()
    return rows + [-1] * (m - kept)


@pytest.mark.parametrize("heads,d,page", [(2, 256, 16), (1, 128, 64), (3, 64, 32), (2, 192, 144)])
@pytest.mark.parametrize("news", [(8, 16, 3), (64, 1, 40), (100, 33, 200)], ids=str)
def test_keep(dec, heads, d, page, news):
    """Paths over one page and several, of every length, scales growing by a row from a page of larger values."""
    g = torch.Generator().manual_seed(sum(news))
    for seed in range(3):
        ends = tuple(n + int(torch.randint(300, (1,), generator=g)) for n in news)
        _keep(dec, ends, news, heads, d, page, [_path(n, 24, g) for n in news], seed)


def test_keep_long_paths(dec):
    """A path of 1024 rows of 1100, and one that is the whole tree already."""
    g = torch.Generator().manual_seed(3)
    rows = torch.randperm(1100, generator=g)[:1024].sort().values.tolist()
    _keep(dec, (1107, 1024), (1100, 1024), 1, 64, 16, [rows, list(range(1024))], 3)


@pytest.mark.parametrize("path,kept", [([0, 1, 2, 3], 0), ([-1, 2, 3, 4], 0), ([2, 2, 3, 4], 1), ([3, 1, 2, 4], 1), ([1, 3, 9, 10], 2),
                                       ([2 ** 31 - 1, 1, 2, 3], 0), ([0, 4, -2 ** 31, 7], 2)])
def test_keep_paths_end_where_they_do_not_grow(dec, path, kept):
    _keep(dec, (29,), (9,), 2, 64, 16, [path], 4)


def test_keep_sequences_at_the_edges(dec):
    """No rows, a length below them, a negative one, positions past the table."""
    path = [[1, 3, 4]] * 4
    _keep(dec, (20, 3, -2, 40), (0, 6, 5, 9), 2, 64, 16, path, 5)
    for pages in (1, 2, 3):
        _keep(dec, (50,), (20,), 2, 64, 16, [[0, 2, 5, 17, 19]], 6, change=lambda c, t: t[:, :pages].contiguous())


def test_keep_bad_pages(dec):
    """A row from a page that is not finite or out of range makes the receiving page so; nothing goes to a page out of range."""
    def scale(v):
        def change(c, t):
            c.k_scale[int(t[0, 3])] = v
            c.v_scale[int(t[0, 3])] = v
            return t
        return change

    def page(i, v):
        def change(c, t):
            t[0, i] = v
            return t
        return change

    for change in (scale(float("nan")), scale(float("inf")), scale(0.0), scale(1e-35), page(3, -1), page(3, 1000), page(2, -1), page(2, 99)):
        cache, table = _keep(dec, (64,), (40,), 2, 64, 16, [[0, 3, 10, 25, 30]], 7, change=change)


def test_keep_replays(dec):
    """A captured call, replayed with other paths and lengths: each replay is what an eager call gives."""
    g = torch.Generator().manual_seed(8)
    start = _random_cache(dec, 12, 2, 16, 64, g)
    cache = dec.Kv8Cache(*(x.clone() for x in start))
    table = _table((80, 60), 16, 12, g)
    path, lens, cu = torch.tensor([[0, 5, 9], [2, 4, 30]], dtype=torch.int32).cuda(), _i32(80, 60), _cu((20, 40))

    def call():
        for x, y in zip(cache, start):
            x.copy_(y)
        dec.kv8_keep(cache, path, table, lens, cu)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for turn in range(3):
        if turn == 1:
            path.copy_(torch.tensor([[3, 17, 19], [39, -1, 3]], dtype=torch.int32))
            lens.copy_(_i32(75, 58))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in cache]
        call()
        assert all(torch.equal(x, y) for x, y in zip(got, cache))
        assert not all(torch.equal(x, y) for x, y in zip(got, start))
