"""The 8-bit paged KV cache (decoder.kv8_append, kv8_read, kv8_attention) against plain forms: the
cache's codes and scales exactly, attention against a float64 softmax over the cached values.

Attention's bound: the output is rounded once (2^-9 of it in bf16, 2^-12 in fp16), the softmax's
weights are rounded to fp16 (2^-12 of each, so at most 2^-12 of the largest |v| that the row sees), a
bf16 query keeps all its bits but for values 2^-14 below the row's largest, and fp32 sums over d and the
tokens add far less. With a factor two of room: |y - ref| <= 2^-8 |ref| (fp16 2^-11) + 2^-10 max |v|.
Needs an MI355X."""

import math

import pytest
import torch

from _gpu import graph_replays_equal, poison_allocator

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    assert torch.cuda.is_available(), "GPU tests need an MI355X"


@pytest.fixture(scope="module")
def dec():
    from vllm_gguf_plugin import decoder

    return decoder


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _cu(lens):
    return torch.tensor([0] + list(lens), device="cuda").cumsum(0).to(torch.int32)


def _random_cache(dec, pages, heads, page, d, g):
    """A cache of random codes and scales over four powers of two."""
    def codes(*s):
        return torch.randint(-127, 128, s, generator=g).to(torch.int8).cuda()

    def scales():
        return (torch.exp2(4 * torch.rand(pages, heads, generator=g)) / 300).cuda()

    return dec.Kv8Cache(codes(pages, heads, page, d), codes(pages, heads, d, page), scales(), scales())


def _table(ends, page, pages, g, spare=1):
    need = [-(-max(e, 0) // page) for e in ends]
    assert sum(need) <= pages
    order = torch.randperm(pages, generator=g)
    t = torch.full((len(ends), max(need + [1]) + spare), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        t[i, :n] = order[at:at + n].to(torch.int32)
        at += n
    return t.cuda()


def _values(cache, table, s, n):
    """float64 K and V [heads, n, d] of positions 0 .. n - 1 of sequence s."""
    page = cache.k.shape[2]
    p = table[s, :-(-n // page)].long()
    k = cache.k[p].double() * cache.k_scale[p].double()[..., None, None]
    v = (cache.v[p].double() * cache.v_scale[p].double()[..., None, None]).transpose(2, 3)
    return [x.permute(1, 0, 2, 3).flatten(1, 2)[:, :n] for x in (k, v)]


def _attention_ref(q, cache, table, ends, news, scale):
    """float64 attention and, for each row, the largest |v| that it sees."""
    hq, heads = q.shape[1], cache.k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    most = torch.zeros(q.shape[0], hq, 1, dtype=torch.float64, device="cuda")
    row = 0
    for s, (end, n) in enumerate(zip(ends, news)):
        for i in range(n):
            see = end - n + i + 1
            if see > 0:
                k, v = _values(cache, table, s, see)
                k, v = k.repeat_interleave(hq // heads, 0), v.repeat_interleave(hq // heads, 0)
                x = (k @ q[row + i].double()[..., None])[..., 0] * scale
                out[row + i] = (torch.softmax(x, -1)[:, None] @ v)[:, 0]
                most[row + i] = v.abs().amax((1, 2))[:, None]
        row += n
    return out, most


def _close(y, ref, most):
    eps = 2.0 ** -8 if y.dtype == torch.bfloat16 else 2.0 ** -11
    bad = (y.double() - ref).abs() > eps * ref.abs() + 2.0 ** -10 * most
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}: {(y.double() - ref).abs().max()}"


def _run_attention(dec, ends, news, hq, heads, d, page, dtype, seed, max_new=None, max_len=None, scale=None):
    g = torch.Generator().manual_seed(seed)
    pages = sum(-(-max(e, 0) // page) for e in ends) + 2
    cache = _random_cache(dec, pages, heads, page, d, g)
    table = _table(ends, page, pages, g)
    q = (torch.randn(sum(news), hq, d, generator=g) * 0.3).to(dtype).cuda()
    poison_allocator()
    y = dec.kv8_attention(q, cache, table, _i32(*ends), _cu(news), max_new or max(news), max_len or max(ends), scale)
    ref, most = _attention_ref(q, cache, table, ends, news, scale or d ** -0.5)
    assert y.shape == q.shape and y.dtype == dtype
    _close(y, ref, most)
    return q, cache, table, y


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("hq,heads,d,page", [(6, 1, 256, 16), (8, 2, 128, 32), (4, 4, 64, 144), (5, 1, 192, 64)])
@pytest.mark.parametrize("news", [(1, 1, 1, 1), (1, 3, 0, 7), (5, 40, 2, 17)], ids=str)
def test_attention(dec, dtype, hq, heads, d, page, news):
    """Decode, verify and prompt rows; contexts of one token, of part of a tile and page, of several
    splits."""
    ends = (max(1, news[0]), 65, 200, 777)
    _run_attention(dec, ends, news, hq, heads, d, page, dtype, 11)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("hq,heads,d,page", [(12, 2, 256, 64), (4, 1, 128, 16)])
def test_attention_prompts(dec, dtype, hq, heads, d, page):
    """Prompts of some hundred rows, whole and behind older tokens."""
    _run_attention(dec, (150, 391, 130), (150, 130, 64), hq, heads, d, page, dtype, 12)


@pytest.mark.parametrize("news", [(2, 9, 4), (2, 150, 4)], ids=str)
def test_attention_rows_that_see_nothing(dec, news):
    """A length of 0 (and one below the sequence's own rows, and a negative one) leaves rows without keys: zeros."""
    ends = (0, 5, -3)
    _, _, _, y = _run_attention(dec, ends, news, 6, 2, 128, 16, torch.bfloat16, 13)
    assert (y[:2] == 0).all() and (y[2:2 + news[1] - 5] == 0).all() and (y[-4:] == 0).all()


@pytest.mark.parametrize("max_new,max_len", [(1, 1), (1000, 100000), (3, 64)])
@pytest.mark.parametrize("news", [(1, 2), (70, 3)], ids=str)
def test_attention_hints_only_size_the_launch(dec, news, max_new, max_len):
    _run_attention(dec, (300, 1000), news, 6, 2, 128, 16, torch.bfloat16, 14, max_new, max_len)


def test_attention_without_workspace(dec):
    """The C entry point without a workspace runs unsplit, with part of one in fewer splits."""
    import ctypes

    q, cache, table, y = _run_attention(dec, (3000, 100), (1, 1), 6, 1, 256, 16, torch.bfloat16, 15)

    class T(ctypes.Structure):
        _fields_ = [("data", ctypes.c_void_p), ("dtype", ctypes.c_int32), ("ndim", ctypes.c_int32),
                    ("size", ctypes.c_int64 * 4), ("stride", ctypes.c_int64 * 4), ("device", ctypes.c_int32)]

    class Cache(ctypes.Structure):
        _fields_ = [("k", T), ("v", T), ("k_scale", T), ("v_scale", T)]

    codes = {torch.float32: 0, torch.bfloat16: 2, torch.int8: 5, torch.int32: 6}

    def desc(t):
        r = T(t.data_ptr(), codes[t.dtype], t.dim())
        r.size[:t.dim()], r.stride[:t.dim()], r.device = list(t.shape), list(t.stride()), t.get_device()
        return r

    lib = ctypes.CDLL(dec.LIB_PATH)
    lib.gguf_kv8_attention_workspace_bytes.restype = ctypes.c_size_t
    P = ctypes.byref
    c = Cache(*(desc(t) for t in cache))
    lens, cu = _i32(3000, 100), _cu((1, 1))
    full = lib.gguf_kv8_attention_workspace_bytes(P(c), P(desc(q)), ctypes.c_int64(2), ctypes.c_int64(1), ctypes.c_int64(3000))
    assert full > 0
    ref, most = _attention_ref(q, cache, table, (3000, 100), (1, 1), 256 ** -0.5)
    for nbytes in (0, full // 3, full):
        ws = torch.full((max(nbytes, 16),), 255, dtype=torch.uint8, device="cuda")
        out = torch.full_like(q, float("nan"))
        rc = lib.gguf_kv8_attention(P(desc(q)), P(c), P(desc(table)), P(desc(lens)), P(desc(cu)), ctypes.c_int64(1),
                                    ctypes.c_int64(3000), ctypes.c_float(256 ** -0.5), P(desc(out)),
                                    ctypes.c_void_p(ws.data_ptr() if nbytes else None), ctypes.c_size_t(nbytes),
                                    ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        assert rc == 0
        torch.cuda.synchronize()
        _close(out, ref, most)
        if nbytes == full:
            assert torch.equal(out, y)


@pytest.mark.parametrize("news", [(4, 3), (100, 3)], ids=str)
def test_attention_pages_out_of_range_and_not_finite(dec, news):
    """Rows that see a page whose number is out of range, or whose scale is not finite, are NaN; the others, also
    those that share its tile, are as ever."""
    g = torch.Generator().manual_seed(16)
    hq, heads, d, page = 6, 2, 128, 16
    ends = (180, 120)
    cache = _random_cache(dec, 30, heads, page, d, g)
    table = _table(ends, page, 30, g)
    q = (torch.randn(sum(news), hq, d, generator=g) * 0.3).to(torch.bfloat16).cuda()
    ref, most = _attention_ref(q, cache, table, ends, news, d ** -0.5)
    last = ends[0] - 1  # only the first sequence's last row or rows see its last page
    sees = [ends[0] - news[0] + i >= last // page * page for i in range(news[0])] + [False] * news[1]
    bad = torch.tensor(sees, device="cuda")
    for spoil in ("far", "negative", "k inf", "k nan", "v inf", "v nan"):
        t, c = table.clone(), dec.Kv8Cache(*(x.clone() for x in cache))
        where = (0, last // page)
        if spoil == "far":
            t[where] = 30
        elif spoil == "negative":
            t[where] = -7
        else:
            x = c.k_scale if spoil[0] == "k" else c.v_scale
            x[t[where].long()] = float(spoil[2:])
            (c.k if spoil[0] == "k" else c.v)[t[where].long()] = 0  # what kv8_append leaves there
        y = dec.kv8_attention(q, c, t, _i32(*ends), _cu(news), max(news), max(ends))
        assert y[bad].isnan().all(), spoil
        _close(y[~bad], ref[~bad], most[~bad])


def test_attention_extreme_scales(dec):
    """V scales over 2^60, and K scales that make one token take all: nothing overflows on the way."""
    g = torch.Generator().manual_seed(17)
    heads, page, d = 2, 16, 128
    cache = _random_cache(dec, 20, heads, page, d, g)
    cache.v_scale.copy_(torch.exp2(60 * torch.rand(20, heads, generator=g) - 30))
    cache.k_scale[3:6] *= 200
    ends, news = (300,), (3,)
    table = _table(ends, page, 20, g)
    q = torch.randn(3, 4, d, generator=g).cuda()
    for dtype, by in ((torch.bfloat16, 1.0), (torch.bfloat16, 2.0 ** 40), (torch.bfloat16, 2.0 ** -40), (torch.float16, 1.0)):
        x = (q * by).to(dtype)
        scale = 0.05 / by
        y = dec.kv8_attention(x, cache, table, _i32(*ends), _cu(news), 3, 300, scale)
        ref, most = _attention_ref(x, cache, table, ends, news, scale)
        if dtype == torch.float16:  # the output's own range
            ref, most = ref.clamp(-65504, 65504), most
            y = y.double().clamp(-65504, 65504).to(torch.float16)
        _close(y, ref, most)


def test_attention_strided_query_other_stream_and_graph(dec):
    """A query that is a slice of a wider projection, on another stream, and replayed from a graph."""
    g = torch.Generator().manual_seed(18)
    hq, heads, d, page = 24, 4, 256, 64
    ends, news = (500, 901, 64), (1, 4, 1)
    cache = _random_cache(dec, 30, heads, page, d, g)
    table = _table(ends, page, 30, g)
    wide = (torch.randn(6, hq, 2 * d, generator=g) * 0.3).to(torch.bfloat16).cuda()
    q = wide[..., :d]
    lens, cu = _i32(*ends), _cu(news)
    ref, most = _attention_ref(q, cache, table, ends, news, d ** -0.5)
    y = dec.kv8_attention(q, cache, table, lens, cu, 4, 901)
    _close(y, ref, most)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = dec.kv8_attention(q, cache, table, lens, cu, 4, 901)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, z)
    graph_replays_equal(lambda: dec.kv8_attention(q, cache, table, lens, cu, 4, 901), y)


def test_offsets_past_32_bits(dec):
    """A pool of more than 2^31 codes, the sequence in its last pages: appended, read back, attended."""
    heads, page, d = 1, 256, 256
    pages = 2 ** 31 // (page * d) + 9
    cache = dec.Kv8Cache.empty(pages, heads, page, d)
    n = 700
    table = torch.tensor([[pages - 1, pages - 3, pages - 2]], dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(19)
    k, v = (torch.randn(n, heads, d, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    dec.kv8_append(cache, k, v, table, _i32(n), _cu((n,)), n)
    kr, vr = dec.kv8_read(cache, table, _i32(0), _cu((n,)), n, n, torch.float32)
    for x, y in ((k, kr), (v, vr)):  # half a step of at most amax / 127
        assert (x.float() - y).abs().max() <= x.abs().max().float() / 127 * 0.5001
    q = (torch.randn(2, 6, d, generator=g) * 0.3).to(torch.bfloat16).cuda()
    y = dec.kv8_attention(q, cache, table, _i32(n), _cu((2,)), 2, n)
    ref, most = _attention_ref(q, cache, table, (n,), (2,), d ** -0.5)
    _close(y, ref, most)
    assert not cache.k_scale[:pages - 3].any() and not cache.k[:4].any()


# ------------------------------------------------------------------------------ append and read


def _append_ref(cache, key, value, table, ends, news):
    """The contract in float32 on the host, token group by token group of a page."""
    k, v, ks, vs = (t.cpu().clone() for t in cache)
    page, room = k.shape[2], table.shape[1] * k.shape[2]
    table, key, value = table.cpu(), key.cpu().float(), value.cpu().float()
    row = 0
    for s, (end, n) in enumerate(zip(ends, news)):
        start = end - n
        p = max(start, 0)
        while p < min(end, room):
            hi = min(end, room, (p // page + 1) * page)
            pid, lo = int(table[s, p // page]), p % page
            if 0 <= pid < k.shape[0]:
                for x, codes, scale, turned in ((key, k, ks, False), (value, v, vs, True)):
                    new = x[row + p - start:row + hi - start]  # [t, heads, d]
                    for h in range(k.shape[1]):
                        c = codes[pid, h].T if turned else codes[pid, h]  # [page, d] view
                        fresh = new[:, h].abs().amax() / 127 if not new[:, h].isnan().any() else torch.tensor(math.nan)
                        if fresh < 2.0 ** -100:
                            fresh = torch.tensor(0.0)
                        was = scale[pid, h].clone() if lo > 0 and start < p // page * page + page and start > p // page * page \
                            else torch.tensor(0.0)
                        now = was if was.isnan() or fresh <= was else fresh
                        if lo > 0 and was != now:
                            c[:lo] = torch.nan_to_num(torch.round(c[:lo].float() * (was / now)), 0, 0, 0).to(torch.int8)
                        inv = 1 / now if now > 0 else torch.tensor(0.0)
                        c[lo:lo + hi - p] = torch.nan_to_num(torch.round(new[:, h] * inv), 0, 0, 0).clamp(-127, 127).to(torch.int8)
                        scale[pid, h] = now
            p = hi
        row += n
    return k, v, ks, vs


def _check_append(dec, cache, key, value, table, ends, news, max_new=None):
    ref = _append_ref(cache, key, value, table, ends, news)
    dec.kv8_append(cache, key, value, table, _i32(*ends), _cu(news), max_new or max(max(news), 1))
    for name, got, want in zip(cache._fields, cache, ref):
        assert torch.equal(got.cpu().nan_to_num(-1), want.nan_to_num(-1)), name


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("heads,d,page", [(2, 128, 16), (1, 256, 64), (3, 64, 144), (1, 192, 32)])
def test_append(dec, dtype, heads, d, page):
    """Prompts, then single tokens and verify groups on top (growing scales), into shuffled pages that
    hold other codes; a sequence without rows; a hint that is too small."""
    g = torch.Generator().manual_seed(21)
    news = (page + 5, 1, 0, 3 * page, 17)
    ends = news
    cache = _random_cache(dec, 40, heads, page, d, g)
    table = _table([e + 2 * page for e in ends], page, 40, g)
    def rows(n, by=1.0):
        return [(torch.randn(n, heads, d, generator=g) * by).to(dtype).cuda() for _ in range(2)]

    _check_append(dec, cache, *rows(sum(news)), table, ends, news, max_new=1)
    for more, by in (((1, 1, 1, 1, 1), 1.0), ((1, 1, 0, 1, 1), 2.0), ((4, 3, 2, 1, page), 0.01), ((1, 2, 3, 4, 5), 30.0)):
        ends = tuple(e + m for e, m in zip(ends, more))
        _check_append(dec, cache, *rows(sum(more), by), table, ends, more)


def test_append_strided_zero_and_not_finite(dec):
    g = torch.Generator().manual_seed(22)
    heads, d, page = 2, 128, 16
    cache = _random_cache(dec, 12, heads, page, d, g)
    table = _table((100,), page, 12, g)
    wide = torch.randn(20, 2 * heads * d + 64, generator=g).to(torch.bfloat16).cuda()
    k = wide[:, :heads * d].view(20, heads, d)
    v = wide[:, heads * d:2 * heads * d].view(20, heads, d)
    _check_append(dec, cache, k, v, table, (20,), (20,))
    zero = torch.zeros(40, heads, d, dtype=torch.bfloat16, device="cuda")
    _check_append(dec, cache, zero, zero, table, (60,), (40,))
    tiny = (torch.randn(2, heads, d, generator=g) * 1e-36).float().cuda()
    _check_append(dec, cache, tiny, tiny, table, (66,), (2,))
    for bad in (math.inf, -math.inf, math.nan):
        x = torch.randn(3, heads, d, generator=g).to(torch.bfloat16).cuda()
        x[1, 0, 5] = bad
        _check_append(dec, cache, x, x.flip(1), table, (83,), (3,))
        kr, _ = dec.kv8_read(cache, table, _i32(80), _cu((3,)), 3, 3)
        assert kr[:, 0].isnan().all() and not kr[:, 1].isnan().any()
        # and a later token does not bring the page back
        y = torch.randn(1, heads, d, generator=g).to(torch.bfloat16).cuda()
        _check_append(dec, cache, y, y, table, (84,), (1,))


def test_append_drops_what_has_no_place(dec):
    """Rows before position 0, past the table, or in a page out of range leave everything else alone."""
    g = torch.Generator().manual_seed(23)
    heads, d, page = 1, 64, 16
    cache = _random_cache(dec, 6, heads, page, d, g)
    table = torch.tensor([[0, 1], [2, -1], [6, 3]], dtype=torch.int32, device="cuda")
    k, v = (torch.randn(60, heads, d, generator=g).cuda() for _ in range(2))
    _check_append(dec, cache, k, v, table, (40, 5, 20), (20, 20, 20))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("heads,d,page", [(2, 128, 16), (1, 256, 64), (2, 64, 144), (1, 192, 32)])
def test_read(dec, dtype, heads, d, page):
    g = torch.Generator().manual_seed(24)
    ends = (1, 3 * page, 2 * page + 7, 40)
    cache = _random_cache(dec, 20, heads, page, d, g)
    table = _table(ends, page, 20, g)
    starts, ns = (0, page - 3, 5, 17), (1, page + 4, 0, 23)
    poison_allocator()
    k, v = dec.kv8_read(cache, table, _i32(*starts), _cu(ns), sum(ns), 1, dtype)
    row = 0
    for s, (a, n) in enumerate(zip(starts, ns)):
        kd, vd = _values(cache, table, s, ends[s])
        # code * scale is one fp32 product, then rounded to dtype
        assert torch.equal(k[row:row + n], kd[:, a:a + n].transpose(0, 1).float().to(dtype))
        assert torch.equal(v[row:row + n], vd[:, a:a + n].transpose(0, 1).float().to(dtype))
        row += n


def test_read_out_of_range_is_nan(dec):
    g = torch.Generator().manual_seed(25)
    cache = _random_cache(dec, 4, 1, 16, 64, g)
    table = torch.tensor([[1, 4]], dtype=torch.int32, device="cuda")
    k, v = dec.kv8_read(cache, table, _i32(-3), _cu((60,)), 60, 60)
    for x in (k, v):
        assert x[:3].isnan().all() and not x[3:19].isnan().any() and x[19:].isnan().all()


def test_append_and_read_in_a_graph(dec):
    g = torch.Generator().manual_seed(26)
    heads, d, page = 2, 128, 16
    cache = _random_cache(dec, 8, heads, page, d, g)
    table = _table((50, 30), page, 8, g)
    k, v = (torch.randn(5, heads, d, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    lens, cu, starts, cu_read = _i32(50, 30), _cu((4, 1)), _i32(0, 0), _cu((50, 30))

    # the same rows again change nothing: their scales are there, and the older codes are on them
    def step():
        dec.kv8_append(cache, k, v, table, lens, cu, 4)
        return dec.kv8_read(cache, table, starts, cu_read, 80, 50)[1]

    graph_replays_equal(step, step())


def _near(y, ref, most):
    """_close, and no NaN (which compares as not beyond any bound)."""
    assert not y.isnan().any()
    _close(y, ref, most)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("news", [(2, 9), (2, 150)], ids=str)
def test_attention_negative_scale(dec, dtype, news):
    """A scale below 0, with scores some 50 apart, in the form for few rows and in that for many."""
    q, cache, table, y = _run_attention(dec, (300, 400), news, 6, 2, 128, 16, dtype, 27, scale=-1.0)
    _near(y, *_attention_ref(q, cache, table, (300, 400), news, -1.0))


@pytest.mark.parametrize("hint", [2 ** 62, 2 ** 63 - 1])
def test_hints_beyond_every_size(dec, hint):
    g = torch.Generator().manual_seed(33)
    for news in ((1, 2), (70, 3)):
        for hq in (6, 8):
            q, cache, table, y = _run_attention(dec, (300, 1000), news, hq, 2, 128, 16, torch.bfloat16, 14, hint, hint)
            _near(y, *_attention_ref(q, cache, table, (300, 1000), news, 128 ** -0.5))
    k, v = (torch.randn(5, 2, 128, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    _check_append(dec, cache, k, v, table, (300, 1000), (2, 3), max_new=hint)
    k, _ = dec.kv8_read(cache, table, _i32(0, 0), _cu((300, 20)), 320, hint, torch.float32)
    assert torch.equal(k[:300], _values(cache, table, 0, 300)[0].transpose(0, 1).float())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("hq,heads,d", [(6, 2, 128), (6, 1, 256)])
@pytest.mark.parametrize("news", [3, 8, 70])
def test_attention_large_v_scale_unseen(dec, news, hq, heads, d, dtype):
    """A page of far larger values takes nothing from the rows before it, which share its tile but do not see it."""
    g = torch.Generator().manual_seed(28)
    end, page = 97, 16
    cache = _random_cache(dec, 9, heads, page, d, g)
    table = _table((end,), page, 9, g)
    cache.v_scale[table[0, end // page].long()] = 2.0 ** 40  # the last token's page, which the last row alone sees
    q = (torch.randn(news, hq, d, generator=g) * 0.3).to(dtype).cuda()
    y = dec.kv8_attention(q, cache, table, _i32(end), _cu((news,)), news, end)
    ref, most = _attention_ref(q, cache, table, (end,), (news,), d ** -0.5)
    _near(y[:-1], ref[:-1], most[:-1])
    if dtype == torch.bfloat16:  # (past fp16's range)
        _near(y[-1:], ref[-1:], most[-1:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("news", [1, 70])
def test_attention_many_small_weights(dec, news, dtype):
    """Half a million tokens of 2^-26 of the first one's weight each, which together are a hundredth of the sum; the first one's
    value is 0."""
    n, d, page = 1 << 19, 64, 256
    cache = dec.Kv8Cache.empty(n // page, 1, page, d)
    table = torch.arange(n // page, dtype=torch.int32, device="cuda")[None]
    cache.k[0, 0, 0] = 127
    g = torch.Generator(device="cuda").manual_seed(29)
    cache.v.copy_(torch.randint(90, 110, cache.v.shape, device="cuda", generator=g))
    cache.v[0, 0, :, 0] = 0
    cache.k_scale.fill_(26 * math.log(2) / (127 * d * 0.125))
    cache.v_scale.fill_(1 / 127)
    q = torch.ones(news, 1, d, dtype=dtype, device="cuda")
    y = dec.kv8_attention(q, cache, table, _i32(n), _cu((news,)), news, 1)  # (one split)
    k, v = _values(cache, table, 0, n)
    w = torch.exp((k[0, :, 0] - k[0, 0, 0]) * d * 0.125)  # all queries are ones, and a key's values alike
    for i in (0, news - 1):
        see = n - news + i + 1
        ref = (w[:see] @ v[0, :see]) / w[:see].sum()
        _near(y[i], ref[None], v.abs().max())


@pytest.mark.parametrize("news", [2, 70])
def test_attention_v_scales_below_the_least(dec, news):
    """V scales below 2^-100, which kv8_append never leaves, count as 0 here too, alone and among others."""
    g = torch.Generator().manual_seed(34)
    heads, page, d, end = 2, 16, 128, 200
    cache = _random_cache(dec, 14, heads, page, d, g)
    table = _table((end,), page, 14, g)
    q = (torch.randn(news, 6, d, generator=g) * 0.3).to(torch.bfloat16).cuda()
    for every in (True, False):
        cache.v_scale[::1 if every else 2] = 1e-40
        y = dec.kv8_attention(q, cache, table, _i32(end), _cu((news,)), news, end)
        if every:
            assert (y == 0).all()
            cache.v_scale.fill_(0.01)
        else:
            _near(y, *_attention_ref(q, cache, table, (end,), (news,), d ** -0.5))


@pytest.mark.parametrize("news", [3, 70])
def test_attention_queries_at_the_end_of_the_range(dec, news):
    """bf16 queries of 2^127 and more, with a scale that makes ordinary scores of them."""
    g = torch.Generator().manual_seed(30)
    heads, page, d, end = 2, 16, 128, 200
    cache = _random_cache(dec, 14, heads, page, d, g)
    cache.k_scale.mul_(0.05)
    table = _table((end,), page, 14, g)
    q = (torch.randn(news, 6, d, generator=g).clamp(-3.9, 3.9) * 2.0 ** 125).to(torch.bfloat16)
    q[:, :, 7] = 1.5 * 2.0 ** 127
    q = q.cuda()
    y = dec.kv8_attention(q, cache, table, _i32(end), _cu((news,)), news, end, 2.0 ** -126)
    ref, most = _attention_ref(q, cache, table, (end,), (news,), 2.0 ** -126)
    _near(y, ref, most)


def _far_scores(dec, news, log_k_scale):
    """Scores of -2^(53 + log_k_scale) times whole numbers: the largest takes all."""
    page, d, end = 16, 64, 75
    cache = dec.Kv8Cache.empty(6, 1, page, d)
    g = torch.Generator().manual_seed(31)
    table = _table((end,), page, 6, g)
    order = 20 + torch.randperm(100, generator=g)[:96].view(6, 1, page, 1)
    cache.k.copy_(order.expand(6, 1, page, d))
    cache.v.copy_(torch.randint(-127, 128, cache.v.shape, generator=g))
    cache.k_scale.fill_(2.0 ** log_k_scale)
    cache.v_scale.fill_(0.01)
    q = torch.full((news, 1, d), -2.0 ** 50, dtype=torch.bfloat16, device="cuda")
    y = dec.kv8_attention(q, cache, table, _i32(end), _cu((news,)), news, end)
    _near(y, *_attention_ref(q, cache, table, (end,), (news,), d ** -0.5))


@pytest.mark.parametrize("news", [1, 70])
def test_attention_scores_beyond_2_to_24(dec, news):
    """Where a score's rounding is far more than the range of a weight."""
    _far_scores(dec, news, 10)


@pytest.mark.parametrize("news", [1, 70])
def test_attention_scores_far_below_zero(dec, news):
    """Scores below -1e30 are scores all the same."""
    _far_scores(dec, news, 43)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("news", [3, 70])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_attention_queries_that_are_not_finite(dec, bad, news, dtype):
    """A query row with an infinity or a NaN is NaN, also where all of its scores are -inf; the others are as ever."""
    g = torch.Generator().manual_seed(32)
    heads, page, d, end = 2, 16, 64, 150
    cache = _random_cache(dec, 12, heads, page, d, g)
    cache.k[..., 5] = -7
    table = _table((end,), page, 12, g)
    q = (torch.randn(news, 6, d, generator=g) * 0.3).to(dtype).cuda()
    ref, most = _attention_ref(q, cache, table, (end,), (news,), d ** -0.5)
    q[1, 4, 5] = bad
    y = dec.kv8_attention(q, cache, table, _i32(end), _cu((news,)), news, end)
    assert y[1, 4].isnan().all()
    y[1, 4], ref[1, 4] = 0, 0
    _near(y, ref, most)


def test_attention_more_rows_than_a_join_takes(dec):
    """2^24 rows of a hint that would split them: unsplit. (They see nothing, but for the last token's.)"""
    hq, d, tokens = 64, 64, (1 << 18) + 3
    g = torch.Generator().manual_seed(35)
    cache = _random_cache(dec, 3, hq, 16, d, g)
    table = _table((20,), 16, 3, g)
    q = torch.zeros(tokens, hq, d, dtype=torch.bfloat16, device="cuda")
    q[-20:] = torch.randn(20, hq, d, generator=g).cuda()
    y = dec.kv8_attention(q, cache, table, _i32(20), _cu((tokens,)), 1, 100000)
    ref, most = _attention_ref(q[-20:], cache, table, (20,), (20,), d ** -0.5)
    assert (y[:-20] == 0).all()
    _near(y[-20:], ref, most)


@pytest.mark.parametrize("hq,heads,d,page", [(6, 1, 256, 64), (4, 2, 128, 16), (2, 2, 64, 144)])
@pytest.mark.parametrize("news", [3, 70])
@pytest.mark.parametrize("end", [4095, 4097, 4128, 8200])
def test_attention_past_a_segment(dec, end, news, hq, heads, d, page):
    """Contexts in one split (a hint of 1) of more tokens than either kernel looks up at a time, and of just fewer."""
    q, cache, table, y = _run_attention(dec, (end, 70), (news, 2), hq, heads, d, page, torch.bfloat16, 36, max_len=1)
    _near(y, *_attention_ref(q, cache, table, (end, 70), (news, 2), d ** -0.5))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("hq,heads,d,page", [(6, 1, 256, 16), (8, 2, 128, 32), (4, 4, 64, 144), (5, 1, 192, 64)])
@pytest.mark.parametrize("news", [(1, 1, 1, 1), (1, 3, 0, 7), (5, 40, 2, 17), (1, 65, 200, 130)], ids=str)
def test_attention_gives_numbers(dec, news, hq, heads, d, page, dtype):
    """The sizes above once more, where a NaN counts."""
    ends = (1 if news[0] == 1 else 5, 65, 200, 777)
    q, cache, table, y = _run_attention(dec, ends, news, hq, heads, d, page, dtype, 37)
    _near(y, *_attention_ref(q, cache, table, ends, news, d ** -0.5))


def test_attention_of_many_short_sequences(dec):
    """More than 65,535 (sequence, head) pairs in a decode step; all sequences lie in the same pages, up to a length of their own."""
    g = torch.Generator().manual_seed(38)
    seqs, heads, d, page, longest = 9001, 8, 64, 16, 40
    cache = _random_cache(dec, 3, heads, page, d, g)
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda").expand(seqs, 3).contiguous()
    lens = (torch.arange(seqs) % longest + 1).to(torch.int32).cuda()
    q = (torch.randn(seqs, 2 * heads, d, generator=g) * 0.3).to(torch.bfloat16).cuda()
    y = dec.kv8_attention(q, cache, table, lens, _cu((1,) * seqs), 1, longest)
    k, v = (x.repeat_interleave(2, 0) for x in _values(cache, table, 0, longest))
    x = torch.matmul(q.double().transpose(0, 1), k.transpose(1, 2).contiguous()) * d ** -0.5  # [heads, seqs, tokens]
    x.masked_fill_(torch.arange(longest, device="cuda") >= lens[:, None], -math.inf)
    ref = torch.matmul(torch.softmax(x, -1), v).transpose(0, 1)
    seen = v.abs().amax(-1).cummax(-1).values  # [heads, tokens]
    _near(y, ref, seen.T[lens.long() - 1][..., None])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("news", [3, 70])
def test_attention_queries_with_a_strong_element(dec, news, dtype):
    """One element 300 times the others. With many rows the others keep 2^-15 of it: that much of the keys' sums of a score, and
    twice as much of a weight, at most, on top of the usual bound."""
    g = torch.Generator().manual_seed(39)
    hq, heads, page, d, end = 6, 2, 16, 128, 300
    cache = _random_cache(dec, 20, heads, page, d, g)
    cache.k[..., 9] = torch.randint(-3, 4, (20, heads, page), generator=g).to(torch.int8)
    table = _table((end,), page, 20, g)
    q = torch.randn(news, hq, d, generator=g) * 0.1
    q[..., 9] = 30.0
    q = q.to(dtype).cuda()
    y = dec.kv8_attention(q, cache, table, _i32(end), _cu((news,)), news, end)
    ref, most = _attention_ref(q, cache, table, (end,), (news,), d ** -0.5)
    room = 0.0
    if news * hq // heads > 64:
        sums = _values(cache, table, 0, end)[0].abs().sum(-1).amax()
        room = 2 * 2.0 ** -15 * 30.0 * float(sums) * d ** -0.5
    assert not y.isnan().any()
    eps = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    assert ((y.double() - ref).abs() <= eps * ref.abs() + (2.0 ** -10 + room) * most).all()
