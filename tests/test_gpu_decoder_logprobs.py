"""decoder.token_logprobs against float64 log_softmax and a stable sort.

Bounds: Z and A are fp32 sums of positive (of one-signed) terms, each within a few 2^-24, in a fixed tree of
depth below 32: log Z within 2^-19, x - m exact to 2^-24 of it: 2^-18 + 2^-22 |value|. Needs an MI355X."""

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


def _close(got, want):
    want = want.to(got.device)
    same = (got.double() == want) | (got.isnan() & want.isnan())
    ok = same | ((got.double() - want).abs() <= 2.0 ** -18 + 2.0 ** -22 * want.abs())
    assert ok.all(), float((got.double() - want).abs().nan_to_num().max())


def _check(dec, x, ids, top):
    poison_allocator()
    lp, rank, ent, tlp, tid = dec.token_logprobs(x, ids, top)
    rows, vocab = x.shape
    assert [t.dtype for t in (lp, rank, ent, tlp, tid)] == [torch.float32, torch.int32, torch.float32, torch.float32, torch.int32]
    assert tlp.shape == tid.shape == (rows, top)
    xd = x.double()
    ref = torch.log_softmax(xd, -1)
    order = torch.sort(xd, descending=True, stable=True).indices
    ok = (ids >= 0) & (ids < vocab)
    at = ids.clamp(0, vocab - 1)[:, None]
    _close(lp, torch.where(ok, ref.gather(1, at)[:, 0], float("nan")))
    place = (order == at).int().argmax(-1) + 1
    assert torch.equal(rank, torch.where(ok, place, 0).int())
    p = ref.exp()
    _close(ent, -torch.where(p == 0, 0.0, p * ref).sum(-1))
    assert torch.equal(tid, order[:, :top].int())
    _close(tlp, ref.gather(1, order[:, :top]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("rows,vocab,top", [(1, 151936, 20), (3, 248320, 64), (5, 50257, 1), (4, 100, 64), (2, 8191, 0),
                                            (2, 8193, 5), (7, 1, 1), (3, 65, 64), (2, 2, 2)])
def test_rows(dec, dtype, rows, vocab, top):
    """Vocabularies of one chunk and many, odd ones (rows that start off every 16-byte boundary); 16-bit
    logits have many ties."""
    g = torch.Generator().manual_seed(41)
    x = (torch.randn(rows, vocab, generator=g) * 3).to(dtype).cuda()
    _check(dec, x, torch.randint(vocab, (rows,), generator=g).cuda(), top)


def test_every_start_of_a_row(dec):
    """Slices of a wider tensor: each element offset of a 16-byte piece, rows further apart than they are long."""
    g = torch.Generator().manual_seed(42)
    for dtype in (torch.float32, torch.bfloat16):
        wide = torch.randn(3, 20011, generator=g).to(dtype).cuda()
        for off in range(9):
            x = wide[:, off:off + 16500 + off]
            _check(dec, x, torch.randint(16500, (3,), generator=g).cuda(), 8)


@pytest.mark.parametrize("kind", ["equal", "ascending", "descending", "masked", "one left", "zeros of both signs", "far apart"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_hard_orders(dec, kind, dtype):
    vocab = 20000
    x = torch.zeros(2, vocab)
    if kind == "ascending":
        x += torch.arange(vocab) * 1e-3
    elif kind == "descending":
        x -= torch.arange(vocab) * 1e-3
    elif kind == "masked":  # a grammar's mask: whole chunks of -inf
        x[:] = -torch.inf
        x[0, 7000:7040] = torch.randn(40, generator=torch.Generator().manual_seed(1))
        x[1, ::5000] = 1.0
    elif kind == "one left":
        x[:] = -torch.inf
        x[:, 12345] = 3.0
    elif kind == "zeros of both signs":
        x[:, ::3] = -0.0
    elif kind == "far apart":
        x[:, 10] = 80.0
        x[:, 15000] = -80.0
        x[1] *= 1e30 if dtype == torch.float32 else 1.0
    _check(dec, x.to(dtype).cuda(), torch.tensor([12345, 15000]).cuda(), 64)


def test_lowest_values_as_masks(dec):
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        x = torch.full((2, 9000), torch.finfo(dtype).min, dtype=dtype)
        x[0, 17], x[0, 8500] = 2.0, 1.0
        _check(dec, x.cuda(), torch.tensor([17, 4000]).cuda(), 5)


def test_no_distribution(dec):
    """A row of -inf alone, of a +inf or a NaN has NaN log probabilities and entropy, as log_softmax has; its
    neighbours are as ever."""
    g = torch.Generator().manual_seed(43)
    x = torch.randn(4, 30000, generator=g)
    x[0], x[1, 29999], x[2, 5] = -torch.inf, torch.inf, torch.nan
    lp, rank, ent, tlp, tid = dec.token_logprobs(x.cuda(), torch.tensor([3, 4, 5, 6]).cuda(), 3)
    assert lp[:3].isnan().all() and ent[:3].isnan().all() and tlp[:3].isnan().all()
    assert tid[0].tolist() == [0, 1, 2] and int(tid[1, 0]) == 29999 and int(tid[2, 0]) == 5
    _check(dec, x[3:].cuda(), torch.tensor([6]).cuda(), 3)


def test_token_ids_out_of_range(dec):
    x = torch.randn(4, 1000, generator=torch.Generator().manual_seed(44)).cuda()
    _check(dec, x, torch.tensor([-1, 1000, 2 ** 40, 999]).cuda(), 4)


def test_strided_ids_no_rows_many_rows(dec):
    g = torch.Generator().manual_seed(45)
    x = torch.randn(66000, 40, generator=g).to(torch.float16).cuda()  # more rows than a launch's second dimension
    ids = torch.randint(40, (66000, 2), generator=g).cuda()[:, 1]
    _check(dec, x, ids, 3)
    assert [t.shape[0] for t in dec.token_logprobs(x[:0], ids[:0], 3)] == [0] * 5


def test_other_stream_and_graph(dec):
    g = torch.Generator().manual_seed(46)
    x = torch.randn(3, 151936, generator=g).to(torch.bfloat16).cuda()
    ids = torch.randint(151936, (3,), generator=g).cuda()
    ref = dec.token_logprobs(x, ids, 20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = dec.token_logprobs(x, ids, 20)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(ref, got))
    for i in range(5):
        graph_replays_equal(lambda: dec.token_logprobs(x, ids, 20)[i], ref[i])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("rows,vocab,top", [(1, 524289, 64), (1, 600000, 64), (3, 600000, 64), (1, 1048575, 33),
                                            (1, 1040000, 16), (2, 1100000, 64)])
def test_wide_rows_with_many_best(dec, rows, vocab, top, dtype):
    """So many chunks that their best are more than a merge of small chunks would hold; the best tokens in the last
    columns."""
    g = torch.Generator().manual_seed(47)
    x = torch.randn(rows, vocab, generator=g)
    x[:, -top:] += 20
    _check(dec, x.to(dtype).cuda(), torch.randint(vocab - top, vocab, (rows,), generator=g).cuda(), top)


@pytest.mark.parametrize("rows", [2, 70])  # chunks of 2048 and of 8192 columns
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("kind", ["among masked", "chunks of NaN", "far below"])
def test_a_nan_far_from_the_maximum(dec, kind, dtype, rows):
    """A NaN whose chunk has nothing that counts beside the row's maximum makes the row NaN all the same."""
    g = torch.Generator().manual_seed(48)
    x = torch.randn(rows, 30000, generator=g)
    first = 20000
    if kind == "chunks of NaN":
        first = 8000
        x[0, first:] = torch.nan
    else:
        x[0, 8000:] = -torch.inf if kind == "among masked" else -200.0
        x[0, first] = torch.nan
    x = x.to(dtype).cuda()
    ids = torch.full((rows,), 3).cuda()
    lp, _, ent, tlp, tid = dec.token_logprobs(x, ids, 3)
    assert lp[0].isnan() and ent[0].isnan() and tlp[0].isnan().all() and int(tid[0, 0]) == first
    _check(dec, x[1:], ids[1:], 3)
