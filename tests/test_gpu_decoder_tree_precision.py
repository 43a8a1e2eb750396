"""How precise decoder.kv8_tree_attention is in fp16, in its form for few rows and in the one for many, against a float64 softmax over the
cached values.

Two roundings to fp16 matter, by at most half a step, 2^-11 of the value (and 2^-25 below the normal range), so by no more than
2^-11 / sqrt(3) on average (root mean square; less where the values spread over their binades): of the output, and of each weight times its V scale, independently, which
moves the output by 2^-11 / sqrt(3) * sqrt(sum w^2 v^2). A weight's type has a least step too: 2^-30 of the largest, as the row's
largest weight is at least 64 of fp16's when it is rounded; half of that, over all tokens, is far below. Scores, sums and the exponential are fp32: scores
of up to 20, an accumulation of up to 16 MFMAs, are off by less than 2^-17, so are weights. Allowed are 1.25 times the two roundings' mean and
2^-15 of sum w |v|; at no place more than 2^-11 |y| + 2^-11 sum w |v| and the same 2^-15. Needs an MI355X."""

import pytest
import torch

from _gpu import poison_allocator
from test_gpu_decoder_kv8 import _cu, _i32, _random_cache, _table, _values
from test_gpu_decoder_tree import HINTS, _bits, _random_mask, _run

pytestmark = pytest.mark.gpu
F16 = torch.float16


@pytest.fixture(scope="module")
def dec():
    from vllm_gguf_plugin import decoder

    assert torch.cuda.is_available(), "GPU tests need an MI355X"
    return decoder


@pytest.mark.parametrize("hint", HINTS)
@pytest.mark.parametrize("hq,heads,d,page", [(4, 2, 64, 64), (4, 2, 128, 16), (3, 1, 192, 32), (6, 2, 256, 64)])
@pytest.mark.parametrize("by", [0.3, 1.0])
def test_roundings(dec, hq, heads, d, page, by, hint):
    """Flat and peaked distributions over some hundred to some thousand tokens."""
    g = torch.Generator().manual_seed(51)
    ends, news = (2100, 333, 77), (40, 33, 50)
    cache = _random_cache(dec, sum(-(-e // page) for e in ends) + 2, heads, page, d, g)
    table, mask = _table(ends, page, cache.k.shape[0], g), _random_mask(sum(news), 1, g)
    q = (torch.randn(sum(news), hq, d, generator=g) * by).to(F16).cuda()
    poison_allocator()
    y = dec.kv8_tree_attention(q, cache, mask.cuda(), table, _i32(*ends), _cu(news), max(news), hint or max(ends)).double()
    row, square, allowed = 0, 0.0, 0.0
    for s, (end, n) in enumerate(zip(ends, news)):
        k, v = (x.repeat_interleave(hq // heads, 0) for x in _values(cache, table, s, end))
        see = torch.ones(n, end, dtype=torch.bool)
        see[:, end - n:] = _bits(mask[row:row + n], n)
        x = torch.matmul(q[row:row + n].double().transpose(0, 1), k.transpose(1, 2).contiguous()) * d ** -0.5
        w = torch.softmax(x.masked_fill(~see.cuda()[None], -torch.inf), -1)
        assert (w.sum(-1) - 1).abs().max() < 1e-9
        ref, size, mean = (w @ v).transpose(0, 1), (w @ v.abs()).transpose(0, 1), (w.square() @ v.square()).transpose(0, 1)
        off = (y[row:row + n] - ref).abs()
        bad = off > 2.0 ** -11 * ref.abs() + (2.0 ** -11 + 2.0 ** -15) * size
        assert not bad.any(), (int(bad.sum()), bad.nonzero()[:3])
        square += off.square().sum()
        allowed += (1.25 ** 2 * 2.0 ** -22 / 3 * (ref.square() + mean) + (2.0 ** -15 * size).square()).sum()
        row += n
    assert square <= allowed, (square / allowed).sqrt()


@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("ends,news", [((70001,), (17,)), ((66000, 5), (12, 5)), ((30, 40000, 41000), (30, 16, 16))], ids=str)
def test_groups_over_all_shares(dec, d, ends, news):
    """One KV head: a group of rows cut into as many shares as there are, alone and behind or before others."""
    _run(dec, ends, news, 3, 1, d, 64, F16, 52, max_len=1 << 24)
