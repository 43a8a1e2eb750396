"""fp16 queries of decoder.kv8_tree_attention keep all their bits, in its form for few rows and in the one for many: rows whose largest
element meets keys of zero while the others, 2^15 below it, decide the scores in their last bits; and rows of subnormal elements.

Bound: that of test_gpu_decoder_tree.py, |y - ref| <= 2^-11 |ref| + 2^-10 max |v|. Elements rounded to 2^-10 of themselves would move the
scores of the first test by up to a quarter, and outputs by some tenth of max |v|. Needs an MI355X."""

import pytest
import torch

from _gpu import poison_allocator
from test_gpu_decoder_kv8 import _close, _cu, _i32, _random_cache, _table
from test_gpu_decoder_tree import HINTS, _random_mask, _tree_ref

pytestmark = pytest.mark.gpu
F16 = torch.float16


@pytest.fixture(scope="module")
def dec():
    from vllm_gguf_plugin import decoder

    assert torch.cuda.is_available(), "GPU tests need an MI355X"
    return decoder


def _check(dec, cache, q, ends, news, page, scale, hint, g):
    table = _table(ends, page, cache.k.shape[0], g)
    mask = _random_mask(sum(news), 1, g).cuda()
    poison_allocator()
    y = dec.kv8_tree_attention(q, cache, mask, table, _i32(*ends), _cu(news), max(news), hint or max(ends), scale)
    ref, most = _tree_ref(q, cache, table, mask, ends, news, scale)
    _close(y, ref, most)


@pytest.mark.parametrize("hint", HINTS)
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("d", [64, 128, 192, 256])
def test_elements_far_below_the_rows_largest(dec, d, sign, hint):
    g = torch.Generator().manual_seed(41)
    ends, news, page = (300, 90), (40, 33), 16
    cache = _random_cache(dec, 30, 1, page, d, g)
    a = torch.randint(-127, 128, (30, 1, page), generator=g)
    cache.k.zero_()
    cache.k[..., 1], cache.k[..., d - 1] = a.cuda().to(torch.int8), (-a).cuda().to(torch.int8)
    cache.k_scale.fill_(2.0)
    cache.v.copy_((a.sign()[:, :, None] * torch.randint(64, 128, (30, 1, d, page), generator=g)).to(torch.int8))
    q = 1 + torch.randint(0, 1024, (sum(news), 2, d), generator=g) / 1024
    q[..., 0] = 2.0 ** 15
    q[..., 1], q[..., d - 1] = 1 + torch.randint(1, 16, q.shape[:2], generator=g) / 1024, 1.0
    _check(dec, cache, q.to(F16).cuda(), ends, news, page, sign * 1.0, hint, g)


@pytest.mark.parametrize("hint", HINTS)
@pytest.mark.parametrize("d", [64, 128, 192, 256])
def test_subnormal_elements(dec, d, hint):
    g = torch.Generator().manual_seed(42)
    ends, news, page = (300, 90), (40, 33), 16
    cache = _random_cache(dec, 30, 1, page, d, g)
    cache.k_scale.fill_(2.0 ** -14)
    q = torch.randint(-1023, 1024, (sum(news), 2, d), generator=g) * 2.0 ** -24
    _check(dec, cache, q.to(F16).cuda(), ends, news, page, 2.0 ** 20, hint, g)
