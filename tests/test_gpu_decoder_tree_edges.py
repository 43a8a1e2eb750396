"""Trees without branches are causal attention: the edges of kv8_attention's tests once more through kv8_tree_attention, with masks that are
lower triangles, in its form for few rows and in the one for many. And pools of more than 2^31 codes. Needs an MI355X."""

import math

import pytest
import torch
import test_gpu_decoder_kv8 as causal

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


class _Tree:
    """The decoder module, its attention by lower triangles; `hint`: of max_len, beyond which the form for many rows is taken from 33
    (of heads of 64 from 65) rows a KV head on."""

    def __init__(self, dec, hint):
        self.dec, self.hint = dec, hint

    def __getattr__(self, name):
        return getattr(self.dec, name)

    def kv8_attention(self, query, cache, table, lens, cu, max_new, max_len, scale=None):
        words = max(1, -(-max_new // 64)) if max_new < 1 << 20 else -(-query.shape[0] // 64)
        starts = cu.long()
        rows = torch.arange(query.shape[0], device="cuda")
        seq = torch.searchsorted(starts, rows, right=True) - 1
        at = rows - starts[seq.clamp(0, len(starts) - 1)]
        bits = (at[:, None] + 1 - 64 * torch.arange(words, device="cuda")).clamp(0, 64)
        one = torch.ones_like(bits)
        mask = torch.where(bits == 64, -one, (one << bits.clamp(max=63)) - 1)
        return self.dec.kv8_tree_attention(query, cache, mask, table, lens, cu, max_new, self.hint or max_len, scale)


@pytest.fixture(params=[None, 1 << 24], ids=["few", "many"])
def tree(request):
    from vllm_gguf_plugin import decoder
    return _Tree(decoder, request.param)


@pytest.mark.parametrize("news", [(4, 3), (100, 3)], ids=str)
def test_pages_out_of_range_and_not_finite(tree, news):
    causal.test_attention_pages_out_of_range_and_not_finite(tree, news)


def test_extreme_scales_and_strides(tree):
    causal.test_attention_extreme_scales(tree)
    causal.test_attention_strided_query_other_stream_and_graph(tree)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
@pytest.mark.parametrize("news", [(2, 9), (2, 150)], ids=str)
def test_negative_scale(tree, dtype, news):
    causal.test_attention_negative_scale(tree, dtype, news)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
@pytest.mark.parametrize("hq,heads,d", [(6, 2, 128), (6, 1, 256), (3, 1, 192), (6, 2, 64)])
@pytest.mark.parametrize("news", [3, 8, 70])
def test_large_v_scale_unseen(tree, news, hq, heads, d, dtype):
    causal.test_attention_large_v_scale_unseen(tree, news, hq, heads, d, dtype)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
@pytest.mark.parametrize("news", [1, 70])
def test_many_small_weights(tree, news, dtype):
    causal.test_attention_many_small_weights(tree, news, dtype)


@pytest.mark.parametrize("news", [2, 70])
def test_v_scales_below_the_least_and_queries_at_the_end_of_the_range(tree, news):
    causal.test_attention_v_scales_below_the_least(tree, news)
    causal.test_attention_queries_at_the_end_of_the_range(tree, news + 1)


@pytest.mark.parametrize("news", [1, 70])
@pytest.mark.parametrize("log_k_scale", [10, 43])
def test_scores_far_from_zero(tree, news, log_k_scale):
    """Scores whose rounding is far more than the range of a weight, and scores below -1e30."""
    causal._far_scores(tree, news, log_k_scale)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
@pytest.mark.parametrize("news", [3, 70])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_queries_that_are_not_finite(tree, bad, news, dtype):
    causal.test_attention_queries_that_are_not_finite(tree, bad, news, dtype)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
@pytest.mark.parametrize("news", [3, 70])
def test_queries_with_a_strong_element(tree, news, dtype):
    causal.test_attention_queries_with_a_strong_element(tree, news, dtype)


@pytest.mark.parametrize("hq,heads,d,page", [(6, 1, 256, 64), (4, 2, 128, 16), (2, 2, 64, 144), (2, 1, 192, 32)])
@pytest.mark.parametrize("news", [3, 70])
@pytest.mark.parametrize("end", [4095, 8200])
def test_past_a_segment(tree, end, news, hq, heads, d, page):
    causal.test_attention_past_a_segment(tree, end, news, hq, heads, d, page)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
@pytest.mark.parametrize("hq,heads,d,page", [(6, 1, 256, 16), (8, 2, 128, 32), (4, 4, 64, 144), (5, 1, 192, 64)])
@pytest.mark.parametrize("news", [(1, 1, 1, 1), (5, 40, 2, 17), (1, 65, 200, 130)], ids=str)
def test_gives_numbers(tree, news, hq, heads, d, page, dtype):
    causal.test_attention_gives_numbers(tree, news, hq, heads, d, page, dtype)


def test_many_short_sequences(tree):
    causal.test_attention_of_many_short_sequences(tree)


@pytest.mark.parametrize("d,page", [(256, 256), (128, 64)])
def test_offsets_past_32_bits(d, page):
    """A pool of more than 2^31 codes, the sequence in its last pages: rotated (by nothing) into them, attended in both forms, a path kept
    and read back."""
    from vllm_gguf_plugin import decoder as dec
    pages = 2 ** 31 // (page * d) + 9
    cache = dec.Kv8Cache.empty(pages, 1, page, d)
    need = -(-700 // page)
    table = (pages - 1 - torch.arange(need)).to(torch.int32).cuda()[None]
    g = torch.Generator().manual_seed(41)
    n, drafts = 700, 40
    k, v = (torch.randn(n, 1, d, generator=g).to(BF16).cuda() for _ in range(2))
    cos_sin = torch.cat([torch.ones(1, 8), torch.zeros(1, 8)], 1).cuda()
    q = (torch.randn(n, 3, d, generator=g) * 0.3).to(BF16).cuda()
    y = dec.kv8_rotary_append(cache, q, k, v, cos_sin, torch.zeros(n, dtype=torch.int64, device="cuda"), table, causal._i32(n), causal._cu((n,)), n)
    assert torch.equal(y, q)
    kr, vr = dec.kv8_read(cache, table, causal._i32(0), causal._cu((n,)), n, n, torch.float32)
    for x, z in ((k, kr), (v, vr)):  # half a step of at most amax / 127
        assert (x.float() - z).abs().max() <= x.abs().max().float() / 127 * 0.5001
    ref, most = causal._attention_ref(q[-drafts:], cache, table, (n,), (drafts,), d ** -0.5)
    for hint in (None, 1 << 24):
        y = _Tree(dec, hint).kv8_attention(q[-drafts:].contiguous(), cache, table, causal._i32(n), causal._cu((drafts,)), drafts, n)
        causal._near(y, ref, most)
    path = torch.tensor([[1, 5, 39, -1]], dtype=torch.int32, device="cuda")
    dec.kv8_keep(cache, path, table, causal._i32(n), causal._cu((drafts,)))
    base = n - drafts
    kk, vv = dec.kv8_read(cache, table, causal._i32(base), causal._cu((3,)), 3, 3, torch.float32)
    for x, z in ((kr, kk), (vr, vv)):  # moved as they are, or rounded once more to another page's scale, which may grow to theirs
        assert (x[[base + 1, base + 5, base + 39]] - z).abs().max() <= x.abs().max() / 127 * 0.5001
    assert not cache.k_scale[:pages - need].any() and not cache.k[:4].any()
