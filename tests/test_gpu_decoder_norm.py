"""Block norms with gate and residual (decoder.residual_norm, decoder.gated_norm) against their formula in 64 bits.

Bound: fp32 sums of squares, at most 400 terms a lane and some 20 steps, are off by 2^-15.5 relative, their root by half; root, sigmoid
(an exponential of an argument rounded to 2^-24 of up to 88), weights and products add less than 2^-17. So u and the second norm's factor
are known to 2^-15, and h to 2^-15 (|residual| + |scale u|); each output is rounded once more, by eps / 2 of itself.
Needs an MI355X."""

import itertools

import pytest
import torch

from _gpu import graph_replays_equal, poison_allocator

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def dec():
    from vllm_gguf_plugin import decoder

    assert torch.cuda.is_available(), "GPU tests need an MI355X"
    return decoder


def _ref(x, residual, weight, inner, gate, act, scale, eps):
    """(out, what it may be off by before its rounding, h, likewise)"""
    u = x.double()
    n = u.shape[-1]
    if inner is not None:
        u = u / torch.sqrt(u.square().sum(-1, keepdim=True) / n + eps) * inner.double()
    if gate is not None:
        g = gate.double()
        u = u * {"none": g, "sigmoid": torch.sigmoid(g), "silu": g * torch.sigmoid(g)}[act]
    u = scale * u
    r = residual.double() if residual is not None else torch.zeros_like(u)
    h, size = r + u, r.abs() + u.abs()
    if weight is None:
        return None, None, h, 2.0 ** -15 * size
    by = weight.double() / torch.sqrt(h.square().sum(-1, keepdim=True) / n + eps)
    return h * by, 2.0 ** -15 * (size * by.abs() + (h * by).abs()), h, 2.0 ** -15 * size


def _check(y, ref, off):
    bad = (y.double() - ref).abs() > torch.finfo(y.dtype).eps / 2 * ref.abs() + off + torch.finfo(y.dtype).smallest_normal * torch.finfo(y.dtype).eps
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:3], y[bad][:3], ref[bad][:3])


def _run(dec, shape, dtype, rdtype, seed, inner, outer, act, residual, scale=1.0, eps=1e-6, view=lambda x: x):
    g = torch.Generator().manual_seed(seed)
    n = shape[-1]

    def rand(dt, by=1.0):
        x = torch.randn(*shape, generator=g) * torch.exp(torch.randn(*shape[:-1], 1, generator=g)) * by
        return view(x.to(dt).cuda())

    x, r = rand(dtype), rand(rdtype, 3.0) if residual else None
    gate = rand(dtype) if act else None
    wi, wo = ((1 + 0.3 * torch.randn(n, generator=g)).cuda() if w else None for w in (inner, outer))
    poison_allocator()
    out, h = dec.residual_norm(x, r, wo, inner_weight=wi, gate=gate, act=act or "none", scale=scale, eps=eps)
    ro, oo, rh, oh = _ref(x, r, wo, wi, gate, act, scale, eps)
    assert h.shape == x.shape and h.dtype == (rdtype if residual else dtype) and h.is_contiguous()
    _check(h, rh, oh)
    assert (out is None) == (not outer)
    if outer:
        assert out.shape == x.shape and out.dtype == dtype and out.is_contiguous()
        _check(out, ro, oo)
    return out, h


SIZES = [1, 7, 8, 64, 96, 128, 192, 256, 511, 512, 520, 1000, 1024, 4096, 4097, 5120, 8192, 8200, 16384, 20000, 32768, 32776, 65536, 70000]


@pytest.mark.parametrize("dtype,rdtype", [(BF16, BF16), (F16, F32), (F32, F32)], ids=str)
@pytest.mark.parametrize("n", SIZES)
def test_sizes(dec, n, dtype, rdtype):
    """From one value to rows beyond the registers, odd ones; one row and some, all parts at once."""
    for rows in (1, 5):
        _run(dec, (rows, n), dtype, rdtype, n, True, True, "silu", True, 0.5)


@pytest.mark.parametrize("n", [128, 5120, 513])
@pytest.mark.parametrize("inner,outer,act,residual", itertools.product([False, True], [False, True], [None, "none", "sigmoid", "silu"], [False, True]))
def test_parts(dec, n, inner, outer, act, residual):
    """Every part there or missing."""
    for dtype, rdtype in ((BF16, F32), (F16, F16)):
        _run(dec, (3, n), dtype, rdtype, 1, inner, outer, act, residual, 0.22, 1e-5)


@pytest.mark.parametrize("shape", [(7, 48, 128), (3, 5, 64), (2, 3, 100), (5, 1, 1024), (4, 2, 5120)], ids=str)
@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
def test_heads(dec, shape, dtype):
    """[rows, heads, n], contiguous and as views of a wider projection, some off the 16-byte grid."""
    _run(dec, shape, dtype, dtype, 2, True, False, "silu", False)
    for lead, more in ((8, 8), (8, 3), (3, 0)):
        wide = lambda x: torch.cat([x[..., :1].expand(*x.shape[:-1], lead), x, x[..., :1].expand(*x.shape[:-1], more)], -1)[..., lead:lead + x.shape[-1]]  # noqa: E731
        _run(dec, shape, dtype, dtype, 3, True, True, "sigmoid", True, view=wide)
    _run(dec, shape, dtype, dtype, 4, True, False, "silu", False, view=lambda x: x.transpose(0, 1).contiguous().transpose(0, 1))


def test_many_rows(dec):
    """More rows than workgroups at a time; rows are independent: a part of a batch gives the batch's bits."""
    for shape in ((3001, 128), (70000, 64), (513, 5120), (2049, 1000)):
        out, h = _run(dec, shape, BF16, BF16, 5, True, True, None, True)
        g = torch.Generator().manual_seed(6)
        x, r, w = torch.randn(*shape, generator=g).bfloat16().cuda(), torch.randn(*shape, generator=g).cuda(), torch.randn(shape[1], generator=g).cuda()
        a, b = dec.residual_norm(x, r, w, inner_weight=w)
        for lo, hi in ((0, 1), (3, 17), (shape[0] - 1, shape[0])):
            c, d = dec.residual_norm(x[lo:hi], r[lo:hi], w, inner_weight=w)
            assert torch.equal(c, a[lo:hi]) and torch.equal(d, b[lo:hi])


@pytest.mark.parametrize("n", [4096, 4104, 5120, 8192, 12296, 16384, 20000])
def test_many_long_rows(dec, n):
    """Rows of many a workgroup's pieces, alone and among more than a thousand: the same bits."""
    g = torch.Generator().manual_seed(8)
    x, r, w = torch.randn(1100, n, generator=g).bfloat16().cuda(), torch.randn(1100, n, generator=g).bfloat16().cuda(), torch.randn(n, generator=g).cuda()
    kw = dict(inner_weight=w, act="silu", scale=0.7)
    a, b = dec.residual_norm(x, r, w, gate=r, **kw)
    for lo, hi in ((0, 1), (511, 540), (1099, 1100)):
        c, d = dec.residual_norm(x[lo:hi], r[lo:hi], w, gate=r[lo:hi], **kw)
        assert torch.equal(c, a[lo:hi]) and torch.equal(d, b[lo:hi])
    _run(dec, (1030, n), BF16, F32, 9, True, True, "sigmoid", True, 0.5)


@pytest.mark.parametrize("dtype,rdtype", [(BF16, F32), (F16, F16), (F32, F32)], ids=str)
@pytest.mark.parametrize("n", [63, 65, 127, 1023, 1025, 4095, 8191, 8193])
def test_odd_lengths(dec, n, dtype, rdtype):
    """Rows of single values, a workgroup each, around what its threads hold; a part of a batch gives the batch's bits."""
    _run(dec, (3, n), dtype, rdtype, 10, True, True, "silu", True, 0.5)
    _run(dec, (2, 3, n), dtype, dtype, 11, True, False, "sigmoid", False)
    g = torch.Generator().manual_seed(12)
    x, r, w = torch.randn(300, n, generator=g).to(dtype).cuda(), torch.randn(300, n, generator=g).to(rdtype).cuda(), torch.randn(n, generator=g).cuda()
    a, b = dec.residual_norm(x, r, w, inner_weight=w)
    for lo, hi in ((0, 1), (100, 117), (299, 300)):
        c, d = dec.residual_norm(x[lo:hi], r[lo:hi], w, inner_weight=w)
        assert torch.equal(c, a[lo:hi]) and torch.equal(d, b[lo:hi])


def test_broadcast_gate_and_residual(dec):
    """Strides of 0: one gate, one residual row for all rows."""
    g = torch.Generator().manual_seed(7)
    x, gate, r = torch.randn(9, 640, generator=g).bfloat16().cuda(), torch.randn(1, 640, generator=g).bfloat16().cuda(), torch.randn(1, 640, generator=g).cuda()
    w = torch.ones(640, device="cuda")
    a = dec.residual_norm(x, r.expand(9, -1), w, gate=gate.expand(9, -1), act="sigmoid")
    b = dec.residual_norm(x, r.repeat(9, 1), w, gate=gate.repeat(9, 1), act="sigmoid")
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_zeros_no_rows_and_values_that_are_not_finite(dec):
    x, w = torch.zeros(4, 1024, dtype=BF16, device="cuda"), torch.ones(1024, device="cuda")
    out, h = dec.residual_norm(x, x, w, inner_weight=w, gate=x, act="silu")
    assert (out == 0).all() and (h == 0).all()
    out, h = dec.residual_norm(x[:0], x[:0], w)
    assert out.shape == h.shape == (0, 1024)
    x[1, 5], x[2, 6] = float("inf"), float("nan")
    out, h = dec.residual_norm(x, None, w)
    assert (out[[0, 3]] == 0).all() and torch.isnan(out[1, 5]) and torch.isnan(out[2]).all() and (out[1, :5] == 0).all()
    # a sigmoid's ends
    gate = torch.tensor([[-1e4, 1e4, float("-inf"), float("inf"), -100.0, 100.0, 0.0, -0.0]], device="cuda")
    one = torch.ones_like(gate)
    s = dec.residual_norm(one, gate=gate, act="sigmoid")[1]
    assert s.tolist() == [[0.0, 1.0, 0.0, 1.0, s[0, 4].item(), 1.0, 0.5, 0.5]] and 0 <= s[0, 4] < 1e-40
    s = dec.residual_norm(one, gate=gate[:, [0, 1, 3, 4, 5, 6, 7, 7]].contiguous(), act="silu")[1]
    assert s[0, 0] == 0 and s[0, 1] == 1e4 and s[0, 2] == float("inf") and s[0, 4] == 100 and (s[0, 5:] == 0).all()


def test_another_stream_and_replays(dec):
    g = torch.Generator().manual_seed(8)
    x, r, w = torch.randn(50, 5120, generator=g).bfloat16().cuda(), torch.randn(50, 5120, generator=g).cuda(), torch.ones(5120, device="cuda")
    torch.cuda.synchronize()
    y = dec.residual_norm(x, r, w, inner_weight=w, gate=x, act="silu")[0]
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        z = dec.residual_norm(x, r, w, inner_weight=w, gate=x, act="silu")[0]
    s.synchronize()
    assert torch.equal(y, z)
    graph_replays_equal(lambda: dec.residual_norm(x, r, w, inner_weight=w, gate=x, act="silu")[0], y)
