"""decoder.residual_norm with fp32 values, to fp32's own precision. Bounds in units of 2^-24 (half a step of fp32, relative):
the gate's exponential and reciprocal are off by two each, its argument's rest by one, sum and products by one each: 12 are allowed,
and two of the least subnormal number where a result is below the normal range. A sum of squares is off by its additions in a row at
most (squares themselves one more), a root by half of that and three, weights, scale and residual by one each. Needs an MI355X."""

import pytest
import torch

pytestmark = pytest.mark.gpu
F32 = torch.float32
HALF, LEAST = 2.0 ** -24, 2.0 ** -149


@pytest.fixture(scope="module")
def dec():
    from vllm_gguf_plugin import decoder

    assert torch.cuda.is_available(), "GPU tests need an MI355X"
    return decoder


def _act(g, act):
    """In 64 bits; a sigmoid by an exponential that does not overflow."""
    g = g.double()
    t = torch.exp(-g.abs())
    s = torch.where(g < 0, t, torch.ones_like(t)) / (1 + t)
    return g * s if act == "silu" else s


@pytest.mark.parametrize("act", ["sigmoid", "silu"])
@pytest.mark.parametrize("n", [4096, 4097, 70001])
def test_gates(dec, n, act):
    """Gates from -120, where sigmoids are no longer numbers of fp32, to 120."""
    gate = torch.linspace(-120, 120, n)[None].repeat(2, 1)
    gate[1] = torch.linspace(-2, 2, n)
    gate = gate.cuda()
    y = dec.residual_norm(torch.ones_like(gate), gate=gate, act=act)[1].double()
    ref = _act(gate, act)
    bad = (y - ref).abs() > 12 * HALF * ref.abs() + 2 * LEAST
    assert not bad.any(), (int(bad.sum()), gate[bad][:3], y[bad][:3], ref[bad][:3])


def _adds(n):
    """The most additions in a row in a row's sum of squares: the lane's, its wave's, then the parts."""
    if n % 8:
        return (2 if n <= 1024 else 8) + 6 + 16
    return 8 + 6 + max(1, n // 512)


@pytest.mark.parametrize("n", [8, 96, 128, 513, 1000, 4097, 5120, 8192, 16384])
@pytest.mark.parametrize("rows", [3, 1100])
def test_norms(dec, n, rows):
    g = torch.Generator().manual_seed(n)
    x, r, gate = (torch.randn(rows, n, generator=g).cuda() for _ in range(3))
    gate *= 20
    wi, wo = ((1 + 0.3 * torch.randn(n, generator=g)).cuda() for _ in range(2))
    out, h = dec.residual_norm(x, r, wo, inner_weight=wi, gate=gate, act="silu", scale=0.5, eps=1e-5)
    root = _adds(n) / 2 + 1 + 3
    u = x.double()
    u = u / torch.sqrt(u.square().mean(-1, keepdim=True) + 1e-5) * wi.double()
    u = 0.5 * u * _act(gate, "silu")
    off = (root + 2 + 12 + 2) * u.abs() + (r.double() + u).abs()  # of h, in units of HALF
    h2 = r.double() + u
    bad = (h.double() - h2).abs() > HALF * off
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:3])
    mean = h2.square().mean(-1, keepdim=True) + 1e-5
    by = wo.double() / torch.sqrt(mean)
    # the second root's mean takes the errors of the row's values: |2 h dh| on average, half of it in the root
    more = (h2.abs() * off).mean(-1, keepdim=True) / mean
    bad = (out.double() - h2 * by).abs() > HALF * (off * by.abs() + (root + more + 2) * (h2 * by).abs())
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:3])
