"""The operators of a decoder's block (rotation into the cache, attention for trees, keeping a path, block norms) in CUDA graphs: each
one's first call of a fresh process made inside a capture, and a captured call replayed with other lengths, pages, masks, paths and
positions in its tensors. Every replay is compared with an eager call bit for bit. Calls on several streams at once,
and C calls with a workspace that does not do. Needs an MI355X."""

import ctypes
import os
import subprocess
import sys

import pytest
import torch
from conftest import PKG_ROOT

pytestmark = pytest.mark.gpu

CHILD = r"""
import sys
import torch
sys.path.insert(0, PKG_ROOT)
from vllm_gguf_plugin import decoder as dec  # loads the library and the ops: no GPU call

torch.zeros(1, device="cuda")  # the HIP context
gen = torch.Generator().manual_seed(0)
bf16, f16 = torch.bfloat16, torch.float16


def rand(*shape, dtype=bf16):
    return torch.randn(*shape, generator=gen).to(dtype).cuda()


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def bits(*shape):
    return torch.randint(-2 ** 63, 2 ** 63 - 1, shape, generator=gen).cuda()


def cache(heads, page, d):
    c = dec.Kv8Cache(torch.randint(-127, 128, (40, heads, page, d), generator=gen).to(torch.int8).cuda(),
                     torch.randint(-127, 128, (40, heads, d, page), generator=gen).to(torch.int8).cuda(),
                     torch.rand(40, heads, generator=gen).cuda() / 100, torch.rand(40, heads, generator=gen).cuda() / 100)
    return c, torch.randperm(40, generator=gen).view(4, 10).to(torch.int32).cuda()


def tree(d, page, new, max_len, dtype=bf16):
    c, table = cache(2, page, d)
    q, mask, lens, cu = rand(4 * new, 6, d, dtype=dtype), bits(4 * new, 1), ints(new, 9 * page, 40, 77), ints(0, new, 2 * new, 3 * new, 4 * new)

    def change():
        lens.copy_(ints(10 * page, new, 0, 100))
        table.copy_(table.flip(1))
        cu.copy_(ints(0, 1, 1, new + 1, 2 * new + 1))
        q.copy_(rand(*q.shape, dtype=dtype))
        mask.copy_(bits(*mask.shape))

    rows = lambda: int(cu[-1])  # rows behind the last offset belong to nobody
    return lambda: [dec.kv8_tree_attention(q, c, mask, table, lens, cu, new, max_len)], change, rows


def rotary(d, dtype, pairs, norms):
    c, table = cache(2, 16, d)
    qkv, lens, cu = rand(12, 10, d, dtype=dtype), ints(30, 8, 1, 160), ints(0, 3, 4, 5, 12)
    cs, at = rand(200, d // 2, dtype=torch.float32), torch.randint(200, (12,), generator=gen).cuda()
    w = rand(d, dtype=torch.float32) if norms else None
    start = [x.clone() for x in c]

    def call():
        for x, y in zip(c, start):
            x.copy_(y)
        return [dec.kv8_rotary_append(c, qkv[:, :6], qkv[:, 6:8], qkv[:, 8:], cs, at, table, lens, cu, 9, pairs, w, w), *c]

    def change():
        lens.copy_(ints(9, 0, 160, 20))
        cu.copy_(ints(0, 9, 9, 10, 12))
        at.copy_(at.flip(0))
        at[0] = 777
        qkv.copy_(rand(*qkv.shape, dtype=dtype))

    return call, change, None


def keep(d, page):
    c, table = cache(2, page, d)
    lens, cu = ints(40, 8, 0, 10 * page), ints(0, 12, 20, 20, 40)
    path = ints(0, 2, 5, 11, 1, 2, 3, -1, -1, 0, 0, 0, 7, 9, 18, 19).view(4, 4)
    start = [x.clone() for x in c]

    def call():
        for x, y in zip(c, start):
            x.copy_(y)
        dec.kv8_keep(c, path, table, lens, cu)
        return [*c]

    def change():
        path.copy_(path.flip(0))
        lens.copy_(ints(13, 9, 50, 33))
        cu.copy_(ints(0, 12, 12, 20, 39))

    return call, change, None


def norm(rows, n, dtype, **kw):
    x, r, g, w = rand(rows, n, dtype=dtype), rand(rows, n, dtype=torch.float32), rand(rows, n, dtype=dtype), rand(n, dtype=torch.float32)
    change = lambda: (x.copy_(rand(rows, n, dtype=dtype)), w.copy_(rand(n, dtype=torch.float32)))
    return lambda: list(dec.residual_norm(x, r, w, inner_weight=w, gate=g, act="silu")), change, None


CASES = {
    "rotary 256": rotary(256, bf16, False, True), "rotary 64, pairs": rotary(64, f16, True, False),
    "rotary 128": rotary(128, torch.float32, False, True),
    "few rows 256": tree(256, 16, 2, 160), "few rows 64": tree(64, 32, 8, 320), "few rows 192": tree(192, 16, 1, 1, f16),
    "many rows 256": tree(256, 64, 30, 1 << 24), "many rows 256, two groups": tree(256, 16, 20, 1 << 24, f16),
    "many rows 192": tree(192, 16, 40, 1 << 24), "many rows 128": tree(128, 64, 30, 1 << 24), "many rows 64": tree(64, 16, 40, 1 << 24),
    "keep 64": keep(64, 16), "keep 256": keep(256, 64),
    "norm": norm(3, 5120, bf16), "norm, many": norm(1100, 8192, f16), "norm, short": norm(70, 96, bf16), "norm, odd": norm(5, 1001, f16),
}
fails = []
for name, (call, change, rows) in CASES.items():
    print("case", name, flush=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for turn in range(3):
        if turn == 1:
            change()
        graph.replay()
        torch.cuda.synchronize()
        seen = [x.clone() for x in got]
        eager = call()
        torch.cuda.synchronize()
        n = rows() if rows else None
        if not all(torch.equal(a[:n].nan_to_num(7), b[:n].nan_to_num(7)) for a, b in zip(seen, eager)):
            fails.append((name, turn))
print("FAILS", fails, flush=True)
"""


def test_first_calls_and_changed_replays():
    p = subprocess.run([sys.executable, "-u", "-c", f"PKG_ROOT = {PKG_ROOT!r}\n" + CHILD], capture_output=True, text=True,
                       timeout=100, env=dict(os.environ))
    print(p.stdout[-3000:])
    assert p.returncode == 0, p.stdout[-1500:] + p.stderr[-3000:]
    assert "FAILS []" in p.stdout, p.stdout[-2000:]


def _tree_call(d, seed, new=40, page=64):
    g = torch.Generator().manual_seed(seed)
    from vllm_gguf_plugin import decoder as dec
    c = dec.Kv8Cache(torch.randint(-127, 128, (64, 2, page, d), generator=g).to(torch.int8).cuda(),
                     torch.randint(-127, 128, (64, 2, d, page), generator=g).to(torch.int8).cuda(),
                     torch.rand(64, 2, generator=g).cuda() / 100, torch.rand(64, 2, generator=g).cuda() / 100)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    q = torch.randn(2 * new, 12, d, generator=g).bfloat16().cuda()
    mask = torch.randint(-2 ** 63, 2 ** 63 - 1, (2 * new, 1), generator=g).cuda()
    table, lens, cu = torch.arange(64, dtype=torch.int32).view(2, 32).cuda(), i32(2000, 1234), i32(0, new, 2 * new)
    return lambda hint: dec.kv8_tree_attention(q, c, mask, table, lens, cu, new, hint)


@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("hint", [2000, 1 << 24])
def test_calls_on_two_streams_at_once(d, hint):
    """Calls in flight beside each other, on streams of their own and in two graphs of one pool: each has the workspace for itself."""
    calls = [_tree_call(d, s) for s in range(2)]
    want = [c(hint) for c in calls]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in calls], [[], []]
    for _ in range(4):
        for c, s, out in zip(calls, streams, got):
            with torch.cuda.stream(s):
                out.append(c(hint))
    torch.cuda.synchronize()
    assert all(torch.equal(y, w) for out, w in zip(got, want) for y in out)

    graphs, outs = [], []
    for c in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            outs.append(c(hint))
        graphs.append(g)
    for _ in range(3):
        for g, out, w in zip(graphs, outs, want):
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, w)
            calls[0](hint)


@pytest.mark.parametrize("d,q_heads,tokens", [(64, 4, 3), (256, 8, 50), (192, 64, 100)])
def test_workspaces_that_do_not_do_are_refused(d, q_heads, tokens):
    from test_decoder_api import _CacheT, _desc
    from vllm_gguf_plugin import decoder as dec
    lib = ctypes.CDLL(dec.LIB_PATH)
    lib.gguf_kv8_tree_attention_workspace_bytes.restype = ctypes.c_size_t
    lib.gguf_decoder_last_error.restype = ctypes.c_char_p
    i64, P = ctypes.c_int64, ctypes.byref

    def on(t):
        r = _desc(t)
        r.device = 0
        return r

    query, cache = torch.zeros(tokens, q_heads, d, dtype=torch.float16, device="cuda"), _CacheT(*map(on, dec.Kv8Cache.empty(4, 2, 16, d)))
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    keep = [query, torch.zeros(tokens, 2, dtype=torch.int64, device="cuda"), ints([[0, 1], [2, 3]]), ints([5, 6]), ints([0, 1, 3])]
    q, mask, table, lens, cu = map(on, keep)
    need = lib.gguf_kv8_tree_attention_workspace_bytes(P(cache), P(q), i64(2), i64(tokens), i64(2 ** 30))
    assert need > 0
    ws = torch.zeros(need + 32, dtype=torch.uint8, device="cuda")
    for data, size in ((ws.data_ptr(), need - 1), (ws.data_ptr() + 1, need), (None, 0), (None, need)):
        assert lib.gguf_kv8_tree_attention(P(q), P(cache), P(mask), P(table), P(lens), P(cu), i64(tokens), i64(2 ** 30), ctypes.c_float(1),
                                           P(q), ctypes.c_void_p(data), ctypes.c_size_t(size), ctypes.c_void_p(None)) == 1
        assert "workspace" in lib.gguf_decoder_last_error().decode(), (data, size, lib.gguf_decoder_last_error())
