"""The decoder operators in CUDA graphs: each one's first call of a fresh process made inside a capture,
and a captured call replayed with other lengths, pages, slots and token ids in its tensors, which
is what a server does. Every replay is compared with an eager call bit for bit. Needs an MI355X."""

import os
import subprocess
import sys

import pytest
from conftest import PKG_ROOT

pytestmark = pytest.mark.gpu

CHILD = r"""
import sys
import torch
sys.path.insert(0, PKG_ROOT)
from vllm_gguf_plugin import decoder as dec  # loads the library and the ops: no GPU call

torch.zeros(1, device="cuda")  # the HIP context
gen = torch.Generator().manual_seed(0)
bf16 = torch.bfloat16


def rand(*shape, dtype=bf16):
    return torch.randn(*shape, generator=gen).to(dtype).cuda()


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def cache(heads, page, d):
    c = dec.Kv8Cache(torch.randint(-127, 128, (40, heads, page, d), generator=gen).to(torch.int8).cuda(),
                     torch.randint(-127, 128, (40, heads, d, page), generator=gen).to(torch.int8).cuda(),
                     torch.rand(40, heads, generator=gen).cuda() / 100, torch.rand(40, heads, generator=gen).cuda() / 100)
    return c, torch.randperm(40, generator=gen).view(4, 10).to(torch.int32).cuda()


def attention(d, page, new, max_len, dtype=bf16):
    c, table = cache(2, page, d)
    q, lens, cu = rand(4 * new, 6, d, dtype=dtype), ints(new, 9 * page, 40, 77), ints(0, new, 2 * new, 3 * new, 4 * new)

    def change():
        lens.copy_(ints(10 * page, new, 0, 100))
        table.copy_(table.flip(1))
        cu.copy_(ints(0, 1, 1, new + 1, 2 * new + 1))
        q.copy_(rand(*q.shape, dtype=dtype))

    rows = lambda: int(cu[-1])  # rows behind the last offset belong to nobody
    return lambda: [dec.kv8_attention(q, c, table, lens, cu, new, max_len)], change, rows


def append():
    c, table = cache(2, 16, 128)
    k, v, lens, cu = rand(12, 2, 128), rand(12, 2, 128), ints(30, 8, 1, 160), ints(0, 3, 4, 5, 12)
    start = [x.clone() for x in c]

    def call():
        for x, y in zip(c, start):
            x.copy_(y)
        dec.kv8_append(c, k, v, table, lens, cu, 9)
        return [*c, *dec.kv8_read(c, table, torch.zeros_like(lens), cu, 12, 9)]

    def change():
        lens.copy_(ints(9, 0, 160, 20))
        cu.copy_(ints(0, 9, 9, 10, 12))
        k.copy_(rand(*k.shape))

    return call, change, None


def delta(dtype, news, steps, dk=128):
    t = sum(news)
    q, k, v = rand(t, 2, dk, dtype=dtype), rand(t, 2, dk, dtype=dtype), rand(t, 4, 64, dtype=dtype)
    g, beta = -rand(t, 4, dtype=torch.float32).abs(), torch.sigmoid(rand(t, 4, dtype=torch.float32))
    first, state = rand(9, 4, 64, dk, dtype=torch.float32), torch.zeros(9, 4, 64, dk, device="cuda")
    slots, cu = ints(0, -1, 2), ints(0, *torch.tensor(news).cumsum(0).tolist())
    out = ints(3, 4, 5, 6, 7, 8).view(3, 2) if steps else ints(3, 4, 5)

    def call():
        state.copy_(first)
        return [dec.gated_delta_rule(q, k, v, g, beta, state, slots, cu, max(news), out_slots=out), state]

    def change():
        slots.copy_(ints(2, 0, -1))
        out.copy_(out.flip(0))
        cu.copy_(ints(0, 1, 1, t))
        v.copy_(rand(*v.shape, dtype=dtype))

    return call, change, None


def logprobs(rows, vocab, top):
    x, ids = rand(rows, vocab), torch.randint(vocab, (rows,), generator=gen).cuda()

    def change():
        x.copy_(rand(rows, vocab))
        ids.copy_(torch.randint(vocab, (rows,), generator=gen).cuda())
        ids[0] = -1

    return lambda: list(dec.token_logprobs(x, ids, top)), change, None


CASES = {
    "append": append(),
    "few rows 256": attention(256, 16, 1, 160), "few rows 64, two tiles": attention(64, 32, 8, 320),
    "few rows 192": attention(192, 16, 1, 1), "few rows 128 fp16": attention(128, 16, 2, 160, torch.float16),
    "many rows 256": attention(256, 64, 30, 640), "many rows 64": attention(64, 16, 40, 160),
    "tokens": delta(bf16, (1, 2, 3), False), "tokens, every state": delta(torch.float16, (1, 2, 3), True, 64),
    "chunks bf16": delta(bf16, (70, 3, 130), False), "chunks fp16": delta(torch.float16, (70, 3, 130), False),
    "chunks fp32": delta(torch.float32, (70, 3, 130), False, 64),
    "logprobs": logprobs(3, 50257, 20), "logprobs, large chunks": logprobs(90, 32000, 3), "logprobs alone": logprobs(2, 9000, 0),
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
