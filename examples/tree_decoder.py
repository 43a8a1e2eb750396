"""A small decoder that verifies trees of drafts, over this framework's operators: GGUF linear layers (Q4_K weights), heads that are
normed and turned by their positions on the way into the 8-bit paged KV cache, attention for trees, gated head norms, norms
before and after each block, and the accepted path kept in the cache.

    python examples/tree_decoder.py [--layers 2] [--prompt 300] [--steps 4] [--depth 3]

Two sequences of different lengths read their prompts as a chain of rows (a tree without branches). Then a step runs, for
each sequence, its next token and two branches of drafts behind it at once; the rows' best tokens say which path is kept, its
keys and values move together in the cache, and the next step goes on behind it. One branch is random, the other holds the tokens that
the model itself has said in a first run (as a lookup in earlier answers would), so that some are kept. Weights are random: the text
means nothing. Needs an MI355X.
"""

import argparse
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "vllm-gsqrco-exl3_amd"))

from vllm_gguf_plugin import decoder, ops  # noqa: E402,F401

Q4_K, BLOCK = 12, 144  # ggml type id, bytes of 256 values
HIDDEN, INNER, VOCAB = 1024, 2048, 4096
HQ, HKV, D, TURN, PAGE = 8, 2, 128, 64, 64  # query heads, KV heads, head size, dims that turn, tokens of a page
POSITIONS = 4096


class Linear:
    """Y = X W^T for a random Q4_K weight: the decode op up to 8 rows, the product op beyond."""

    def __init__(self, n, k, gen):
        w = torch.randint(0, 256, (n, k // 256, BLOCK), dtype=torch.uint8, generator=gen)
        scale = torch.tensor([2.6e-4 * (1024 / k) ** 0.5, 1.8e-3 * (1024 / k) ** 0.5], dtype=torch.float16)
        w[..., :4] = scale.view(torch.uint8)
        self.w, self.n = w.reshape(n, -1).cuda(), n

    def __call__(self, x):
        if x.shape[0] <= 8:
            return torch.ops._C_gguf.lcpp_mul_mat_vec_q(self.w, x, Q4_K, self.n)
        return torch.ops._C_gguf.lcpp_mul_mat_q(self.w, x, Q4_K, self.n)


class Step:
    """The ragged batch of one step: a tree of rows a sequence (their parents), behind `lens` older tokens."""

    def __init__(self, trees, lens, table):
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        news = [len(t) for t in trees]
        self.cu, self.ends, self.table = i32([0] + list(torch.tensor(news).cumsum(0))), i32([n + m for n, m in zip(lens, news)]), table
        self.max_new, self.max_len = max(news), max(n + m for n, m in zip(lens, news))
        self.mask = decoder.tree_mask(trees).cuda()
        at = []
        for tree, n in zip(trees, lens):
            depth = []
            for p in tree:
                depth.append(depth[p] + 1 if p >= 0 else n)
            at += depth
        self.positions = torch.tensor(at, device="cuda")


class Layer:
    def __init__(self, gen, pages):
        self.qkv, self.out = Linear((2 * HQ + 2 * HKV) * D, HIDDEN, gen), Linear(HIDDEN, HQ * D, gen)
        self.up, self.down = Linear(2 * INNER, HIDDEN, gen), Linear(HIDDEN, INNER, gen)
        weight = lambda n: (1 + 0.1 * torch.randn(n, generator=gen)).cuda()  # noqa: E731
        self.q_weight, self.k_weight, self.o_weight = weight(D), weight(D), weight(D)
        self.before, self.between, self.after_attention, self.after_mlp = (weight(HIDDEN) for _ in range(4))
        self.cache = decoder.Kv8Cache.empty(pages, HKV, PAGE, D)

    def attention(self, x, s, cos_sin):
        q, gate, k, v = self.qkv(x).view(-1, 2 * HQ + 2 * HKV, D).split((HQ, HQ, HKV, HKV), 1)
        q = decoder.kv8_rotary_append(self.cache, q, k, v, cos_sin, s.positions, s.table, s.ends, s.cu, s.max_new,
                                      q_weight=self.q_weight, k_weight=self.k_weight)
        o = decoder.kv8_tree_attention(q, self.cache, s.mask, s.table, s.ends, s.cu, s.max_new, s.max_len)
        return self.out(decoder.gated_norm(o, gate, self.o_weight).view(-1, HQ * D))

    def mlp(self, x):
        gate, up = self.up(x).chunk(2, -1)
        return self.down(torch.nn.functional.silu(gate) * up)


class Model:
    def __init__(self, layers, pages, seed=0):
        gen = torch.Generator().manual_seed(seed)
        self.embed = torch.randn(VOCAB, HIDDEN, generator=gen).to(torch.bfloat16).cuda()
        self.layers = [Layer(gen, pages) for _ in range(layers)]
        self.head, self.last = Linear(VOCAB, HIDDEN, gen), (1 + 0.1 * torch.randn(HIDDEN, generator=gen)).cuda()
        turn = torch.arange(POSITIONS)[:, None] * 10000.0 ** (-torch.arange(TURN // 2) / (TURN // 2))
        self.cos_sin = torch.cat([turn.cos(), turn.sin()], -1).float().cuda()

    def __call__(self, tokens, s):
        x, h = decoder.residual_norm(self.embed[tokens], weight=self.layers[0].before)
        for i, layer in enumerate(self.layers):
            y = layer.attention(x, s, self.cos_sin)
            x, h = decoder.residual_norm(y, h, layer.between, inner_weight=layer.after_attention)
            y = layer.mlp(x)
            following = self.layers[i + 1].before if i + 1 < len(self.layers) else self.last
            x, h = decoder.residual_norm(y, h, following, inner_weight=layer.after_mlp)
        return self.head(x)

    def keep(self, path, s):
        for layer in self.layers:
            decoder.kv8_keep(layer.cache, path, s.table, s.ends, s.cu)


def follow(tree, rows, best):
    """The accepted rows: from the root on the child that holds its parent's best token."""
    path = [0]
    while True:
        nxt = [i for i, p in enumerate(tree) if p == path[-1] and rows[i] == best[path[-1]]]
        if not nxt:
            return path
        path.append(nxt[0])


def generate(layers=2, prompts=(300, 117), steps=4, depth=3, seed=0, known=None):
    """Returns the sequences' texts (the last token of each not yet read), how many rows each step kept, and the last step's logits of
    the sequences' last kept rows. known: texts that the drafts are looked up in."""
    n = len(prompts)
    gen = torch.Generator().manual_seed(seed + 1)
    texts = [torch.randint(VOCAB, (p,), generator=gen).tolist() for p in prompts]
    pages = -(-(max(prompts) + steps * (depth + 1) + 2 * depth + 1) // PAGE)
    model = Model(layers, n * pages, seed)
    table = torch.randperm(n * pages, generator=gen).view(n, pages).to(torch.int32).cuda()

    trees = [[i - 1 for i in range(p)] for p in prompts]
    logits = model(torch.tensor(sum(texts, []), device="cuda"), Step(trees, [0] * n, table))
    logits = logits[torch.tensor(prompts).cumsum(0).cuda() - 1]
    lens, kept = list(prompts), []
    for s, t in enumerate(logits.argmax(-1).tolist()):
        texts[s].append(t)
    tree = [-1] + list(range(depth)) + [0] * (depth > 0) + list(range(depth + 1, 2 * depth))  # the root and two chains
    for _ in range(steps):
        rows = []
        for s in range(n):
            told = (known[s][lens[s] + 1:lens[s] + 1 + depth] if known else []) + [0] * depth
            rows.append([texts[s][-1]] + torch.randint(VOCAB, (depth,), generator=gen).tolist() + told[:depth])
        step = Step([tree] * n, lens, table)
        logits = model(torch.tensor(sum(rows, []), device="cuda"), step).view(n, len(tree), VOCAB)
        best = logits.argmax(-1).tolist()
        paths = [follow(tree, rows[s], best[s]) for s in range(n)]
        model.keep(torch.tensor([p + [-1] * (len(tree) - len(p)) for p in paths], dtype=torch.int32, device="cuda"), step)
        for s, p in enumerate(paths):
            texts[s] += [best[s][i] for i in p]
            lens[s] += len(p)
        logits = logits[torch.arange(n), torch.tensor([p[-1] for p in paths])]
        kept.append([len(p) for p in paths])
    return texts, kept, logits


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--prompt", type=int, default=300)
    ap.add_argument("--steps", type=int, default=4)
    ap.add_argument("--depth", type=int, default=3)
    a = ap.parse_args()
    prompts = (a.prompt, max(1, a.prompt * 2 // 5))
    first, _, _ = generate(a.layers, prompts, a.steps * (a.depth + 1), 0)
    texts, kept, _ = generate(a.layers, prompts, a.steps, a.depth, known=first)
    for s, t in enumerate(texts):
        print(f"sequence {s}: {len(t)} tokens, the last {t[-8:]}, kept a step: {[k[s] for k in kept]}")
