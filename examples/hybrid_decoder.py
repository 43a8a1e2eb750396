"""A small hybrid decoder over this framework's operators: GGUF linear layers (Q4_K weights through
GGUFLinearMethod's ops), linear-attention layers with the gated delta rule, attention layers over the
8-bit paged KV cache, and token log probabilities behind the head.

    python examples/hybrid_decoder.py [--layers 4] [--prompt 300] [--tokens 8] [--drafts 3]

It reads a prompt for two sequences of different lengths, decodes token by token, then verifies drafted tokens: a
group of drafts runs at once, their log probabilities say how many are kept, and the states after
the last kept token go on (the recurrent states by slot, the cache by its length). Weights are
random, so the text means nothing. Needs an MI355X; the sizes are small, the calls are those of a
large model.
"""

import argparse
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "vllm-gsqrco-exl3_amd"))

from vllm_gguf_plugin import decoder, ops  # noqa: E402,F401

Q4_K, BLOCK = 12, 144  # ggml type id, bytes of 256 values
HIDDEN, VOCAB = 1024, 4096
HQ, HKV, D, PAGE = 12, 2, 128, 64          # attention layers
HK, HV, DK, DV = 2, 8, 128, 128            # linear-attention layers


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


def norm(x):
    return (x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-6)).to(x.dtype)


class Batch:
    """The ragged batch of one step: rows, lengths after it, pages and state slots."""

    def __init__(self, news, ends, table, slots, out_slots):
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        self.cu, self.ends = i32([0] + list(torch.tensor(news).cumsum(0))), i32(ends)
        self.table, self.slots, self.out_slots = table, i32(slots), i32(out_slots)
        self.max_new, self.max_len = max(news), max(ends)


class DeltaLayer:
    def __init__(self, gen, slots):
        self.qkv, self.gates = Linear(2 * HK * DK + HV * DV, HIDDEN, gen), Linear(2 * 16, HIDDEN, gen)
        self.out = Linear(HIDDEN, HV * DV, gen)
        self.state = torch.zeros(slots, HV, DV, DK, device="cuda")

    def __call__(self, x, b):
        t = x.shape[0]
        y = self.qkv(x)
        q, k = y[:, :HK * DK].view(t, HK, DK), y[:, HK * DK:2 * HK * DK].view(t, HK, DK)
        v = y[:, 2 * HK * DK:].view(t, HV, DV)
        gates = self.gates(x).float()
        g = -0.3 * torch.nn.functional.softplus(gates[:, :HV])
        beta = torch.sigmoid(gates[:, 16:16 + HV])
        o = decoder.gated_delta_rule(q, k, v, g, beta, self.state, b.slots, b.cu, b.max_new, out_slots=b.out_slots)
        return self.out(norm(o.reshape(t, HV * DV)))


class AttentionLayer:
    def __init__(self, gen, pages):
        self.qkv, self.out = Linear((HQ + 2 * HKV) * D, HIDDEN, gen), Linear(HIDDEN, HQ * D, gen)
        self.cache = decoder.Kv8Cache.empty(pages, HKV, PAGE, D)

    def __call__(self, x, b):
        q, k, v = self.qkv(x).view(-1, HQ + 2 * HKV, D).split((HQ, HKV, HKV), 1)
        decoder.kv8_append(self.cache, k, v, b.table, b.ends, b.cu, b.max_new)
        o = decoder.kv8_attention(q, self.cache, b.table, b.ends, b.cu, b.max_new, b.max_len)
        return self.out(o.reshape(x.shape[0], HQ * D))


class Model:
    def __init__(self, layers, pages, slots, seed=0):
        gen = torch.Generator().manual_seed(seed)
        self.embed = torch.randn(VOCAB, HIDDEN, generator=gen).to(torch.bfloat16).cuda()
        self.layers = [AttentionLayer(gen, pages) if i % 4 == 3 else DeltaLayer(gen, slots) for i in range(layers)]
        self.head = Linear(VOCAB, HIDDEN, gen)

    def __call__(self, tokens, b):
        x = self.embed[tokens]
        for layer in self.layers:
            x = x + layer(norm(x), b)
        return self.head(norm(x))


def generate(layers=4, prompts=(300, 117), tokens=8, drafts=3, seed=0):
    """Returns each sequence's tokens and their log probabilities."""
    n = len(prompts)
    gen = torch.Generator().manual_seed(seed + 1)
    texts = [torch.randint(VOCAB, (p,), generator=gen).tolist() for p in prompts]
    room = -(-(max(prompts) + tokens + drafts + 2) // PAGE)  # pages: the decoded tokens, a verify pass, one token more
    # slots 0 .. n - 1 hold the states, the others the states after each row of a verify pass
    m = drafts + 1
    model = Model(layers, n * room, n + n * m, seed)
    table = torch.randperm(n * room, generator=gen).view(n, room).to(torch.int32).cuda()
    lens, logprobs = list(prompts), [[] for _ in range(n)]

    # the prompt: states from zero (-1), kept in the sequences' slots
    logits = model(torch.tensor(sum(texts, []), device="cuda"), Batch(prompts, lens, table, [-1] * n, list(range(n))))
    last = torch.tensor(prompts).cumsum(0).cuda() - 1
    nxt = logits[last].argmax(-1)
    for _ in range(tokens):  # one token a sequence
        lens = [x + 1 for x in lens]
        logits = model(nxt, Batch([1] * n, lens, table, list(range(n)), list(range(n))))
        for s, t in enumerate(nxt.tolist()):
            texts[s].append(t)
        nxt = logits.argmax(-1)
        lp, _, _, _, _ = decoder.token_logprobs(logits, nxt, 4)
        for s, v in enumerate(lp.tolist()):
            logprobs[s].append(v)

    # a verify pass: the sampled token and `drafts` guesses behind it
    guess = torch.randint(VOCAB, (n, drafts), generator=gen).cuda()
    rows = torch.cat([nxt[:, None], guess], 1)
    kept_slots = [[n + s * m + i for i in range(m)] for s in range(n)]
    logits = model(rows.flatten(), Batch([m] * n, [x + m for x in lens], table, list(range(n)), kept_slots))
    given = torch.cat([guess, nxt[:, None]], 1).flatten()  # (nothing is drafted behind the last row: any token)
    _, ranks, _, _, best = decoder.token_logprobs(logits, given, 1)
    good = (ranks.view(n, m)[:, :drafts] == 1).long().cumprod(-1).sum(-1).tolist()  # drafts that are the best tokens
    nxt = best.view(n, m)[torch.arange(n), torch.tensor(good)].long()
    for s in range(n):
        texts[s] += rows[s, :1 + good[s]].tolist()
        lens[s] += 1 + good[s]
    # go on from the state after the last kept row; the cache simply ends there
    slots = [kept_slots[s][good[s]] for s in range(n)]
    lens = [x + 1 for x in lens]
    logits = model(nxt, Batch([1] * n, lens, table, slots, list(range(n))))
    return texts, logprobs, logits


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=300)
    ap.add_argument("--tokens", type=int, default=8)
    ap.add_argument("--drafts", type=int, default=3)
    a = ap.parse_args()
    texts, logprobs, logits = generate(a.layers, (a.prompt, max(1, a.prompt * 2 // 5)), a.tokens, a.drafts)
    for s, t in enumerate(texts):
        print(f"sequence {s}: {len(t)} tokens, the last {t[-(a.tokens + 1):]}, log probabilities "
              + " ".join(f"{v:.2f}" for v in logprobs[s]))
