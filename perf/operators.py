"""Measured work of the decoder operators that stand between the GGUF linear layers: the 8-bit paged
KV cache (kv8_append with kv8_read, kv8_attention), the gated delta rule and the token log
probabilities, as vllm_gguf_plugin.decoder serves them.

The sizes are those of the 27B decoder whose linear layers perf/cases.py times: attention layers of
24 query and 4 key / value heads of 256 (q 6144, k and v 1024), linear-attention layers of 16 key
and 48 value heads of 128 (a fused qkv of 10240 rows), heads of 151936 and 248320 rows; and those of
a generic 4096-wide model (32 query and 8 key / value heads of 128). The "op" of a case says which
operator it calls:
  append     kv8_append of new tokens, then kv8_read of the pages that it touched
  attention  kv8_attention: one token a sequence (decode), some (verify) or many (a prompt's chunk)
  delta      gated_delta_rule; with "steps" the state after every token is kept, as a verify pass needs
  logprobs   token_logprobs of one given token a row, with the best "top" alternatives
Lengths of ragged batches are drawn from the case's own "mix", not from the seed of its inputs.
"""

import math
import os
import random
import sys

import torch

own = False  # False: run() computes the plain forms; True: it calls the framework's operators

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _append(seqs, new, before, heads=4, d=256, page=64, dtype="bf16", mix=0):
    return {"op": "append", "seqs": seqs, "new": new, "before": before, "heads": heads, "d": d, "page": page,
            "dtype": dtype, "mix": mix}


def _attention(seqs, new, ctx, hq=24, hkv=4, d=256, page=64, dtype="bf16", mix=0):
    return {"op": "attention", "seqs": seqs, "new": new, "ctx": ctx, "hq": hq, "hkv": hkv, "d": d, "page": page,
            "dtype": dtype, "mix": mix}


def _delta(seqs, new, hk=16, hv=48, dk=128, dv=128, dtype="bf16", steps=False, mix=0):
    return {"op": "delta", "seqs": seqs, "new": new, "hk": hk, "hv": hv, "dk": dk, "dv": dv, "dtype": dtype,
            "steps": steps, "mix": mix}


def _logprobs(rows, vocab, top, dtype="bf16"):
    return {"op": "logprobs", "rows": rows, "vocab": vocab, "top": top, "dtype": dtype}


def listed():
    return [
        # one decode step of 32 sequences: a token each into pages that hold older ones
        dict(_append(32, 1, 4000, mix=1), name="append-decode-b32"),
        # an 8192-token prompt into an empty cache
        dict(_append(1, 8192, 0), name="append-prompt-8192"),
        # one sequence early in a chat: the call's latency counts
        dict(_attention(1, 1, 701), name="attn-decode-b1-701"),
        # a full decode batch of ragged contexts up to 16K
        dict(_attention(64, 1, 16384, mix=2), name="attn-decode-b64-16k"),
        # a verify pass of three drafted tokens and one more, long contexts, pages of 16
        dict(_attention(8, 4, 32768, page=16, mix=3), name="attn-verify-b8x4-32k"),
        # the second chunk of 2048 tokens of a long prompt, up to position 8192
        dict(_attention(1, 2048, 8192), name="attn-prompt-2048-8k"),
        # a ragged batch of short prompts of a 4096-wide model in fp16
        dict(_attention(7, 777, 1100, hq=32, hkv=8, d=128, page=16, dtype="fp16", mix=4), name="attn-prompts-b7-fp16"),
        # one token of one sequence through a linear-attention layer
        dict(_delta(1, 1), name="delta-decode-b1"),
        # a verify pass of 32 sequences, the state after each of four tokens kept
        dict(_delta(32, 4, steps=True), name="delta-verify-b32x4"),
        # an 8192-token prompt of one sequence
        dict(_delta(1, 8192), name="delta-prompt-8192"),
        # one sampled row with 20 alternatives
        dict(_logprobs(1, 151936, 20, "fp32"), name="logprobs-b1-top20"),
        # prompt log probabilities of a 512-token chunk
        dict(_logprobs(512, 248320, 5), name="logprobs-512-top5"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "delta", "delta", "logprobs"])
    mix = rng.randrange(1, 1 << 30)
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "append":
        heads, d = rng.choice([(4, 256), (8, 128), (2, 64), (1, 192)])
        seqs = _log(rng, 1, 64)
        new = 1 if rng.random() < 0.4 else _log(rng, 2, 8192 // seqs)
        return _append(seqs, new, _log(rng, 1, 4096), heads, d, rng.choice([16, 32, 64, 144]), dtype, mix)
    if op == "attention":
        hq, hkv, d = rng.choice([(24, 4, 256), (24, 4, 256), (32, 8, 128), (8, 8, 64), (12, 1, 192)])
        page = rng.choice([16, 32, 64, 144])
        kind = rng.random()
        if kind < 0.45:
            seqs = _log(rng, 1, 64)
            return _attention(seqs, 1, _log(rng, 100, 16384), hq, hkv, d, page, dtype, mix)
        if kind < 0.7:
            seqs = _log(rng, 1, 8)
            return _attention(seqs, rng.randint(2, 8), _log(rng, 100, 32768), hq, hkv, d, page, dtype, mix)
        new = _log(rng, 16, 2048)
        return _attention(1 if new > 512 else rng.randint(1, 4), new, min(8192, new + _log(rng, 1, 6144)), hq, hkv, d,
                          page, dtype, mix)
    if op == "delta":
        hk, hv, dk, dv = rng.choice([(16, 48, 128, 128), (16, 48, 128, 128), (16, 32, 128, 128), (4, 4, 64, 128)])
        kind = rng.random()
        if kind < 0.35:
            return _delta(_log(rng, 1, 64), 1, hk, hv, dk, dv, rng.choice(["bf16", "fp32"]), False, mix)
        if kind < 0.6:
            return _delta(_log(rng, 1, 32), rng.randint(2, 6), hk, hv, dk, dv, dtype, True, mix)
        seqs = _log(rng, 1, 8)
        return _delta(seqs, _log(rng, 20, 8192 // seqs), hk, hv, dk, dv, dtype, False, mix)
    vocab = rng.choice([151936, 248320, 32000, 50257, 100003])
    dtype = "bf16" if vocab > 200000 else rng.choice(["bf16", "fp16", "fp32"])
    return _logprobs(_log(rng, 1, 512), vocab, rng.choice([0, 1, 5, 20]), dtype)


# ------------------------------------------------------------------------------------------ sizes


def _lengths(case, top, least):
    """Each sequence's length: `top` for one of them, the others drawn between its tenth and it."""
    rng = random.Random(case["mix"])
    n = [max(least, _log(rng, max(1, top // 10), max(1, top))) for _ in range(case["seqs"])]
    n[rng.randrange(len(n))] = top
    return n


def _new_tokens(case):
    """New tokens a sequence: equal numbers up to 8 (decode, verify), ragged prompts beyond."""
    return [case["new"]] * case["seqs"] if case["new"] <= 8 else _lengths(case, case["new"], 1)


def _ends(case):
    """Each sequence's length after the call."""
    new = _new_tokens(case)
    if case["op"] == "append":
        rng = random.Random(case["mix"] + 1)
        return [n + (rng.randrange(case["before"]) if case["before"] else 0) for n in new]
    ctx = _lengths(case, case["ctx"], 1)
    return [max(c, n) for c, n in zip(ctx, new)]


def _first_touched(case):
    """The first position of the page in which each sequence's new tokens begin."""
    return [(e - n) // case["page"] * case["page"] for e, n in zip(_ends(case), _new_tokens(case))]


def work(case):
    if case["op"] == "append":
        row = case["heads"] * case["d"] * 2  # K and V values of a token
        new, back = sum(_new_tokens(case)), sum(e - f for e, f in zip(_ends(case), _first_touched(case)))
        return {"bytes": row * (new * 3 + back * 3), "flops": row * (new * 3 + back)}
    if case["op"] == "attention":
        new, ends = _new_tokens(case), _ends(case)
        seen = sum(n * e - n * (n - 1) // 2 for n, e in zip(new, ends))
        return {"bytes": sum(ends) * case["hkv"] * case["d"] * 2 + sum(new) * case["hq"] * case["d"] * 4,
                "flops": 4 * seen * case["hq"] * case["d"]}
    if case["op"] == "delta":
        t, size = sum(_new_tokens(case)), 4 if case["dtype"] == "fp32" else 2
        state = case["hv"] * case["dk"] * case["dv"] * 4
        states = case["seqs"] + (t if case["steps"] else case["seqs"])
        return {"bytes": t * (2 * case["hk"] * case["dk"] + 2 * case["hv"] * case["dv"]) * size + t * case["hv"] * 8 +
                states * state, "flops": 6 * t * case["hv"] * case["dk"] * case["dv"]}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * (4 if case["dtype"] == "fp32" else 2) + case["rows"] * (20 + 8 * case["top"]), "flops": 4 * n}


# ----------------------------------------------------------------------------------------- inputs


def _offsets(n):
    cu = [0]
    for x in n:
        cu.append(cu[-1] + x)
    return cu


def _pages(case, ends, gen):
    """A block table over a pool of shuffled pages, and the pool's size."""
    each = [-(-e // case["page"]) for e in ends]
    total = sum(each)
    order = torch.randperm(total + 3, generator=gen)[:total]  # three pages belong to nobody
    table = torch.zeros(len(ends), max(each), dtype=torch.int32)
    at = 0
    for i, n in enumerate(each):
        table[i, :n] = order[at:at + n]
        at += n
    return table.cuda(), total + 3


def prepare(case, seed):
    host = torch.Generator().manual_seed(seed)
    dev = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=dev)

    if case["op"] == "logprobs":
        x = normal(case["rows"], case["vocab"]) * 2.5
        best = torch.randint(case["vocab"], (case["rows"], 8), device="cuda", generator=dev)
        x.scatter_add_(1, best, 6 + 3 * normal(case["rows"], 8))  # a few likely tokens a row
        ids = torch.randint(case["vocab"], (case["rows"],), device="cuda", generator=dev)
        likely = torch.rand(case["rows"], device="cuda", generator=dev) < 0.7
        return {"case": case, "logits": x.to(dtype), "ids": torch.where(likely, best[:, 0], ids)}

    new = _new_tokens(case)
    cu = torch.tensor(_offsets(new), dtype=torch.int32).cuda()
    t = sum(new)
    s = {"case": case, "cu": cu, "max_new": max(new)}
    if case["op"] == "delta":
        hk, hv, dk, dv = case["hk"], case["hv"], case["dk"], case["dv"]
        x = normal(t, 2 * hk * dk + hv * dv).to(dtype)  # one fused projection, as the layer has it
        s["q"], s["k"] = x[:, :hk * dk].view(t, hk, dk), x[:, hk * dk:2 * hk * dk].view(t, hk, dk)
        s["v"] = x[:, 2 * hk * dk:].view(t, hv, dv)
        rate = torch.exp(torch.rand(hv, device="cuda", generator=dev) * 6 - 5)  # slow and fast heads
        s["g"] = -rate * torch.nn.functional.softplus(normal(t, hv))
        s["beta"] = torch.sigmoid(normal(t, hv))
        n = case["seqs"]
        kept = n * case["new"] if case["steps"] else n
        s["state"] = torch.zeros(n + kept, hv, dv, dk, device="cuda")
        s["state"][:n] = 0.3 * normal(n, hv, dv, dk)
        s["slots"] = torch.randperm(n, generator=host).to(torch.int32).cuda()
        out = n + torch.arange(kept, dtype=torch.int32)
        s["out_slots"] = (out.view(n, -1) if case["steps"] else out).cuda()
        return s

    ends = _ends(case)
    s["table"], pages = _pages(case, ends, host)
    s["ends"] = torch.tensor(ends, dtype=torch.int32).cuda()
    s["max_len"] = max(ends)
    heads, d, page = case["heads" if case["op"] == "append" else "hkv"], case["d"], case["page"]
    # codes of normal values with a page's largest at 127 or so, keys with a few strong channels
    s["k"] = (normal(pages, heads, page, d) * 36).round_().clamp_(-127, 127).to(torch.int8)
    s["v"] = (normal(pages, heads, d, page) * 36).round_().clamp_(-127, 127).to(torch.int8)
    s["ks"] = torch.exp(0.3 * normal(pages, heads)) / 36
    s["vs"] = torch.exp(0.3 * normal(pages, heads)) / 36
    if case["op"] == "append":
        kv = normal(2, t, heads, d)
        kv[0, ..., ::37] *= 4
        s["key"], s["value"] = kv[0].to(dtype), kv[1].to(dtype)
        first = _first_touched(case)
        back = [e - f for e, f in zip(ends, first)]
        s["first"] = torch.tensor(first, dtype=torch.int32).cuda()
        s["cu_back"] = torch.tensor(_offsets(back), dtype=torch.int32).cuda()
        s["back"], s["max_back"] = sum(back), max(back)
    else:
        s["q"] = (normal(t, case["hq"], d) * 1.5).to(dtype)
    return s


# ------------------------------------------------------------------------------------ plain forms


def _ragged(cu, total):
    """(sequence, index in it) of each of the `total` tokens of cu_seqlens `cu`."""
    at = torch.arange(total, device=cu.device)
    seq = torch.searchsorted(cu.long(), at, right=True) - 1
    return seq, at - cu.long()[seq]


def _plain_append(s):
    case = s["case"]
    page, t = case["page"], s["key"].shape[0]
    seq, at = _ragged(s["cu"], t)
    start = s["ends"].long() - (s["cu"][1:] - s["cu"][:-1]).long()  # older tokens of each sequence
    pos = start[seq] + at
    pid = s["table"].long()[seq, pos // page]
    off = pos % page
    older = torch.zeros(s["ks"].shape[0], dtype=torch.long, device="cuda")  # older tokens of a touched page
    older[pid] = (start[seq] - pos // page * page).clamp(min=0)
    touched = torch.zeros_like(older, dtype=torch.bool)
    touched[pid] = True
    for x, codes, scale, tokens in ((s["key"], s["k"], s["ks"], 2), (s["value"], s["v"], s["vs"], 3)):
        x = x.float()
        most = torch.zeros_like(scale).index_reduce_(0, pid, x.abs().amax(-1), "amax")
        fresh = most / 127
        fresh = torch.where(fresh < 2.0 ** -100, 0.0, fresh)
        was = torch.where((older > 0)[:, None], scale, 0.0)
        now = torch.maximum(was, fresh)
        ratio = torch.where(now > was, was / now, 1.0)[touched]  # rescales what the page holds
        old = codes[touched]
        shape = [1, 1, 1, 1]
        shape[tokens] = page
        keep = (torch.arange(page, device="cuda").view(shape) < older[touched].view(-1, 1, 1, 1))
        codes[touched] = torch.where(keep, torch.round(old.float() * ratio[:, :, None, None]).to(torch.int8), old)
        inv = torch.where(now > 0, 1 / now, 0.0)
        q = torch.round(x * inv[pid][..., None]).clamp(-127, 127).to(torch.int8)
        if tokens == 2:
            codes[pid, :, off] = q
        else:
            codes[pid, :, :, off] = q
        scale[touched] = now[touched]


def _plain_values(s, seq, pos, dtype):
    """K and V of the given positions as the cache holds them: [..., heads, d]."""
    page = s["case"]["page"]
    pid, off = s["table"].long()[seq, pos // page], pos % page
    k = s["k"][pid, :, off].float() * s["ks"][pid][..., None]
    v = s["v"][pid, :, :, off].float() * s["vs"][pid][..., None]
    return k.to(dtype), v.to(dtype)


def _plain_attention(s):
    case = s["case"]
    n, rep = case["seqs"], case["hq"] // case["hkv"]
    seq, at = _ragged(s["cu"], s["q"].shape[0])
    q = torch.zeros(n, s["max_new"], *s["q"].shape[1:], device="cuda")
    q[seq, at] = s["q"].float()
    q = q.view(n, s["max_new"], case["hkv"], rep, -1).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [n, hkv, rep * new, d]
    pos = torch.arange(s["max_len"], device="cuda")
    ends = s["ends"].long()[:, None]
    k, v = _plain_values(s, torch.arange(n, device="cuda")[:, None], torch.minimum(pos[None], ends - 1), torch.float32)
    x = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) * case["d"] ** -0.5
    x = x.view(n, case["hkv"], rep, s["max_new"], -1)
    new = (s["cu"][1:] - s["cu"][:-1]).long()[:, None]
    last = ends - new + torch.arange(s["max_new"], device="cuda")[None]  # the last position a query sees
    x = x.masked_fill((pos > last[..., None])[:, None, None], -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e30))
    o = torch.matmul(p.flatten(2, 3), v.permute(0, 2, 1, 3).contiguous())
    o = o.view(n, case["hkv"], rep, s["max_new"], -1) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return o.permute(0, 3, 1, 2, 4).flatten(2, 3)[seq, at].to(s["q"].dtype)


def _plain_delta(s):
    """The chunked form over chunks of 64 tokens of all sequences at once (of one token where few
    are new), each padded with tokens that change nothing."""
    case = s["case"]
    n, hv, c = case["seqs"], case["hv"], 1 if s["max_new"] <= 8 else 64
    chunks = -(-s["max_new"] // c)
    seq, at = _ragged(s["cu"], s["q"].shape[0])

    def padded(x):
        y = torch.zeros(n, chunks * c, *x.shape[1:], device="cuda")
        y[seq, at] = x
        return y.view(n, chunks, c, hv, -1).permute(1, 0, 3, 2, 4).contiguous()  # [chunks, n, hv, c, .]

    def keys(x):
        x = x.float()
        x = x * torch.rsqrt((x * x).sum(-1, keepdim=True) + 1e-6)
        return padded(x.repeat_interleave(hv // case["hk"], 1))

    q, k, v = keys(s["q"]) * case["dk"] ** -0.5, keys(s["k"]), padded(s["v"].float())
    beta, gate = padded(s["beta"][..., None]), padded(s["g"][..., None]).cumsum(-2)
    low = torch.ones(c, c, dtype=torch.bool, device="cuda").tril()
    decay = torch.exp((gate - gate.transpose(-1, -2)).masked_fill(~low, -math.inf))
    kt = k.transpose(-1, -2).contiguous()
    a = (beta * torch.matmul(k, kt) * decay).tril(-1)
    scores = torch.matmul(q, kt) * decay
    inv = torch.eye(c, device="cuda").expand_as(a).clone()
    for i in range(1, c):  # rows of (1 + a)^-1 by forward substitution, of all chunks at once
        inv[..., i, :i] = -torch.matmul(a[..., i:i + 1, :i], inv[..., :i, :i]).squeeze(-2)
    grow, rest = torch.exp(gate), torch.exp(gate[..., -1:, :] - gate)
    w, u = torch.matmul(inv, beta * grow * k), torch.matmul(inv, beta * v)
    kr = (rest * k).transpose(-1, -2).contiguous()
    state = s["state"][s["slots"].long()].transpose(-1, -2).contiguous()  # [n, hv, dk, dv]
    out = torch.empty_like(v)
    for i in range(chunks):
        fresh = u[i] - torch.matmul(w[i], state)
        out[i] = torch.matmul(grow[i] * q[i], state) + torch.matmul(scores[i], fresh)
        state = grow[i][..., -1:, :] * state + torch.matmul(kr[i], fresh)
        if case["steps"]:
            s["state"][s["out_slots"][:, i].long()] = state.transpose(-1, -2)
    if not case["steps"]:
        s["state"][s["out_slots"].long()] = state.transpose(-1, -2)
    out = out.permute(1, 0, 3, 2, 4).reshape(n, chunks * c, hv, -1)[seq, at]
    return [out.to(s["q"].dtype), s["state"][n:]]


def _plain_logprobs(s):
    x, ids, top = s["logits"].float(), s["ids"][:, None], s["case"]["top"]
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(-1, keepdim=True)
    lse = m + torch.log(total)
    entropy = lse - (e * x).sum(-1, keepdim=True) / total
    given = x.gather(1, ids)
    index = torch.arange(x.shape[1], device="cuda")
    rank = 1 + ((x > given) | ((x == given) & (index < ids))).sum(-1)
    # a key that orders by value, then by the lower index
    bits = x.view(torch.int32).long()
    key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 20) + ((1 << 20) - 1 - index)
    best = (1 << 20) - 1 - (key.topk(top, -1).values & ((1 << 20) - 1))
    return [(given - lse)[:, 0], rank.int(), entropy[:, 0], x.gather(1, best) - lse, best.int()]


# -------------------------------------------------------------------------------------------- run


def run(state):
    s, case = state, state["case"]
    if own:
        return _own(s, case)
    if case["op"] == "append":
        _plain_append(s)
        seq, at = _ragged(s["cu_back"], s["back"])
        return list(_plain_values(s, seq, s["first"].long()[seq] + at, s["key"].dtype))
    if case["op"] == "attention":
        return _plain_attention(s)
    return _plain_delta(s) if case["op"] == "delta" else _plain_logprobs(s)


def _own(s, case):
    path = os.path.join(_ROOT, "vllm-gsqrco-exl3_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from vllm_gguf_plugin import decoder

    if case["op"] == "logprobs":
        return list(decoder.token_logprobs(s["logits"], s["ids"], case["top"]))
    if case["op"] == "delta":
        out = decoder.gated_delta_rule(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], s["slots"], s["cu"],
                                       s["max_new"], out_slots=s["out_slots"])
        return [out, s["state"][case["seqs"]:]]
    cache = decoder.Kv8Cache(s["k"], s["v"], s["ks"], s["vs"])
    if case["op"] == "append":
        decoder.kv8_append(cache, s["key"], s["value"], s["table"], s["ends"], s["cu"], s["max_new"])
        return list(decoder.kv8_read(cache, s["table"], s["first"], s["cu_back"], s["back"], s["max_back"],
                                     s["key"].dtype))
    return decoder.kv8_attention(s["q"], cache, s["table"], s["ends"], s["cu"], s["max_new"], s["max_len"])


# --------------------------------------------------------------------- the definitions in 64 bits


def _exact_append(s):
    """Sequence by sequence and page by page: what the touched pages hold after the new tokens."""
    case = s["case"]
    page, cu, ends, first = case["page"], s["cu"].tolist(), s["ends"].tolist(), s["first"].tolist()
    table = s["table"].tolist()
    both = []
    for x, codes, scales, turned in ((s["key"], s["k"], s["ks"], False), (s["value"], s["v"], s["vs"], True)):
        parts = []
        for i, end in enumerate(ends):
            start = end - (cu[i + 1] - cu[i])
            for p0 in range(first[i], end, page):
                pid, lo, hi = table[i][p0 // page], max(start, p0), min(end, p0 + page)
                fresh = x[cu[i] + lo - start:cu[i] + hi - start].double()  # [tokens, heads, d]
                now = (fresh.abs().amax((0, 2)).float() / 127).double()
                if start > p0:
                    held = codes[pid].transpose(1, 2) if turned else codes[pid]
                    held = held[:, :start - p0].permute(1, 0, 2).double()
                    was = scales[pid].double()
                    now = torch.maximum(now, was)
                    held = torch.round(held * (was / now)[:, None])
                    parts.append(held * now[:, None])
                parts.append(torch.round(fresh / now[:, None]).clamp(-127, 127) * now[:, None])
        both.append(torch.cat(parts))
    return both


def _exact_attention(s):
    case = s["case"]
    page, rep = case["page"], case["hq"] // case["hkv"]
    cu, ends = s["cu"].tolist(), s["ends"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, end in enumerate(ends):
        pids = s["table"][i, :-(-end // page)].long()
        k = (s["k"][pids].double() * s["ks"][pids].double()[..., None, None]).permute(1, 0, 2, 3).flatten(1, 2)[:, :end]
        v = (s["v"][pids].double() * s["vs"][pids].double()[..., None, None]).permute(1, 0, 3, 2).flatten(1, 2)[:, :end]
        n = cu[i + 1] - cu[i]
        hidden = torch.arange(end, device="cuda") > torch.arange(end - n, end, device="cuda")[:, None]
        for h in range(case["hq"]):
            x = s["q"][cu[i]:cu[i + 1], h].double() @ k[h // rep].T / math.sqrt(case["d"])
            out[cu[i]:cu[i + 1], h] = torch.softmax(x.masked_fill(hidden, -math.inf), -1) @ v[h // rep]
    return out


def _exact_delta(s):
    """Token by token, all sequences of a length still running at once."""
    case = s["case"]
    rep, cu = case["hv"] // case["hk"], s["cu"].long()
    n = case["seqs"]
    new = cu[1:] - cu[:-1]
    longest = torch.argsort(new, descending=True)
    lengths = new[longest].tolist()
    state = s["state"][s["slots"].long()[longest]].double()  # [n, hv, dv, dk]
    out = torch.zeros(s["v"].shape, dtype=torch.float64, device="cuda")
    kept = torch.zeros(s["state"][n:].shape, dtype=torch.float64, device="cuda")
    unit = [x.double() / torch.sqrt(x.double().square().sum(-1, keepdim=True) + 1e-6) for x in (s["q"], s["k"])]
    g, beta, v = s["g"].double().exp(), s["beta"].double(), s["v"].double()
    running = n
    for i in range(s["max_new"]):
        while lengths[running - 1] <= i:
            running -= 1
        at = cu[:-1][longest[:running]] + i
        q, k = (x[at].repeat_interleave(rep, 1) for x in unit)
        m = state[:running] * g[at][..., None, None]
        fresh = beta[at][..., None] * (v[at] - torch.matmul(m, k[..., None])[..., 0])
        m += fresh[..., None] * k[..., None, :]
        state[:running] = m
        out[at] = torch.matmul(m, q[..., None])[..., 0] / math.sqrt(case["dk"])
        if case["steps"]:
            kept[s["out_slots"][longest[:running], i].long() - n] = m
    if not case["steps"]:
        kept[s["out_slots"][longest].long() - n] = state
    return [out, kept]


def _exact_logprobs(s):
    rows = []
    for x, t in zip(s["logits"], s["ids"].tolist()):
        lp = torch.log_softmax(x.double(), -1)
        order = torch.sort(x.double(), descending=True, stable=True).indices
        best = order[:s["case"]["top"]]
        rows.append((lp[t], (order == t).nonzero()[0, 0] + 1, -(lp.exp() * lp).sum(), lp[best], best))
    return [torch.stack(x) for x in zip(*rows)]


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "delta": _exact_delta,
            "logprobs": _exact_logprobs}[case["op"]](s)
