"""Measured work of the operators of a decode or verify step's attention block, as
vllm_gguf_plugin.decoder serves them: norms with their residual and gate (residual_norm, gated_norm),
the position rotation on the way into the 8-bit paged cache (kv8_rotary_append), attention for a tree of
drafted tokens (kv8_tree_attention), and moving the accepted path to its place (kv8_keep).

The sizes are those of the 27B decoder whose linear layers perf/cases.py times: 5120 wide, attention
layers of 24 query and 4 key / value heads of 256, 48 value heads of 128 in its linear-attention layers; and those
of a generic 4096-wide model (32 query and 8 key / value heads of 128). The "op" of a case says which
operator it calls:
  rotary  kv8_rotary_append of new tokens (with the heads' norms where "norms"), then kv8_read of the pages that it touched
  tree    kv8_tree_attention of a tree of "new" drafted tokens a sequence
  keep    kv8_keep of one path of each sequence's tree, then kv8_read of the rows kept
  norm    residual_norm of [rows, n], or gated_norm of [rows, heads, n] where there is no residual
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
EPS = 1e-6


def _rotary(seqs, new, before, hq=24, heads=4, d=256, rot=64, pairs=False, norms=True, page=64, dtype="bf16", mix=0):
    return {"op": "rotary", "seqs": seqs, "new": new, "before": before, "hq": hq, "heads": heads, "d": d, "rot": rot,
            "pairs": pairs, "norms": norms, "page": page, "dtype": dtype, "mix": mix}


def _tree(seqs, new, ctx, hq=24, heads=4, d=256, page=64, dtype="bf16", mix=0):
    return {"op": "tree", "seqs": seqs, "new": new, "ctx": ctx, "hq": hq, "heads": heads, "d": d, "page": page,
            "dtype": dtype, "mix": mix}


def _keep(seqs, new, before, heads=4, d=256, page=64, mix=0):
    return {"op": "keep", "seqs": seqs, "new": new, "before": before, "heads": heads, "d": d, "page": page,
            "dtype": "bf16", "mix": mix}


def _norm(rows, n, heads=1, inner=False, residual="bf16", act="none", scale=1.0, dtype="bf16"):
    return {"op": "norm", "rows": rows, "n": n, "heads": heads, "inner": inner, "residual": residual, "act": act,
            "scale": scale, "dtype": dtype}


def listed():
    return [
        # one decode step of 32 sequences: a token each into pages that hold older ones
        dict(_rotary(32, 1, 4000, mix=1), name="rotary-decode-b32"),
        # a verify pass of 16 drafts in each of 8 sequences of a 4096-wide fp16 model: all dims rotate, in pairs
        dict(_rotary(8, 16, 4000, 32, 8, 128, 128, True, False, 16, "fp16", mix=2), name="rotary-verify-b8x16-fp16"),
        # an 8192-token prompt into an empty cache
        dict(_rotary(1, 8192, 0), name="rotary-prompt-8192"),
        # one sequence, a small tree, early in a chat: the call's latency counts
        dict(_tree(1, 8, 1999), name="tree-b1x8-2k"),
        # 16 drafts in each of 8 ragged sequences of long contexts
        dict(_tree(8, 16, 32768, mix=3), name="tree-b8x16-32k"),
        # an odd tree of 47 drafts over middle contexts
        dict(_tree(4, 47, 16000, mix=4), name="tree-b4x47-16k"),
        # the largest trees of a mask word, a full batch of a 4096-wide fp16 model, pages of 16
        dict(_tree(32, 64, 8192, 32, 8, 128, 16, "fp16", mix=5), name="tree-b32x64-8k-fp16"),
        # the accepted path of one sequence's 8 drafts
        dict(_keep(1, 8, 2000, mix=6), name="keep-b1x8"),
        # of 64 sequences' 64 drafts, over pages of 16
        dict(_keep(64, 64, 4000, 8, 128, 16, mix=7), name="keep-b64x64"),
        # the norm before a block of a decode step of 4 rows
        dict(_norm(4, 5120), name="norm-decode-4x5120"),
        # the norm after a block, its residual scale and the next block's norm, a prompt's rows
        dict(_norm(8192, 5120, inner=True, scale=0.5), name="norm-sandwich-8192x5120"),
        # the gated norm of each head behind the linear attention, a prompt's rows
        dict(_norm(8192, 128, 48, True, "none", "silu"), name="norm-gated-8192x48x128"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "tree", "tree", "tree", "keep", "norm", "norm"])
    mix = rng.randrange(1, 1 << 30)
    page = rng.choice([16, 32, 64, 144])
    if op == "rotary":
        hq, heads, d, rot = rng.choice([(24, 4, 256, 64), (24, 4, 256, 256), (32, 8, 128, 128), (8, 2, 64, 32), (12, 1, 192, 96)])
        seqs = _log(rng, 1, 64)
        new = 1 if rng.random() < 0.3 else _log(rng, 2, 64) if rng.random() < 0.5 else _log(rng, 2, max(2, 8192 // seqs))
        return _rotary(seqs, new, _log(rng, 1, 4096), hq, heads, d, rot, rng.random() < 0.4, rng.random() < 0.5, page,
                       rng.choice(["bf16", "fp16", "fp32"]), mix)
    if op == "tree":
        hq, heads, d = rng.choice([(24, 4, 256), (24, 4, 256), (32, 8, 128), (8, 8, 64), (12, 1, 192)])
        seqs, new = _log(rng, 1, 32), _log(rng, 1, 100)
        most = 32 * 64 * 8192 // (seqs * new)  # no more than the largest listed one
        return _tree(seqs, new, _log(rng, 100, max(200, min(32768, most))), hq, heads, d, page, rng.choice(["bf16", "bf16", "fp16"]), mix)
    if op == "keep":
        heads, d = rng.choice([(4, 256), (8, 128), (2, 64), (1, 192)])
        return _keep(_log(rng, 1, 64), _log(rng, 2, 100), _log(rng, 1, 4096), heads, d, page, mix)
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if rng.random() < 0.4:
        return _norm(_log(rng, 1, 4096), rng.choice([64, 96, 128, 128, 192, 256]), rng.choice([8, 24, 48]), True, "none",
                     rng.choice(["silu", "sigmoid"]), 1.0, dtype)
    return _norm(_log(rng, 1, 8192), rng.choice([1024, 2560, 4096, 4097, 5120, 5120, 2880]), 1, rng.random() < 0.5,
                 rng.choice([dtype, "fp32"]), rng.choice(["none", "none", "sigmoid"]), rng.choice([1.0, 0.22]), dtype)


# ------------------------------------------------------------------------------------------ sizes


def _lengths(case, top, least):
    """Each sequence's length: `top` for one of them, the others drawn between its tenth and it."""
    rng = random.Random(case["mix"])
    n = [max(least, _log(rng, max(1, top // 10), max(1, top))) for _ in range(case["seqs"])]
    n[rng.randrange(len(n))] = top
    return n


def _new_tokens(case):
    """New tokens a sequence: equal numbers of drafts, ragged prompts beyond 100."""
    return [case["new"]] * case["seqs"] if case["new"] <= 100 else _lengths(case, case["new"], 1)


def _ends(case):
    """Each sequence's length with its new tokens."""
    new = _new_tokens(case)
    if case["op"] == "tree":
        return [c + n for c, n in zip(_lengths(case, case["ctx"], 0), new)]
    rng = random.Random(case["mix"] + 1)
    return [n + (rng.randrange(case["before"]) if case["before"] else 0) for n in new]


def _first_touched(case):
    """The first position of the page in which each sequence's new tokens begin."""
    return [(e - n) // case["page"] * case["page"] for e, n in zip(_ends(case), _new_tokens(case))]


def _kept(case):
    """How many rows of each sequence's tree are kept."""
    rng = random.Random(case["mix"] + 2)
    return [rng.randint(1, max(1, min(n, 8))) for n in _new_tokens(case)]


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm":
        n = case["rows"] * case["heads"] * case["n"]
        if case["residual"] == "none":
            return {"bytes": n * 3 * size, "flops": 8 * n}
        each = 2 * size + 2 * (4 if case["residual"] == "fp32" else 2) + (size if case["act"] != "none" else 0)
        return {"bytes": n * each, "flops": 8 * n}
    new, ends = _new_tokens(case), _ends(case)
    t, row = sum(new), case["heads"] * case["d"]
    if case["op"] == "tree":
        seen = sum(n * (e - n) + n * n // 4 for n, e in zip(new, ends))
        return {"bytes": sum(ends) * row * 2 + t * (case["hq"] * case["d"] * 4 + 8), "flops": 4 * seen * case["hq"] * case["d"]}
    if case["op"] == "keep":
        k = sum(_kept(case))
        return {"bytes": k * row * 2 * (2 + 3), "flops": k * row * 4}
    back = sum(e - f for e, f in zip(ends, _first_touched(case)))
    return {"bytes": t * (row * 2 * (size + 1) + case["hq"] * case["d"] * 2 * size + case["rot"] * 4) + back * row * 2 * 3,
            "flops": t * (case["hq"] * case["d"] * 6 + row * 10)}


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


def _trees(case, seed):
    """Each sequence's tree, as its rows' parents (-1 for the first row, the token sampled last)."""
    rng = random.Random(seed)
    return [[-1] + [rng.randrange(max(0, i - 9), i) for i in range(1, n)] for n in _new_tokens(case)]


def prepare(case, seed):
    host = torch.Generator().manual_seed(seed)
    dev = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=dev)

    if case["op"] == "norm":
        shape = (case["rows"], case["heads"], case["n"])[::1 if case["residual"] == "none" else 2]  # heads only without a residual
        s = {"case": case, "x": (normal(*shape) * torch.exp(0.5 * normal(*shape[:-1], 1))).to(dtype)}
        s["inner"] = 1 + 0.2 * normal(case["n"]) if case["inner"] else None
        s["gate"] = normal(*shape).to(dtype) if case["act"] != "none" else None
        s["residual"] = (3 * normal(*shape)).to(DTYPES[case["residual"]]) if case["residual"] != "none" else None
        s["weight"] = 1 + 0.2 * normal(case["n"]) if s["residual"] is not None else None
        return s

    new, ends = _new_tokens(case), _ends(case)
    cu = torch.tensor(_offsets(new), dtype=torch.int32).cuda()
    t, heads, d, page = sum(new), case["heads"], case["d"], case["page"]
    s = {"case": case, "cu": cu, "max_new": max(new), "max_len": max(ends)}
    s["table"], pages = _pages(case, ends, host)
    s["ends"] = torch.tensor(ends, dtype=torch.int32).cuda()
    # codes of normal values with a page's largest at 127 or so
    s["k"] = (normal(pages, heads, page, d) * 36).round_().clamp_(-127, 127).to(torch.int8)
    s["v"] = (normal(pages, heads, d, page) * 36).round_().clamp_(-127, 127).to(torch.int8)
    s["ks"] = torch.exp(0.3 * normal(pages, heads)) / 36
    s["vs"] = torch.exp(0.3 * normal(pages, heads)) / 36
    if case["op"] == "rotary":
        hq, rot = case["hq"], case["rot"]
        x = normal(t, hq + 2 * heads, d)  # one fused projection, as the layer has it
        x[:, hq:hq + heads, ::37] *= 4  # keys with a few strong channels
        x = x.to(dtype)
        s["query"], s["key"], s["value"] = x[:, :hq], x[:, hq:hq + heads], x[:, hq + heads:]
        s["qw"], s["kw"] = (1 + 0.2 * normal(d), 1 + 0.2 * normal(d)) if case["norms"] else (None, None)
        inv = 1e6 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
        angle = torch.arange(max(ends), dtype=torch.float64)[:, None] * inv
        s["cos_sin"] = torch.cat([torch.cos(angle), torch.sin(angle)], 1).float().cuda()
        s["positions"] = torch.cat([torch.arange(e - n, e) for n, e in zip(new, ends)]).cuda()
        first = _first_touched(case)
        back = [e - f for e, f in zip(ends, first)]
    else:
        trees = _trees(case, seed)
    if case["op"] == "tree":
        words = -(-max(new) // 64)
        mask = []
        for tree in trees:  # a row sees itself and its ancestors
            rows = []
            for i, p in enumerate(tree):
                rows.append((rows[p] if p >= 0 else 0) | 1 << i)
            mask += [[(r >> 64 * w & (1 << 64) - 1) - (1 << 64) * (r >> 64 * w + 63 & 1) for w in range(words)] for r in rows]
        s["mask"] = torch.tensor(mask, dtype=torch.int64).cuda()
        s["q"] = (normal(t, case["hq"], d) * 1.5).to(dtype)
        return s
    if case["op"] == "keep":
        rng, paths = random.Random(seed + 1), []
        for tree, n in zip(trees, _kept(case)):
            path = [rng.randrange(n - 1, len(tree))]
            while path[0] >= 0:
                path.insert(0, tree[path[0]])
            rows = path[1:n + 1]
            rows += [r for r in range(rows[-1] + 1, len(tree))][:n - len(rows)]  # n rows: the path, and the next ones where it ends
            rows += [-1] * (8 - len(rows))
            paths.append(rows)
        s["path"] = torch.tensor(paths, dtype=torch.int32).cuda()
        s["start"] = s["ends"] - (cu[1:] - cu[:-1])
        first, back = (s["ends"] - (cu[1:] - cu[:-1])).tolist(), [sum(r >= 0 for r in p) for p in paths]
        del s["max_len"]
    s["first"] = torch.tensor(first, dtype=torch.int32).cuda()
    s["cu_back"] = torch.tensor(_offsets(back), dtype=torch.int32).cuda()
    s["back"], s["max_back"] = sum(back), max(back)
    return s


# ------------------------------------------------------------------------------------ plain forms


def _ragged(cu, total):
    """(sequence, index in it) of each of the `total` tokens of cu_seqlens `cu`."""
    at = torch.arange(total, device=cu.device)
    seq = torch.searchsorted(cu.long(), at, right=True) - 1
    return seq, at - cu.long()[seq]


def _plain_values(s, seq, pos, dtype):
    """K and V of the given positions as the cache holds them: [..., heads, d]."""
    page = s["case"]["page"]
    pid, off = s["table"].long()[seq, pos // page], pos % page
    k = s["k"][pid, :, off].float() * s["ks"][pid][..., None]
    v = s["v"][pid, :, :, off].float() * s["vs"][pid][..., None]
    return k.to(dtype), v.to(dtype)


def _plain_read(s):
    seq, at = _ragged(s["cu_back"], s["back"])
    return list(_plain_values(s, seq, s["first"].long()[seq] + at, torch.bfloat16))


def _plain_turn(x, weight, table, pairs):
    """Rows [tokens, heads, d] in fp32, normed where there is a weight, turned by the table's rows [tokens, rot]."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight
    rot = table.shape[1]
    c, n = table[:, None, :rot // 2], table[:, None, rot // 2:]
    a, b = (x[..., :rot:2], x[..., 1:rot:2]) if pairs else (x[..., :rot // 2], x[..., rot // 2:rot])
    y = [a * c - b * n, b * c + a * n]
    y = torch.stack(y, -1).flatten(-2) if pairs else torch.cat(y, -1)
    return torch.cat([y, x[..., rot:]], -1)


def _plain_rotary(s):
    case = s["case"]
    page, t = case["page"], s["key"].shape[0]
    table = s["cos_sin"][s["positions"]]
    query = _plain_turn(s["query"], s["qw"], table, case["pairs"])
    key = _plain_turn(s["key"], s["kw"], table, case["pairs"])
    seq, at = _ragged(s["cu"], t)
    start = s["ends"].long() - (s["cu"][1:] - s["cu"][:-1]).long()  # older tokens of each sequence
    pos = start[seq] + at
    pid = s["table"].long()[seq, pos // page]
    off = pos % page
    older = torch.zeros(s["ks"].shape[0], dtype=torch.long, device="cuda")  # older tokens of a touched page
    older[pid] = (start[seq] - pos // page * page).clamp(min=0)
    touched = torch.zeros_like(older, dtype=torch.bool)
    touched[pid] = True
    for x, codes, scale, tokens in ((key, s["k"], s["ks"], 2), (s["value"].float(), s["v"], s["vs"], 3)):
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
    return [query.to(s["query"].dtype), *_plain_read(s)]


def _bits(mask, new):
    """[rows, words] of int64 as [rows, new] truth values."""
    at = torch.arange(new, device="cuda")
    return (mask[:, at // 64] >> (at % 64) & 1).bool()


def _plain_tree(s):
    case = s["case"]
    n, rep, new = case["seqs"], case["hq"] // case["heads"], case["new"]
    q = s["q"].float().view(n, new, case["heads"], rep, -1).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [n, heads, rep * new, d]
    pos = torch.arange(s["max_len"], device="cuda")
    ends = s["ends"].long()[:, None]
    k, v = _plain_values(s, torch.arange(n, device="cuda")[:, None], torch.minimum(pos[None], ends - 1), torch.float32)
    x = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) * case["d"] ** -0.5
    x = x.view(n, case["heads"], rep, new, -1)
    at = pos[None] - (ends - new)  # a position's place among the drafts
    seen = _bits(s["mask"], new).view(n, new, new)
    seen = torch.gather(seen, 2, at.clamp(0, new - 1)[:, None].expand(-1, new, -1))
    seen = (at < 0)[:, None] | seen & (at < new)[:, None]
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e30))
    o = torch.matmul(p.flatten(2, 3), v.permute(0, 2, 1, 3).contiguous())
    o = o.view(n, case["heads"], rep, new, -1) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return o.permute(0, 3, 1, 2, 4).reshape(s["q"].shape).to(s["q"].dtype)


def _plain_keep(s):
    """All rows at once: what the pages that rows move to need, their codes again, then the rows."""
    page, table = s["case"]["page"], s["table"].long()
    seq, at = torch.nonzero(s["path"] >= 0, as_tuple=True)
    start = s["start"].long()[seq]
    there, here = start + at, start + s["path"].long()[seq, at]
    pid, src = table[seq, there // page], table[seq, here // page]
    off, src_off = there % page, here % page
    other = (pid != src)[:, None]
    for codes, scale, read in ((s["k"], s["ks"], lambda c: c[src, :, src_off]), (s["v"], s["vs"], lambda c: c[src, :, :, src_off])):
        rows, was = read(codes).float(), scale.clone()
        need = rows.abs().amax(-1).double() / 127 * was[src].double()
        now = was.index_reduce(0, pid, torch.where(other, need, 0.0).float(), "amax")
        ratio = was / now
        touched = torch.zeros(len(was), dtype=torch.bool, device="cuda").index_fill_(0, pid, True)
        codes[touched] = torch.round(codes[touched].float() * ratio[touched][:, :, None, None]).to(torch.int8)
        rows = torch.round(rows * (was[src] / now[pid])[..., None]).to(torch.int8)
        if codes is s["k"]:
            codes[pid, :, off] = rows
        else:
            codes[pid, :, :, off] = rows
        scale.copy_(now)
    return _plain_read(s)


def _plain_norm(s):
    x = s["x"].float()
    if s["inner"] is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s["inner"]
    if s["gate"] is not None:
        g = s["gate"].float()
        x = x * (1 / (1 + torch.exp(-g))) * (g if s["case"]["act"] == "silu" else 1.0)
    if s["residual"] is None:
        return x.to(s["x"].dtype)
    h = s["residual"].float() + s["case"]["scale"] * x
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * s["weight"]
    return [y.to(s["x"].dtype), h.to(s["residual"].dtype)]


# -------------------------------------------------------------------------------------------- run


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        return _own(s, s["case"])
    return {"rotary": _plain_rotary, "tree": _plain_tree, "keep": _plain_keep, "norm": _plain_norm}[op](s)


def _own(s, case):
    path = os.path.join(_ROOT, "vllm-gsqrco-exl3_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from vllm_gguf_plugin import decoder

    if case["op"] == "norm":
        if s["residual"] is None:
            return decoder.gated_norm(s["x"], s["gate"], s["inner"], act=case["act"], eps=EPS)
        return list(decoder.residual_norm(s["x"], s["residual"], s["weight"], inner_weight=s["inner"], gate=s["gate"],
                                          act=case["act"], scale=case["scale"], eps=EPS))
    cache = decoder.Kv8Cache(s["k"], s["v"], s["ks"], s["vs"])
    if case["op"] == "tree":
        return decoder.kv8_tree_attention(s["q"], cache, s["mask"], s["table"], s["ends"], s["cu"], s["max_new"], s["max_len"])
    out = []
    if case["op"] == "rotary":
        out = [decoder.kv8_rotary_append(cache, s["query"], s["key"], s["value"], s["cos_sin"], s["positions"], s["table"],
                                         s["ends"], s["cu"], s["max_new"], interleaved=case["pairs"], q_weight=s["qw"],
                                         k_weight=s["kw"], eps=EPS)]
    else:
        decoder.kv8_keep(cache, s["path"], s["table"], s["ends"], s["cu"])
    return out + list(decoder.kv8_read(cache, s["table"], s["first"], s["cu_back"], s["back"], s["max_back"], torch.bfloat16))


# --------------------------------------------------------------------- the definitions in 64 bits


def _exact_turned(x, weight, table, pairs):
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.double()
    half = table.shape[1] // 2
    z = torch.complex(table[:, :half].double(), table[:, half:].double())[:, None]
    y = x.clone()
    if pairs:
        y[..., :2 * half] = torch.view_as_real(torch.view_as_complex(x[..., :2 * half].unflatten(-1, (half, 2)).contiguous()) * z).flatten(-2)
    else:
        w = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * z
        y[..., :half], y[..., half:2 * half] = w.real, w.imag
    return y


def _exact_rotary(s):
    """Sequence by sequence and page by page: what the touched pages hold after the new tokens."""
    case = s["case"]
    page, cu, ends, first = case["page"], s["cu"].tolist(), s["ends"].tolist(), s["first"].tolist()
    turn, tables = s["cos_sin"][s["positions"]], s["table"].tolist()
    out = [_exact_turned(s["query"], s["qw"], turn, case["pairs"])]
    key = _exact_turned(s["key"], s["kw"], turn, case["pairs"])
    for x, codes, scales, turned in ((key, s["k"], s["ks"], False), (s["value"].double(), s["v"], s["vs"], True)):
        parts = []
        for i, end in enumerate(ends):
            start = end - (cu[i + 1] - cu[i])
            for p0 in range(first[i], end, page):
                pid, lo, hi = tables[i][p0 // page], max(start, p0), min(end, p0 + page)
                fresh = x[cu[i] + lo - start:cu[i] + hi - start]  # [tokens, heads, d]
                now = (fresh.abs().amax((0, 2)).float() / 127).double()
                if start > p0:
                    held = codes[pid].transpose(1, 2) if turned else codes[pid]
                    held = held[:, :start - p0].permute(1, 0, 2).double()
                    was = scales[pid].double()
                    now = torch.maximum(now, was)
                    parts.append(torch.round(held * (was / now)[:, None]) * now[:, None])
                parts.append(torch.round(fresh / now[:, None]).clamp(-127, 127) * now[:, None])
        out.append(torch.cat(parts))
    return out


def _exact_tree(s):
    case = s["case"]
    rep, cu, ends = case["hq"] // case["heads"], s["cu"].tolist(), s["ends"].tolist()
    page = case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, end in enumerate(ends):
        pids = s["table"][i, :-(-end // page)].long()
        k = (s["k"][pids].double() * s["ks"][pids].double()[..., None, None]).permute(1, 0, 2, 3).flatten(1, 2)[:, :end]
        v = (s["v"][pids].double() * s["vs"][pids].double()[..., None, None]).permute(1, 0, 3, 2).flatten(1, 2)[:, :end]
        n = cu[i + 1] - cu[i]
        words = [[w & (1 << 64) - 1 for w in r] for r in s["mask"][cu[i]:cu[i + 1]].tolist()]
        hidden = torch.tensor([[not r[j // 64] >> j % 64 & 1 for j in range(n)] for r in words], device="cuda")
        hidden = torch.cat([torch.zeros(n, end - n, dtype=torch.bool, device="cuda"), hidden], 1)
        for h in range(case["hq"]):
            x = s["q"][cu[i]:cu[i + 1], h].double() @ k[h // rep].T / math.sqrt(case["d"])
            out[cu[i]:cu[i + 1], h] = torch.softmax(x.masked_fill(hidden, -math.inf), -1) @ v[h // rep]
    return out


def _exact_keep(s):
    """Row by row, into each page's own values."""
    page, tables, both = s["case"]["page"], s["table"].tolist(), []
    paths, starts = s["path"].tolist(), s["start"].tolist()
    for codes, scales, turned in ((s["k"], s["ks"], False), (s["v"], s["vs"], True)):
        codes = (codes.transpose(2, 3) if turned else codes).cpu().double()  # [pages, heads, page, d]
        scales, parts = scales.cpu().double(), []
        for table, path, start in zip(tables, paths, starts):
            moves = [(table[(start + r) // page], (start + r) % page, table[(start + j) // page]) for j, r in enumerate(path) if r >= 0]
            rows = [codes[p, :, o] for p, o, _ in moves]
            now = {}
            for (p, _, to), row in zip(moves, rows):
                held = now.get(to, scales[to])
                now[to] = held if p == to else torch.maximum(held, row.abs().amax(-1) / 127 * scales[p])
            for (p, _, to), row in zip(moves, rows):
                step = now[to].float().double()
                parts.append(torch.round(row * (scales[p] / step)[:, None]) * step[:, None])
        both.append(torch.stack(parts).cuda())
    return both


def _exact_norm(s):
    u = s["x"].double()
    if s["inner"] is not None:
        u = u / torch.sqrt(u.square().mean(-1, keepdim=True) + EPS) * s["inner"].double()
    if s["gate"] is not None:
        act = {"silu": torch.nn.functional.silu, "sigmoid": torch.sigmoid}[s["case"]["act"]]
        u = u * act(s["gate"].double())
    if s["residual"] is None:
        return u
    h = s["residual"].double() + s["case"]["scale"] * u
    return [torch.nn.functional.rms_norm(h, (s["case"]["n"],), s["weight"].double(), EPS), h]


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "tree": _exact_tree, "keep": _exact_keep, "norm": _exact_norm}[case["op"]](s)
