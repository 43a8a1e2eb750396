"""Operators of a decoder between its GGUF linear layers, and behind its head: the 8-bit paged KV
cache, the position rotation on the way into it and its attention, also for trees of drafted tokens, block norms with
their gates and residuals, the gated delta rule (linear attention) and token log probabilities.

They are torch.ops._C_gguf.<name>, served by the HIP kernels of libgguf_decoder.so
(include/gguf_decoder.h states what each does with every argument); the functions here are the same
with defaults. Calls run on torch's current stream, never wait for the GPU and may be captured in a
CUDA graph: lengths, page tables, slots and token ids stay on the device, and the Python numbers
(max_new, max_len) only size the launch. A refused argument raises RuntimeError.

A batch of sequences is ragged: `cu_seqlens` [seqs + 1] (int32, on the device) holds each sequence's
first row.

    cache = Kv8Cache.empty(pages=512, heads=4, page=64, head_size=256)
    kv8_append(cache, k, v, block_table, seq_lens, cu_seqlens, max_new)
    y = kv8_attention(q, cache, block_table, seq_lens, cu_seqlens, max_new, max_len)
    normed, residual = residual_norm(y, residual, weight)
    q = kv8_rotary_append(cache, q, k, v, cos_sin, positions, block_table, seq_lens, cu_seqlens, max_new)
    y = kv8_tree_attention(q, cache, tree_mask, block_table, seq_lens, cu_seqlens, max_new, max_len)
    kv8_keep(cache, path, block_table, seq_lens, cu_seqlens)
    o = gated_delta_rule(q, k, v, g, beta, state, slots, cu_seqlens, max_new)
    o = gated_norm(o, gate, weight)
    logprobs, ranks, entropy, top_logprobs, top_ids = token_logprobs(logits, token_ids, top=20)
"""

from __future__ import annotations

import os
from typing import NamedTuple

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libgguf_decoder.so")
OPS_LIB = os.path.join(_HERE, "_C_gguf_decoder_ops.so")

_registered = False


def register() -> None:
    """Load the ops once per process. Raises if the native library or its op registration is not
    built: there is no fallback path."""
    global _registered
    if _registered:
        return
    for path in (LIB_PATH, OPS_LIB):
        if not os.path.exists(path):
            raise ImportError(f"{path} is not built: run vllm-gsqrco-exl3_amd/build.py "
                              "(or __graft_entry__.build())")
    torch.ops.load_library(OPS_LIB)

    @torch.library.register_fake("_C_gguf::kv8_append")
    def _(key, value, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, cu_seqlens, max_new):
        return None

    @torch.library.register_fake("_C_gguf::kv8_read")
    def _(k_cache, v_cache, k_scale, v_scale, block_table, starts, cu_seqlens, tokens, max_tokens, dtype):
        shape = (tokens, k_cache.shape[1], k_cache.shape[3])
        return k_cache.new_empty(shape, dtype=dtype), k_cache.new_empty(shape, dtype=dtype)

    @torch.library.register_fake("_C_gguf::kv8_attention")
    def _(query, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, cu_seqlens, max_new, max_len, scale):
        return query.new_empty(query.shape)

    @torch.library.register_fake("_C_gguf::kv8_tree_attention")
    def _(query, k_cache, v_cache, k_scale, v_scale, tree_mask, block_table, seq_lens, cu_seqlens, max_new, max_len, scale):
        return query.new_empty(query.shape)

    @torch.library.register_fake("_C_gguf::kv8_rotary_append")
    def _(query, key, value, k_cache, v_cache, k_scale, v_scale, cos_sin, positions, block_table, seq_lens, cu_seqlens,
          max_new, interleaved, q_weight, k_weight, eps):
        return query.new_empty(query.shape)

    @torch.library.register_fake("_C_gguf::kv8_keep")
    def _(k_cache, v_cache, k_scale, v_scale, path, block_table, seq_lens, cu_seqlens):
        return None

    @torch.library.register_fake("_C_gguf::residual_norm")
    def _(x, residual, gate, act, inner_weight, weight, scale, eps):
        return (x.new_empty(x.shape if weight is not None else (0,)),
                x.new_empty(x.shape, dtype=x.dtype if residual is None else residual.dtype))

    @torch.library.register_fake("_C_gguf::gated_delta_rule")
    def _(q, k, v, g, beta, state, slots, cu_seqlens, max_new, out_slots, scale, l2norm):
        return v.new_empty(v.shape)

    @torch.library.register_fake("_C_gguf::token_logprobs")
    def _(logits, token_ids, top):
        n = logits.shape[0]
        return (logits.new_empty(n, dtype=torch.float32), logits.new_empty(n, dtype=torch.int32),
                logits.new_empty(n, dtype=torch.float32), logits.new_empty((n, top), dtype=torch.float32),
                logits.new_empty((n, top), dtype=torch.int32))

    _registered = True


register()
_ops = torch.ops._C_gguf


class Kv8Cache(NamedTuple):
    """A paged KV cache in 8 bits: codes k [pages, heads, page, head_size] and v [pages, heads,
    head_size, page] (int8), and one fp32 scale for each (page, head) of either."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    @classmethod
    def empty(cls, pages: int, heads: int, page: int, head_size: int, device="cuda") -> "Kv8Cache":
        """A cache of `pages` pages of `page` tokens (a multiple of 16); head_size 64, 128, 192 or 256."""
        def codes(*shape):
            return torch.zeros(*shape, dtype=torch.int8, device=device)

        return cls(codes(pages, heads, page, head_size), codes(pages, heads, head_size, page),
                   torch.zeros(pages, heads, device=device), torch.zeros(pages, heads, device=device))


def kv8_append(cache: Kv8Cache, key, value, block_table, seq_lens, cu_seqlens, max_new: int) -> None:
    """Write the rows of key and value [tokens, heads, head_size] (fp32, fp16 or bf16) as the last
    positions of their sequences: sequence s, of seq_lens[s] tokens with them, lies in the pages
    block_table[s]. A (page, head)'s scale grows where new values need it, and the page's older codes
    are then rounded to it. max_new: the most rows of a sequence."""
    _ops.kv8_append(key, value, *cache, block_table, seq_lens, cu_seqlens, max_new)


def kv8_read(cache: Kv8Cache, block_table, starts, cu_seqlens, tokens: int, max_tokens: int,
             dtype=torch.bfloat16):
    """The cached keys and values of positions starts[s] on, as many as cu_seqlens has rows for the
    sequence (`tokens` in all, at most max_tokens of one): two [tokens, heads, head_size] of dtype."""
    return _ops.kv8_read(*cache, block_table, starts, cu_seqlens, tokens, max_tokens, dtype)


def kv8_attention(query, cache: Kv8Cache, block_table, seq_lens, cu_seqlens, max_new: int, max_len: int,
                  scale: float | None = None):
    """Causal attention of query [tokens, q_heads, head_size] (fp16 or bf16), the last rows of their
    sequences, over the cache that holds their own keys already. scale: 1 / sqrt(head_size) unless given.
    max_new, max_len: the most rows and the longest seq_lens of a sequence."""
    if scale is None:
        scale = query.shape[-1] ** -0.5
    return _ops.kv8_attention(query, *cache, block_table, seq_lens, cu_seqlens, max_new, max_len, scale)


def kv8_rotary_append(cache: Kv8Cache, query, key, value, cos_sin, positions, block_table, seq_lens, cu_seqlens,
                      max_new: int, interleaved: bool = False, q_weight=None, k_weight=None, eps: float = 1e-6):
    """kv8_append of the keys turned by their positions, and the queries [tokens, q_heads, head_size] turned: returned in their
    dtype. cos_sin fp32 [positions, r] holds the cosines and then the sines of r / 2 angles a position; dims i and i + r / 2
    of a head turn together (interleaved: 2i and 2i + 1), those from r on stay. positions int64 [tokens]: a draft's is
    its depth's. q_weight, k_weight fp32 [head_size]: the heads are normed by their root mean square first."""
    return _ops.kv8_rotary_append(query, key, value, *cache, cos_sin, positions, block_table, seq_lens, cu_seqlens, max_new,
                                  interleaved, q_weight, k_weight, eps)


def tree_mask(parents):
    """The int64 [tokens, words] mask of kv8_tree_attention, on the host, for a batch of trees: each a list of its rows' parents (row
    numbers before the row's own, -1 for none). A row sees itself and its ancestors."""
    words = max(1, -(-max((len(t) for t in parents), default=0) // 64))
    out = []
    for tree in parents:
        rows = []
        for i, p in enumerate(tree):
            if not -1 <= p < i:
                raise ValueError(f"row {i} cannot have parent {p}")
            rows.append((rows[p] if p >= 0 else 0) | 1 << i)
        for r in rows:
            w = [r >> 64 * j & (1 << 64) - 1 for j in range(words)]
            out.append([x - (1 << 64) if x >> 63 else x for x in w])
    return torch.tensor(out, dtype=torch.int64).view(-1, words)


def kv8_tree_attention(query, cache: Kv8Cache, tree_mask, block_table, seq_lens, cu_seqlens, max_new: int, max_len: int,
                       scale: float | None = None):
    """Attention of a tree of drafts, query [tokens, q_heads, head_size] (fp16 or bf16): a row sees all of its sequence's
    positions before the sequence's own rows, and of these row j where bit j % 64 of tree_mask[row, j // 64] is set. The
    cache holds the drafts' keys and values as the sequence's last positions, in the rows' order."""
    if scale is None:
        scale = query.shape[-1] ** -0.5
    return _ops.kv8_tree_attention(query, *cache, tree_mask, block_table, seq_lens, cu_seqlens, max_new, max_len, scale)


def kv8_keep(cache: Kv8Cache, path, block_table, seq_lens, cu_seqlens) -> None:
    """Move row path[s, j] (int32 [seqs, m]) of each sequence's last rows, its drafts, to their j-th place in the cache: a
    path grows strictly and ends at its first entry that does not (or is out of range, as -1). The arguments are those the drafts were
    appended with; afterwards the sequence is as long as its older tokens and the path."""
    _ops.kv8_keep(*cache, path, block_table, seq_lens, cu_seqlens)


_ACTS = {"none": 0, "sigmoid": 1, "silu": 2}


def residual_norm(x, residual=None, weight=None, *, inner_weight=None, gate=None, act: str = "none", scale: float = 1.0,
                  eps: float = 1e-6):
    """Norms before and after a block with its gate and residual, over the last dimension of x [rows, n] or [rows, heads, n]:
        u = x, normed by inner_weight, times act(gate);  h = residual + scale * u;  out = h, normed by weight
    with RMS norms (weights fp32 [n]); every part may be missing. act: "none" (the gate itself), "sigmoid" or "silu" of a gate like x;
    without a gate it does nothing. Returns (out, h): out in x's dtype (None without weight), h in residual's (x's dtype or fp32)."""
    if act not in _ACTS:
        raise RuntimeError(f"residual_norm: act={act!r} is not one of {', '.join(_ACTS)}")
    out, hidden = _ops.residual_norm(x, residual, gate, _ACTS[act], inner_weight, weight, scale, eps)
    return (None if weight is None else out), hidden


def gated_norm(x, gate, weight, *, act: str = "silu", eps: float = 1e-6):
    """x [rows, n] or [rows, heads, n] normed over its last dimension by weight (fp32 [n]), times act(gate): the norm behind
    linear attention's heads."""
    return residual_norm(x, inner_weight=weight, gate=gate, act=act, eps=eps)[1]


def gated_delta_rule(q, k, v, g, beta, state, slots, cu_seqlens, max_new: int, out_slots=None,
                     scale: float | None = None, l2norm: bool = True):
    """Linear attention with the gated delta rule: q, k [tokens, hk, dk], v [tokens, hv, dv] (fp32, fp16
    or bf16), g (log decay) and beta fp32 [tokens, hv]; returns [tokens, hv, dv]. state fp32 [slots, hv,
    dv, dk]: sequence s starts from state[slots[s]] (from zero where that is -1) and its last state goes
    to out_slots[s], or with a two-dimensional out_slots [seqs, m] the states after each of its first m tokens
    do (-1: not kept); without out_slots, back to slots[s]. scale: 1 / sqrt(dk) unless given; l2norm: q and
    k are divided by their norms first. max_new: the most rows of a sequence."""
    if scale is None:
        scale = q.shape[-1] ** -0.5
    return _ops.gated_delta_rule(q, k, v, g, beta, state, slots, cu_seqlens, max_new, out_slots, scale, l2norm)


def token_logprobs(logits, token_ids, top: int = 0):
    """For each row of logits [rows, vocab]: the log probability of token_ids[row] (int64) and its rank
    (1: the most likely), the distribution's entropy, and the `top` most likely tokens' log probabilities
    and ids, equal ones by index: (fp32 [rows], int32 [rows], fp32 [rows], fp32 [rows, top], int32 [rows, top])."""
    return _ops.token_logprobs(logits, token_ids, top)
