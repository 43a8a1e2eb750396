"""Operators of a decoder between its GGUF linear layers, and behind its head: the 8-bit paged KV
cache and its attention, the gated delta rule (linear attention) and token log probabilities.

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
    o = gated_delta_rule(q, k, v, g, beta, state, slots, cu_seqlens, max_new)
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
