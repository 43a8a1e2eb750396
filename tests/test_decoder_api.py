"""libgguf_decoder.so exports what include/gguf_decoder.h declares and nothing else, and the decoder
operators (vllm_gguf_plugin.decoder) refuse what they cannot take, with a message, before any GPU
access: the checks run on host tensors here, where a call that passes them all ends with "must be
CUDA tensors"."""

import ctypes
import os
import re
import subprocess

import pytest
import torch

from conftest import ROOT

from vllm_gguf_plugin import decoder


def _declared():
    src = open(os.path.join(ROOT, "include", "gguf_decoder.h")).read()
    return sorted(set(re.findall(r"GGUF_DEC_API\s+[\w\s\*]+?\b(gguf_\w+)\s*\(", src)))


def test_exports_are_the_header():
    names = _declared()
    assert {"gguf_kv8_append", "gguf_kv8_read", "gguf_kv8_attention", "gguf_gated_delta_rule", "gguf_token_logprobs",
            "gguf_decoder_last_error"} <= set(names)
    lib = ctypes.CDLL(decoder.LIB_PATH)
    for name in names:
        assert hasattr(lib, name), name
    out = subprocess.run(["nm", "-D", "--defined-only", decoder.LIB_PATH], capture_output=True, text=True).stdout
    assert {l.split()[-1] for l in out.splitlines() if " T " in l} == set(names)


def _cache(pages=4, heads=2, page=16, d=64, **change):
    c = decoder.Kv8Cache.empty(pages, heads, page, d, device="cpu")
    return c._replace(**change)


def _ints(*v):
    return torch.tensor(v, dtype=torch.int32)


def _kv(**change):
    a = dict(cache=_cache(), key=torch.zeros(3, 2, 64), value=torch.zeros(3, 2, 64),
             block_table=torch.zeros(2, 2, dtype=torch.int32), seq_lens=_ints(5, 6), cu_seqlens=_ints(0, 1, 3), max_new=2)
    a.update(change)
    return decoder.kv8_append(a["cache"], a["key"], a["value"], a["block_table"], a["seq_lens"], a["cu_seqlens"], a["max_new"])


def _read(**change):
    a = dict(cache=_cache(), block_table=torch.zeros(2, 2, dtype=torch.int32), starts=_ints(0, 0),
             cu_seqlens=_ints(0, 1, 3), tokens=3, max_tokens=2, dtype=torch.float16)
    a.update(change)
    return decoder.kv8_read(**a)


def _attention(**change):
    a = dict(query=torch.zeros(3, 4, 64, dtype=torch.float16), cache=_cache(),
             block_table=torch.zeros(2, 2, dtype=torch.int32), seq_lens=_ints(5, 6), cu_seqlens=_ints(0, 1, 3), max_new=2,
             max_len=6, scale=None)
    a.update(change)
    return decoder.kv8_attention(**a)


def _delta(**change):
    a = dict(q=torch.zeros(3, 2, 64), k=torch.zeros(3, 2, 64), v=torch.zeros(3, 4, 32), g=torch.zeros(3, 4),
             beta=torch.zeros(3, 4), state=torch.zeros(5, 4, 32, 64), slots=_ints(0, 1), cu_seqlens=_ints(0, 1, 3),
             max_new=2, out_slots=None)
    a.update(change)
    return decoder.gated_delta_rule(**a)


def _logprobs(**change):
    a = dict(logits=torch.zeros(3, 100), token_ids=torch.zeros(3, dtype=torch.int64), top=5)
    a.update(change)
    return decoder.token_logprobs(**a)


@pytest.mark.parametrize("call", [_kv, _read, _attention, _delta, _logprobs], ids=lambda f: f.__name__)
def test_host_tensors_pass_the_checks_and_are_refused(call):
    with pytest.raises(RuntimeError, match="must be CUDA tensors"):
        call()


BAD_CACHES = [
    (dict(k=torch.zeros(4, 2, 16, 64)), "must be int8"),
    (dict(k_scale=torch.zeros(4, 2, dtype=torch.float16)), "must be fp32"),
    (dict(k=torch.zeros(4, 2, 24, 64, dtype=torch.int8)), "multiple of 16"),
    (dict(k=torch.zeros(4, 2, 16, 80, dtype=torch.int8)), "head size 80"),
    (dict(v=torch.zeros(4, 2, 16, 64, dtype=torch.int8)), "head size, page"),
    (dict(v_scale=torch.zeros(4, 1)), r"\[pages, heads\]"),
    (dict(k=torch.zeros(4, 2, 16, 128, dtype=torch.int8)[..., :64]), "contiguous"),
    (dict(k=torch.zeros(4 * 2 * 16 * 64 + 8, dtype=torch.int8)[8:].view(4, 2, 16, 64)[:]), None),
    (dict(k_scale=torch.zeros(8)), "4 dimensions"),
]


@pytest.mark.parametrize("change,message", BAD_CACHES, ids=range(len(BAD_CACHES)))
@pytest.mark.parametrize("call", [_kv, _read, _attention], ids=lambda f: f.__name__)
def test_caches_refused(call, change, message):
    c = _cache(**change)
    if message is None:  # 8 bytes past a 16-byte boundary
        assert c.k.data_ptr() % 16 == 8
        message = "16-byte aligned"
    with pytest.raises(RuntimeError, match=message):
        call(cache=c)


@pytest.mark.parametrize("call", [_kv, _read, _attention], ids=lambda f: f.__name__)
@pytest.mark.parametrize("change,message", [
    (dict(block_table=torch.zeros(3, 2, dtype=torch.int32)), "block_table"),
    (dict(block_table=torch.zeros(2, 2, dtype=torch.int64)), "block_table"),
    (dict(block_table=torch.zeros(2, 0, dtype=torch.int32)), "no pages"),
    (dict(block_table=torch.zeros(2, 4, dtype=torch.int32)[:, ::2]), "unit inner stride"),
    (dict(cu_seqlens=torch.zeros(3, dtype=torch.int64)), "cu_seqlens"),
    (dict(cu_seqlens=_ints(0)), "cu_seqlens"),
    (dict(cu_seqlens=torch.zeros(6, dtype=torch.int32)[::2]), "cu_seqlens"),
])
def test_tables_refused(call, change, message):
    with pytest.raises(RuntimeError, match=message):
        call(**change)


@pytest.mark.parametrize("change,message", [
    (dict(key=torch.zeros(3, 2, 64, dtype=torch.float64)), "float dtype"),
    (dict(value=torch.zeros(3, 2, 64, dtype=torch.bfloat16)), "share one float dtype"),
    (dict(value=torch.zeros(2, 2, 64)), r"\[tokens, 2, 64\]"),
    (dict(key=torch.zeros(3, 1, 64)), r"\[tokens, 2, 64\]"),
    (dict(key=torch.zeros(3, 2, 128)[..., ::2]), "unit inner stride"),
    (dict(key=torch.zeros(3, 2, 66)[..., :64]), "16-byte aligned rows"),
    (dict(seq_lens=_ints(1)), "seq_lens"),
    (dict(max_new=-1), "max_new"),
])
def test_append_refused(change, message):
    with pytest.raises(RuntimeError, match=message):
        _kv(**change)


@pytest.mark.parametrize("change,message", [
    (dict(starts=_ints(0)), "starts"), (dict(dtype=torch.int32), "float dtype"), (dict(max_tokens=-1), "max_tokens"),
    (dict(tokens=-1), "number of tokens")])
def test_read_refused(change, message):
    with pytest.raises(RuntimeError, match=message):
        _read(**change)


@pytest.mark.parametrize("change,message", [
    (dict(query=torch.zeros(3, 4, 64)), "fp16 or bf16"),
    (dict(query=torch.zeros(3, 4, 128, dtype=torch.float16)), "head size"),
    (dict(query=torch.zeros(3, 3, 64, dtype=torch.float16)), "no multiple"),
    (dict(query=torch.zeros(3, 4, 128, dtype=torch.float16)[..., ::2]), "unit inner stride"),
    (dict(query=torch.zeros(4, 64, dtype=torch.float16)), "query and out"),
    (dict(seq_lens=torch.zeros(2, dtype=torch.int64)), "seq_lens"),
    (dict(max_new=-1), "max_new"), (dict(max_len=-1), "max_len"),
    (dict(scale=float("nan")), "scale"),
])
def test_attention_refused(change, message):
    with pytest.raises(RuntimeError, match=message):
        _attention(**change)


@pytest.mark.parametrize("change,message", [
    (dict(q=torch.zeros(3, 2, 64, dtype=torch.float16)), "share one float dtype"),
    (dict(k=torch.zeros(3, 1, 64)), "one shape"),
    (dict(v=torch.zeros(2, 4, 32)), "as many tokens"),
    (dict(q=torch.zeros(3, 2, 96), k=torch.zeros(3, 2, 96)), "key head size 96"),
    (dict(v=torch.zeros(3, 4, 24), state=torch.zeros(5, 4, 24, 64)), "value head size 24"),
    (dict(v=torch.zeros(3, 3, 32)), "no multiple"),
    (dict(v=torch.empty(2 * (1 << 23) + 128, dtype=torch.float32).as_strided((3, 4, 32), (1 << 23, 32, 1))), "2.22"),
    (dict(v=torch.zeros(3, 4, 33)[..., :32]), "16-byte aligned rows"),
    (dict(g=torch.zeros(3, 4, dtype=torch.bfloat16)), "g and beta"),
    (dict(beta=torch.zeros(3, 8)[:, ::2]), "g and beta"),
    (dict(state=torch.zeros(5, 4, 64, 32)), "state"),
    (dict(state=torch.zeros(5, 4, 32, 64, dtype=torch.bfloat16)), "state"),
    (dict(state=torch.zeros(5, 4, 32, 128)[..., :64]), "state"),
    (dict(slots=_ints(0)), "slots"),
    (dict(out_slots=_ints(0)), "out_slots"),
    (dict(out_slots=torch.zeros(2, 0, dtype=torch.int32)), "out_slots"),
    (dict(cu_seqlens=_ints(0)), "cu_seqlens"),
    (dict(max_new=-1), "max_new"),
    (dict(scale=float("inf")), "scale"),
])
def test_delta_refused(change, message):
    with pytest.raises(RuntimeError, match=message):
        _delta(**change)


@pytest.mark.parametrize("change,message", [
    (dict(logits=torch.zeros(3, 100, dtype=torch.int32)), "float"),
    (dict(logits=torch.zeros(100)), r"\[rows, vocab\]"),
    (dict(logits=torch.zeros(3, 200)[:, ::2]), "unit inner stride"),
    (dict(logits=torch.zeros(3, 0)), "no columns"),
    (dict(token_ids=torch.zeros(3, dtype=torch.int32)), "token_ids"),
    (dict(token_ids=torch.zeros(2, dtype=torch.int64)), "token_ids"),
    (dict(top=65), "top=65"), (dict(top=-1), "top"),
    (dict(logits=torch.zeros(3, 4)), "top=5"),
])
def test_logprobs_refused(change, message):
    with pytest.raises(RuntimeError, match=message):
        _logprobs(**change)


def test_fake_implementations_have_the_ops_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        def empty(*shape, dtype=torch.float16):
            return torch.empty(*shape, dtype=dtype)

        i32 = torch.int32
        c = decoder.Kv8Cache(empty(4, 2, 16, 64, dtype=torch.int8), empty(4, 2, 64, 16, dtype=torch.int8),
                             empty(4, 2, dtype=torch.float32), empty(4, 2, dtype=torch.float32))
        table, lens, cu = empty(2, 2, dtype=i32), empty(2, dtype=i32), empty(3, dtype=i32)
        y = decoder.kv8_attention(empty(3, 4, 64), c, table, lens, cu, 2, 6)
        assert y.shape == (3, 4, 64) and y.dtype == torch.float16
        k, v = decoder.kv8_read(c, table, lens, cu, 3, 2)
        assert k.shape == v.shape == (3, 2, 64) and k.dtype == torch.bfloat16
        assert decoder.kv8_append(c, empty(3, 2, 64), empty(3, 2, 64), table, lens, cu, 2) is None
        f32 = torch.float32
        o = decoder.gated_delta_rule(empty(3, 2, 64), empty(3, 2, 64), empty(3, 4, 32), empty(3, 4, dtype=f32),
                                     empty(3, 4, dtype=f32), empty(5, 4, 32, 64, dtype=f32), lens, cu, 2)
        assert o.shape == (3, 4, 32)
        out = decoder.token_logprobs(empty(3, 100), empty(3, dtype=torch.int64), 7)
        assert [tuple(x.shape) for x in out] == [(3,), (3,), (3,), (3, 7), (3, 7)]


class _T(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("dtype", ctypes.c_int32), ("ndim", ctypes.c_int32),
                ("size", ctypes.c_int64 * 4), ("stride", ctypes.c_int64 * 4), ("device", ctypes.c_int32)]


class _CacheT(ctypes.Structure):
    _fields_ = [("k", _T), ("v", _T), ("k_scale", _T), ("v_scale", _T)]


_CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.int8: 5, torch.int32: 6, torch.int64: 7}


def _desc(t):
    r = _T(t.data_ptr(), _CODES[t.dtype], t.dim())
    r.size[:t.dim()], r.stride[:t.dim()], r.device = list(t.shape), list(t.stride()), -1
    return r


@pytest.mark.parametrize("hint", [2 ** 62, 2 ** 63 - 1])
def test_hints_beyond_every_size_are_no_trouble(hint):
    """max_new, max_len and max_tokens may be any number: what the tensors hold bounds them before any arithmetic."""
    c = _cache()
    for call in (lambda: _kv(max_new=hint), lambda: _read(max_tokens=hint), lambda: _attention(max_new=hint, max_len=hint),
                 lambda: _attention(query=torch.zeros(3, 8, 64, dtype=torch.float16), max_new=hint, max_len=6),
                 lambda: _delta(max_new=hint)):
        with pytest.raises(RuntimeError, match="must be CUDA tensors"):
            call()

    lib = ctypes.CDLL(decoder.LIB_PATH)
    lib.gguf_kv8_attention_workspace_bytes.restype = ctypes.c_size_t
    cache = _CacheT(*(_desc(t) for t in c))
    q = _desc(torch.zeros(3, 8, 64, dtype=torch.float16))

    def workspace(max_new, max_len):
        return lib.gguf_kv8_attention_workspace_bytes(ctypes.byref(cache), ctypes.byref(q), ctypes.c_int64(2),
                                                      ctypes.c_int64(max_new), ctypes.c_int64(max_len))

    assert workspace(hint, 6) == workspace(3, 6)
    assert 0 < workspace(hint, hint) == workspace(3, 2 ** 31 - 1)


def test_tensors_without_memory_are_refused():
    """A C caller's NULL where a tensor has elements: an error, for each tensor of each entry point."""
    lib = ctypes.CDLL(decoder.LIB_PATH)
    lib.gguf_decoder_last_error.restype = ctypes.c_char_p
    i64, f32, P, null = ctypes.c_int64, ctypes.c_float, ctypes.byref, ctypes.c_void_p(None)
    c = _cache()
    table, lens, cu, rows = torch.zeros(2, 2, dtype=torch.int32), _ints(5, 6), _ints(0, 1, 3), torch.zeros(3, 2, 64)
    half, state = torch.zeros(3, 4, 64, dtype=torch.float16), torch.zeros(5, 4, 32, 64)
    v, gate, ids = torch.zeros(3, 4, 32), torch.zeros(3, 4), torch.zeros(3, dtype=torch.int64)
    f, i, ft, it = (torch.zeros(3, *s, dtype=d) for s, d in (((), torch.float32), ((), torch.int32), ((5,), torch.float32),
                                                             ((5,), torch.int32)))
    ws = torch.zeros(1 << 20, dtype=torch.uint8)
    room = (ctypes.c_void_p(ws.data_ptr() + -ws.data_ptr() % 16), ctypes.c_size_t((1 << 20) - 16), null)
    calls = {
        "kv8_append": (["cache", rows, rows, table, lens, cu], lambda a: (*a, i64(2), null)),
        "kv8_read": (["cache", table, lens, cu, rows, rows], lambda a: (*a[:4], i64(2), *a[4:], null)),
        "kv8_attention": ([half, "cache", table, lens, cu, half],
                          lambda a: (*a[:5], i64(2), i64(6), f32(1), a[5], *room)),
        "gated_delta_rule": ([rows, rows, v, gate, gate, state, lens, lens, cu, v],
                             lambda a: (*a[:9], i64(2), f32(1), 1, a[9], *room)),
        "token_logprobs": ([torch.zeros(3, 100), ids, f, i, f, ft, it], lambda a: (*a[:2], i64(5), *a[2:], *room)),
    }
    for name, (tensors, order) in calls.items():
        call = getattr(lib, "gguf_" + name)
        for spoil in range(-1, len(tensors)):
            for part in range(4 if spoil >= 0 and isinstance(tensors[spoil], str) else 1):
                descs = [_CacheT(*map(_desc, c)) if isinstance(t, str) else _desc(t) for t in tensors]
                if spoil >= 0:
                    d = descs[spoil]
                    (d if isinstance(d, _T) else getattr(d, ("k", "v", "k_scale", "v_scale")[part])).data = None
                assert call(*order([P(d) for d in descs])) == 1
                message = lib.gguf_decoder_last_error().decode()
                assert ("must be CUDA tensors" if spoil < 0 else "no data") in message, (name, spoil, part, message)


def test_no_rows_need_no_memory():
    """Tensors without elements may have no memory: the checks end where those of other host tensors do."""
    for call in (lambda: _kv(key=torch.zeros(0, 2, 64), value=torch.zeros(0, 2, 64)), lambda: _read(tokens=0),
                 lambda: _attention(query=torch.zeros(0, 4, 64, dtype=torch.float16)),
                 lambda: _logprobs(logits=torch.zeros(0, 100), token_ids=torch.zeros(0, dtype=torch.int64)),
                 lambda: _logprobs(top=0)):
        with pytest.raises(RuntimeError, match="must be CUDA tensors"):
            call()
