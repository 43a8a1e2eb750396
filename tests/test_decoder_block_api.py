"""The decoder operators of an attention block (kv8_rotary_append, kv8_tree_attention, kv8_keep, residual_norm and gated_norm)
refuse what they cannot take, with a message, before any GPU access: host tensors here, where a call that passes all
checks ends with "must be CUDA tensors". And the mask of a batch of trees, which is made on the host."""

import ctypes
import random

import pytest
import torch

from test_decoder_api import _cache, _CacheT, _desc, _ints, _T

from vllm_gguf_plugin import decoder

BF16, F16, F64, I32, I64 = torch.bfloat16, torch.float16, torch.float64, torch.int32, torch.int64


def _rotary(**change):
    a = dict(cache=_cache(), query=torch.zeros(3, 4, 64), key=torch.zeros(3, 2, 64), value=torch.zeros(3, 2, 64),
             cos_sin=torch.zeros(9, 32), positions=torch.zeros(3, dtype=I64), block_table=torch.zeros(2, 2, dtype=I32),
             seq_lens=_ints(5, 6), cu_seqlens=_ints(0, 1, 3), max_new=2)
    a.update(change)
    return decoder.kv8_rotary_append(**a)


def _tree(**change):
    a = dict(query=torch.zeros(3, 4, 64, dtype=F16), cache=_cache(), tree_mask=torch.zeros(3, 1, dtype=I64),
             block_table=torch.zeros(2, 2, dtype=I32), seq_lens=_ints(5, 6), cu_seqlens=_ints(0, 1, 3), max_new=2, max_len=6)
    a.update(change)
    return decoder.kv8_tree_attention(**a)


def _keep(**change):
    a = dict(cache=_cache(), path=torch.zeros(2, 4, dtype=I32), block_table=torch.zeros(2, 2, dtype=I32), seq_lens=_ints(5, 6),
             cu_seqlens=_ints(0, 1, 3))
    a.update(change)
    return decoder.kv8_keep(**a)


def _norm(**change):
    a = dict(x=torch.zeros(3, 40), residual=torch.zeros(3, 40), weight=torch.zeros(40), inner_weight=torch.zeros(40),
             gate=torch.zeros(3, 40), act="silu")
    a.update(change)
    return decoder.residual_norm(**a)


CALLS = [_rotary, _tree, _keep, _norm]


@pytest.mark.parametrize("call", CALLS, ids=lambda f: f.__name__)
def test_host_tensors_pass_the_checks_and_are_refused(call):
    with pytest.raises(RuntimeError, match="must be CUDA tensors"):
        call()


@pytest.mark.parametrize("call,change", [
    (_rotary, dict(q_weight=torch.zeros(64), k_weight=torch.zeros(64), interleaved=True, eps=0.0)),
    (_rotary, dict(cos_sin=torch.zeros(1, 64))), (_rotary, dict(max_new=2 ** 62)),
    (_rotary, dict(query=torch.zeros(0, 4, 64), key=torch.zeros(0, 2, 64), value=torch.zeros(0, 2, 64), positions=torch.zeros(0, dtype=I64))),
    (_tree, dict(tree_mask=torch.zeros(3, 7, dtype=I64))), (_tree, dict(tree_mask=torch.zeros(1, 1, dtype=I64).expand(3, 1))),
    (_tree, dict(max_new=2 ** 62, max_len=2 ** 63 - 1)), (_keep, dict(path=torch.zeros(2, 0, dtype=I32))),
    (_keep, dict(path=torch.zeros(2, 1024, dtype=I32))), (_norm, dict(weight=None)), (_norm, dict(residual=None, gate=None, inner_weight=None)),
    (_norm, dict(x=torch.zeros(3, 40, dtype=BF16), gate=torch.zeros(1, 40, dtype=BF16).expand(3, 40))),
    (_norm, dict(x=torch.zeros(0, 40), residual=torch.zeros(0, 40), gate=None)), (_norm, dict(act="none")),
    (lambda **c: decoder.gated_norm(torch.zeros(3, 5, 40), torch.zeros(3, 9, 40)[:, :5], torch.zeros(40), **c), {}),
], ids=range(15))
def test_allowed(call, change):
    with pytest.raises(RuntimeError, match="must be CUDA tensors"):
        call(**change)


@pytest.mark.parametrize("call", CALLS[:3], ids=lambda f: f.__name__)
@pytest.mark.parametrize("change,message", [
    (dict(block_table=torch.zeros(3, 2, dtype=I32)), "block_table"), (dict(block_table=torch.zeros(2, 2, dtype=I64)), "block_table"),
    (dict(block_table=torch.zeros(2, 0, dtype=I32)), "no pages"), (dict(cu_seqlens=torch.zeros(3, dtype=I64)), "cu_seqlens"),
    (dict(cu_seqlens=_ints(0)), "cu_seqlens"), (dict(seq_lens=_ints(1)), "seq_lens"), (dict(seq_lens=torch.zeros(2)), "seq_lens"),
    (dict(cache=_cache(k=torch.zeros(4, 2, 24, 64, dtype=torch.int8))), "multiple of 16"),
    (dict(cache=_cache(v=torch.zeros(4, 2, 16, 64, dtype=torch.int8))), "head size, page"),
    (dict(cache=_cache(k_scale=torch.zeros(4, 2, dtype=F16))), "must be fp32"),
])
def test_caches_and_tables_refused(call, change, message):
    with pytest.raises(RuntimeError, match=message):
        call(**change)


@pytest.mark.parametrize("change,message", [
    (dict(query=torch.zeros(3, 4, 64, dtype=F16)), "share one float dtype"),
    (dict(key=torch.zeros(3, 2, 64, dtype=F64)), "share one float dtype"),
    (dict(key=torch.zeros(3, 1, 64)), r"\[tokens, 2, 64\]"), (dict(value=torch.zeros(2, 2, 64)), r"\[tokens, 2, 64\]"),
    (dict(query=torch.zeros(2, 4, 64)), "query must be"), (dict(query=torch.zeros(3, 0, 64)), "query must be"),
    (dict(query=torch.zeros(3, 4, 128)), "query must be"), (dict(query=torch.zeros(3, 64)), "query, key and value"),
    (dict(query=torch.zeros(3, 4, 128)[..., ::2]), "unit inner stride"), (dict(key=torch.zeros(3, 2, 66)[..., :64]), "16-byte aligned rows"),
    (dict(cos_sin=torch.zeros(9, 24)), "cos_sin"), (dict(cos_sin=torch.zeros(9, 80)), "cos_sin"), (dict(cos_sin=torch.zeros(0, 32)), "cos_sin"),
    (dict(cos_sin=torch.zeros(9, 32, dtype=BF16)), "cos_sin"), (dict(cos_sin=torch.zeros(9, 33)[:, :32]), "cos_sin"),
    (dict(cos_sin=torch.zeros(9, 64)[:, ::2]), "cos_sin"), (dict(positions=torch.zeros(3, dtype=I32)), "positions"),
    (dict(positions=torch.zeros(2, dtype=I64)), "positions"), (dict(positions=torch.zeros(6, dtype=I64)[::2]), "positions"),
    (dict(q_weight=torch.zeros(64, dtype=BF16)), "q_weight"), (dict(k_weight=torch.zeros(32)), "q_weight and k_weight"),
    (dict(k_weight=torch.zeros(65)[1:]), "16-byte aligned"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(max_new=-1), "max_new"),
])
def test_rotary_refused(change, message):
    with pytest.raises(RuntimeError, match=message):
        _rotary(**change)


@pytest.mark.parametrize("change,message", [
    (dict(query=torch.zeros(3, 4, 64)), "fp16 or bf16"), (dict(query=torch.zeros(3, 3, 64, dtype=F16)), "no multiple"),
    (dict(tree_mask=torch.zeros(3, 1, dtype=I32)), "tree_mask"), (dict(tree_mask=torch.zeros(2, 1, dtype=I64)), "tree_mask"),
    (dict(tree_mask=torch.zeros(3, dtype=I64)), "tree_mask"), (dict(tree_mask=torch.zeros(3, 0, dtype=I64)), "tree_mask"),
    (dict(tree_mask=torch.zeros(3, 4, dtype=I64)[:, ::2]), "tree_mask"), (dict(max_len=-1), "max_len"), (dict(scale=float("inf")), "scale"),
])
def test_tree_attention_refused(change, message):
    with pytest.raises(RuntimeError, match=message):
        _tree(**change)


@pytest.mark.parametrize("change,message", [
    (dict(path=torch.zeros(2, 4, dtype=I64)), "path"), (dict(path=torch.zeros(3, 4, dtype=I32)), "path"),
    (dict(path=torch.zeros(4, dtype=I32)), "path"), (dict(path=torch.zeros(2, 8, dtype=I32)[:, ::2]), "path"),
    (dict(path=torch.zeros(2, 1025, dtype=I32)), "longer than 1024"),
])
def test_keep_refused(change, message):
    with pytest.raises(RuntimeError, match=message):
        _keep(**change)


@pytest.mark.parametrize("change,message", [
    (dict(x=torch.zeros(3, 40, dtype=I32)), "float"), (dict(x=torch.zeros(40)), "x must be"), (dict(x=torch.zeros(3, 0)), "no columns"),
    (dict(x=torch.zeros(3, 80)[:, ::2]), "unit inner stride"), (dict(residual=torch.zeros(3, 41)), "residual"),
    (dict(residual=torch.zeros(3, 40, dtype=BF16)), "residual"), (dict(residual=torch.zeros(1, 3, 40)), "residual"),
    (dict(gate=torch.zeros(3, 40, dtype=BF16)), "gate"), (dict(gate=torch.zeros(2, 40)), "gate"),
    (dict(weight=torch.zeros(40, dtype=BF16)), "weights"), (dict(inner_weight=torch.zeros(39)), "weights"),
    (dict(weight=torch.zeros(80)[::2]), "weights"), (dict(act="gelu"), "gelu"), (dict(eps=-1e-6), "eps"), (dict(scale=float("nan")), "scale"),
])
def test_norm_refused(change, message):
    with pytest.raises(RuntimeError, match=message):
        _norm(**change)


def test_fake_implementations_have_the_ops_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        def empty(*shape, dtype=F16):
            return torch.empty(*shape, dtype=dtype)

        f32 = torch.float32
        c = decoder.Kv8Cache(empty(4, 2, 16, 64, dtype=torch.int8), empty(4, 2, 64, 16, dtype=torch.int8), empty(4, 2, dtype=f32),
                             empty(4, 2, dtype=f32))
        table, lens, cu = empty(2, 2, dtype=I32), empty(2, dtype=I32), empty(3, dtype=I32)
        q = decoder.kv8_rotary_append(c, empty(3, 4, 64), empty(3, 2, 64), empty(3, 2, 64), empty(9, 32, dtype=f32), empty(3, dtype=I64),
                                      table, lens, cu, 2)
        assert q.shape == (3, 4, 64) and q.dtype == F16
        y = decoder.kv8_tree_attention(q, c, empty(3, 1, dtype=I64), table, lens, cu, 2, 6)
        assert y.shape == (3, 4, 64) and y.dtype == F16
        assert decoder.kv8_keep(c, empty(2, 4, dtype=I32), table, lens, cu) is None
        out, h = decoder.residual_norm(empty(3, 40), empty(3, 40, dtype=f32), empty(40, dtype=f32))
        assert out.shape == h.shape == (3, 40) and out.dtype == F16 and h.dtype == f32
        out, h = decoder.residual_norm(empty(3, 40), empty(3, 40))
        assert out is None and h.dtype == F16
        assert decoder.gated_norm(empty(3, 5, 40), empty(3, 5, 40), empty(40, dtype=f32)).shape == (3, 5, 40)


def test_tree_masks():
    rng = random.Random(0)
    trees = [[], [-1], [-1, 0, 0, 2, -1], [-1] + [rng.randrange(i) for i in range(1, 140)]]
    m = decoder.tree_mask(trees)
    assert m.shape == (146, 3) and m.dtype == I64
    at = 0
    for tree in trees:
        for i in range(len(tree)):
            seen, j = set(), i
            while j >= 0:
                seen.add(j)
                j = tree[j]
            assert {j for j in range(192) if int(m[at + i, j // 64]) >> j % 64 & 1} == seen
        at += len(tree)
    assert decoder.tree_mask([[-1, 0]]).tolist() == [[1], [3]]
    assert decoder.tree_mask([]).shape == (0, 1)
    for bad in ([0], [-1, 1], [-2], [-1, 0, 5]):
        with pytest.raises(ValueError, match="parent"):
            decoder.tree_mask([bad])


def test_tensors_without_memory_are_refused():
    """A C caller's NULL where a tensor has elements: an error, for each tensor of each entry point. Optional ones may be NULL
    themselves."""
    lib = ctypes.CDLL(decoder.LIB_PATH)
    lib.gguf_decoder_last_error.restype = ctypes.c_char_p
    i64, f32, P, null = ctypes.c_int64, ctypes.c_float, ctypes.byref, ctypes.c_void_p(None)
    c = _cache()
    table, lens, cu, rows, w = torch.zeros(2, 2, dtype=I32), _ints(5, 6), _ints(0, 1, 3), torch.zeros(3, 2, 64), torch.zeros(64)
    half, mask, x = torch.zeros(3, 4, 64, dtype=F16), torch.zeros(3, 1, dtype=I64), torch.zeros(3, 64)
    ws = torch.zeros(1 << 20, dtype=torch.uint8)
    room = (ctypes.c_void_p(ws.data_ptr() + -ws.data_ptr() % 16), ctypes.c_size_t((1 << 20) - 16), null)
    calls = {
        "kv8_rotary_append": (["cache", rows, rows, rows, torch.zeros(9, 32), torch.zeros(3, dtype=I64), table, lens, cu, w, w, rows],
                              lambda a: (*a[:9], i64(2), 0, *a[9:11], f32(1e-6), a[11], null), (9, 10)),
        "kv8_tree_attention": ([half, "cache", mask, table, lens, cu, half],
                               lambda a: (*a[:6], i64(2), i64(6), f32(1), a[6], *room), ()),
        "kv8_keep": (["cache", torch.zeros(2, 4, dtype=I32), table, lens, cu], lambda a: (*a, null), ()),
        "residual_norm": ([x, x, x, w, w, x, x], lambda a: (*a[:3], 2, *a[3:5], f32(1), f32(1e-6), *a[5:], null), (1, 2, 3)),
    }
    for name, (tensors, order, optional) in calls.items():
        call = getattr(lib, "gguf_" + name)

        def refused(descs, message):
            assert call(*order([d if d is None else P(d) for d in descs])) == 1
            assert message in lib.gguf_decoder_last_error().decode(), (name, lib.gguf_decoder_last_error())

        for spoil in range(-1, len(tensors)):
            for part in range(4 if spoil >= 0 and isinstance(tensors[spoil], str) else 1):
                descs = [_CacheT(*map(_desc, c)) if isinstance(t, str) else _desc(t) for t in tensors]
                if spoil >= 0:
                    d = descs[spoil]
                    (d if isinstance(d, _T) else getattr(d, ("k", "v", "k_scale", "v_scale")[part])).data = None
                refused(descs, "must be CUDA tensors" if spoil < 0 else "no data")
        for spoil in range(len(tensors)):
            descs = [_CacheT(*map(_desc, c)) if isinstance(t, str) else _desc(t) for t in tensors]
            descs[spoil] = None
            refused(descs, "must be CUDA tensors" if spoil in optional else "")


def test_tree_workspaces():
    """Hints beyond every size count as what the tensors hold."""
    lib = ctypes.CDLL(decoder.LIB_PATH)
    lib.gguf_kv8_tree_attention_workspace_bytes.restype = ctypes.c_size_t
    i64, P = ctypes.c_int64, ctypes.byref
    for d, q_heads, tokens in ((64, 4, 3), (256, 8, 50), (192, 64, 100)):
        c = _cache(d=d)
        cache, q = _CacheT(*map(_desc, c)), _desc(torch.zeros(tokens, q_heads, d, dtype=F16))

        def bytes_of(max_new, max_len):
            return lib.gguf_kv8_tree_attention_workspace_bytes(P(cache), P(q), i64(2), i64(max_new), i64(max_len))

        for hint in (2 ** 62, 2 ** 63 - 1):
            assert bytes_of(hint, 6) == bytes_of(tokens, 6)
            assert 0 < bytes_of(hint, hint) == bytes_of(tokens, 2 ** 31 - 1)


@pytest.mark.parametrize("size", [(3, (1 << 30) + 1), (3, 2, (1 << 31) - 1), (1 << 20, 1 << 20, 8), ((1 << 31) - 1, 2, 8)], ids=str)
def test_norms_of_too_many_values(size):
    """A C caller's sizes beyond what an index holds."""
    lib = ctypes.CDLL(decoder.LIB_PATH)
    lib.gguf_decoder_last_error.restype = ctypes.c_char_p
    x = _desc(torch.zeros(3, 8) if len(size) == 2 else torch.zeros(3, 3, 8))
    x.size[:len(size)] = list(size)
    null = ctypes.c_void_p(None)
    assert lib.gguf_residual_norm(ctypes.byref(x), null, null, 0, null, null, ctypes.c_float(1), ctypes.c_float(0), ctypes.byref(x), null, null) == 1
    assert "too many" in lib.gguf_decoder_last_error().decode()
