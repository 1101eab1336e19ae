"""Refusals of the paged-cache operators: the C entry points check their arguments before any CUDA call, so
they are tested without a GPU (pointers are never followed)."""
import ctypes

import pytest
import torch

OK, SHAPE, ALIGN, UNSUPPORTED, ARG = 0, -1, -2, -3, -5
PTR = 1 << 20


def cache(**kw):
    from qmtp import _lib

    d = dict(k=PTR, v=PTR, table=PTR, lens=PTR, pages=10, ld_table=4, n_kv=2, page=16, Dh=128, table_w=4, B=2)
    d.update(kw)
    return _lib.PagedCacheArgs(**d)


def attn(**kw):
    from qmtp import _lib

    d = dict(q=PTR, gate=None, out=PTR, q_ld=0, gate_ld=0, gate_hs=0, T=4, n_q=4, scale=0.1, window=0, sinks=0)
    d.update(kw)
    return _lib.PagedArgs(**d)


BAD_CACHE = [
    (dict(k=None), ARG), (dict(v=None), ARG), (dict(table=None), ARG), (dict(lens=None), ARG), (dict(B=0), SHAPE),
    (dict(B=4097), SHAPE), (dict(n_kv=0), SHAPE), (dict(n_kv=65537), SHAPE), (dict(pages=0), SHAPE), (dict(table_w=0), SHAPE),
    (dict(ld_table=3), SHAPE), (dict(Dh=96), UNSUPPORTED), (dict(Dh=512), UNSUPPORTED), (dict(page=8), UNSUPPORTED),
    (dict(page=48), UNSUPPORTED), (dict(page=512), UNSUPPORTED), (dict(pages=1 << 27), SHAPE),
    (dict(table_w=1 << 28, ld_table=1 << 28), SHAPE), (dict(k=PTR + 8), ALIGN), (dict(v=PTR + 2), ALIGN)]
BAD_ATTN = [
    (dict(q=None), ARG), (dict(out=None), ARG), (dict(scale=0.0), ARG), (dict(scale=-1.0), ARG),
    (dict(scale=float("nan")), ARG), (dict(scale=float("inf")), ARG), (dict(window=-1), ARG), (dict(sinks=-1), ARG),
    (dict(T=0), SHAPE), (dict(n_q=0), SHAPE), (dict(n_q=5), SHAPE), (dict(n_q=1 << 30), SHAPE), (dict(n_q=130), UNSUPPORTED), (dict(q_ld=4), SHAPE),
    (dict(q_ld=504), SHAPE), (dict(gate=PTR, gate_ld=12), SHAPE), (dict(gate=PTR, gate_hs=4), SHAPE),
    (dict(q=PTR + 8), ALIGN), (dict(out=PTR + 2), ALIGN), (dict(gate=PTR + 2), ALIGN)]


@pytest.mark.parametrize("change,code", BAD_CACHE)
def test_cache_refusals(change, code):
    from qmtp import _lib

    L, c = _lib.lib(), cache(**change)
    assert L.qmtp_paged_attention(ctypes.byref(attn()), ctypes.byref(c), PTR, 1 << 30, None) == code
    assert L.qmtp_paged_prompt(ctypes.byref(attn()), PTR, ctypes.byref(c), PTR, 1 << 30, None) == code
    assert L.qmtp_paged_append(PTR, 2048, 4, None, 4, 0, None, None, 1e-6, None, None, 0, 0, PTR, ctypes.byref(c), None) == code


@pytest.mark.parametrize("change,code", BAD_ATTN + [(dict(T=3), SHAPE), (dict(T=18), UNSUPPORTED)])
def test_attention_refusals(change, code):
    from qmtp import _lib

    assert _lib.lib().qmtp_paged_attention(ctypes.byref(attn(**change)), ctypes.byref(cache()), PTR, 1 << 30, None) == code


@pytest.mark.parametrize("change,code", BAD_ATTN)
def test_prompt_refusals(change, code):
    from qmtp import _lib

    L = _lib.lib()
    assert L.qmtp_paged_prompt(ctypes.byref(attn(**change)), PTR, ctypes.byref(cache()), PTR, 1 << 30, None) == code
    assert L.qmtp_paged_prompt(ctypes.byref(attn()), None, ctypes.byref(cache()), PTR, 1 << 30, None) == ARG


def test_attention_workspace():
    from qmtp import _lib

    L = _lib.lib()
    long = cache(table_w=100, ld_table=100)
    n = L.qmtp_paged_attention_workspace(ctypes.byref(attn()), ctypes.byref(long))
    assert n >= 2 * 13 * 2 * 4 * (128 + 2) * 4  # B x slabs of 128 in 1600 x S x heads x (head_dim + 2) floats
    assert L.qmtp_paged_attention_workspace(ctypes.byref(attn()), ctypes.byref(cache(B=0))) == 0  # a refused call
    call = lambda ws, size: L.qmtp_paged_attention(ctypes.byref(attn()), ctypes.byref(long), ws, size, None)
    assert call(None, n) == ARG and call(PTR, n - 1) == SHAPE and call(PTR + 8, n) == ALIGN
    # a window needs the slabs it can touch, not the whole table's
    huge = cache(table_w=100000, ld_table=100000)
    w = L.qmtp_paged_attention_workspace(ctypes.byref(attn(window=1024, sinks=4)), ctypes.byref(huge))
    assert 0 < w < 2 * 16 * 2 * 4 * (128 + 2) * 4


@pytest.mark.parametrize("change,code", [
    (dict(qkv=None), ARG), (dict(q_out=None), ARG), (dict(cos=PTR), ARG), (dict(eps=-1.0), ARG), (dict(eps=float("nan")), ARG),
    (dict(T=0), SHAPE), (dict(T=3), SHAPE), (dict(n_q=0), SHAPE), (dict(n_q=1 << 30), SHAPE), (dict(ld=1020), SHAPE), (dict(ld=1016), SHAPE),
    (dict(gated=1), SHAPE), (dict(cos=PTR, sin=PTR, rotary=24, max_pos=9), UNSUPPORTED),
    (dict(cos=PTR, sin=PTR, rotary=144, max_pos=9), UNSUPPORTED), (dict(cos=PTR, sin=PTR, rotary=0, max_pos=9), UNSUPPORTED),
    (dict(cos=PTR, sin=PTR, rotary=32, max_pos=0), SHAPE), (dict(qkv=PTR + 2), ALIGN), (dict(q_out=PTR + 8), ALIGN),
    (dict(q_w=PTR + 2), ALIGN), (dict(k_w=PTR + 2), ALIGN), (dict(cos=PTR + 4, sin=PTR, rotary=32, max_pos=9), ALIGN)])
def test_append_refusals(change, code):
    from qmtp import _lib

    d = dict(qkv=PTR, ld=1024, T=4, cu=None, n_q=4, gated=0, q_w=None, k_w=None, eps=1e-6, cos=None, sin=None, rotary=0,
             max_pos=0, q_out=PTR)
    d.update(change)
    assert _lib.lib().qmtp_paged_append(*d.values(), ctypes.byref(cache()), None) == code


def test_python_refuses_cpu_tensors():
    from qmtp import paged

    x = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        paged.PagedCache(x, x.clone())
    with pytest.raises(ValueError):
        paged.PagedCache(x, x[:2])


@pytest.mark.parametrize("struct, pack", [("PagedCacheArgs", "PAGED_CACHE_ARGS"), ("PagedArgs", "PAGED_ARGS")])
def test_packed_arguments_have_the_structures_layout(struct, pack):
    from qmtp import _lib

    cls = getattr(_lib, struct)
    values = [float(i) + 0.5 if t is ctypes.c_float else i + 1 for i, (_, t) in enumerate(cls._fields_)]
    got = cls.from_buffer_copy(getattr(_lib, pack).pack(*values))
    assert [getattr(got, name) for name, _ in cls._fields_] == values
