"""Attention over a key/value cache kept in pages: several sequences served from one pool.

The decoder (``qmtp.mtp``) runs one conversation on contiguous caches; these operators are the same
attention layer for a batch of them (mtp.py:143-153 in the reference serves one at a time):

  append_qkv        per-head q/k RMS norms, position rotation and the cache write, one launch
  attention         the newest 1..8 tokens of every sequence (decode, verify): split over the cache's
                    length and joined
  prompt_attention  a ragged batch of prompt chunks, on the tensor cores

A sequence's tokens live in pages named by its row of ``table``; ``lens`` counts them, this call's new
tokens included.  Both are device tensors that the kernels read when they run, so a captured CUDA graph
follows them.  Attention optionally has a sliding window with first tokens that stay visible (sinks), and
the sigmoid output gate of the model's attention layers.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib

MAX_NEW = 8  # new tokens per sequence that ``attention`` takes
BF16 = torch.bfloat16


class PagedCache:
    """Key and value pages, bf16 [pages, n_kv, page, head_dim] each (head_dim 64, 128 or 256; page a power
    of two, 16 .. 256).  Handing pages to sequences, and taking them back, is the caller's."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        _need(k.dim() == 4 and k.shape == v.shape, "k and v are [pages, n_kv, page, head_dim], of one shape")
        _tensor("k", k, BF16, k.device)
        _tensor("v", v, BF16, k.device)
        _lib.require_cuda(k, v)
        self.k, self.v = k, v

    @classmethod
    def empty(cls, pages: int, n_kv: int, head_dim: int, page: int = 64, device="cuda") -> "PagedCache":
        """A pool of unset pages (a page may hold anything before its rows are appended)."""
        shape = (pages, n_kv, page, head_dim)
        return cls(torch.empty(shape, dtype=BF16, device=device), torch.empty(shape, dtype=BF16, device=device))

    @property
    def n_kv(self) -> int:
        return self.k.shape[1]

    @property
    def page(self) -> int:
        return self.k.shape[2]

    @property
    def head_dim(self) -> int:
        return self.k.shape[3]

    def _args(self, table: torch.Tensor, lens: torch.Tensor) -> "_lib.PagedCacheArgs":
        dev = self.k.device
        _tensor("table", table, torch.int32, dev)
        _tensor("lens", lens, torch.int32, dev)
        _need(table.dim() == 2 and lens.dim() == 1 and table.shape[0] == lens.shape[0],
              "table is [sequences, pages of a sequence], lens [sequences]")
        _need(table.shape[1] > 0 and table.stride(1) == 1 and lens.is_contiguous(), "table rows and lens need to be contiguous")
        B, W = table.shape
        ld = table.stride(0) if B > 1 else W
        pages, n_kv, page, dh = self.k.shape
        return _lib.PagedCacheArgs(k=self.k.data_ptr(), v=self.v.data_ptr(), table=table.data_ptr(),
                                   lens=lens.data_ptr(), pages=pages, ld_table=ld, n_kv=n_kv, page=page, Dh=dh,
                                   table_w=W, B=B)


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(f"qmtp.paged: {what}")


def _tensor(name: str, t: torch.Tensor, dtype, device) -> None:
    if not t.is_cuda:
        raise RuntimeError("qmtp ops run on CUDA tensors only (no CPU fallback)")
    _need(t.dtype == dtype, f"{name} has type {t.dtype}, not {dtype}")
    _need(t.device == device, f"{name} is on {t.device}, the cache on {device}")


def append_qkv(qkv, cache: PagedCache, table, lens, cu=None, *, n_heads: int, gated: bool = False, q_norm=None,
               k_norm=None, cos=None, sin=None, eps: float = 1e-6, out=None):
    """Splits projection rows into heads, norms and rotates q and k, writes k and v to their pages.

    qkv bf16 [T, >= width]: per row n_heads query heads (``gated``: (q, gate) pairs), then the key heads,
    then the value heads.  cu int32 [B + 1]: rows cu[b] .. cu[b+1] are sequence b's new tokens, the last
    ones of its lens[b]; None: the same number of rows for every sequence.  q_norm, k_norm bf16 [head_dim]
    or None; cos, sin fp32 [positions, rotary / 2] or None (``qmtp.model.rope_tables``); the rotation turns
    the first 2 * cos.shape[1] dims.  Everything is computed in fp32 and rounded once.

    -> (q bf16 [T, n_heads, head_dim], gate: a view [T, n_heads, head_dim] of qkv, or None).  Rows of no
    sequence, and rows at a negative position (lens[b] below the row count), are left as they were."""
    dev, dh = cache.k.device, cache.head_dim
    _tensor("qkv", qkv, BF16, dev)
    _need(qkv.dim() == 2 and qkv.stride(1) == 1, "qkv is [rows, width] with contiguous rows")
    T, per = qkv.shape[0], 2 if gated else 1
    width = (n_heads * per + 2 * cache.n_kv) * dh
    _need(n_heads >= 1 and qkv.shape[1] >= width, f"a row of qkv needs {width} values")
    B = table.shape[0]
    _check_cu(cu, B, dev)
    for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
        if w is not None:
            _tensor(name, w, BF16, dev)
            _need(w.shape == (dh,) and w.is_contiguous(), f"{name} is [head_dim], contiguous")
    _need((cos is None) == (sin is None), "cos and sin go together")
    if cos is not None:
        for name, t in (("cos", cos), ("sin", sin)):
            _tensor(name, t, torch.float32, dev)
            _need(t.dim() == 2 and t.shape == cos.shape and t.is_contiguous(), "cos and sin are [positions, rotary / 2], contiguous")
    if out is None:
        out = torch.empty((T, n_heads, dh), dtype=BF16, device=dev)
    else:
        _tensor("out", out, BF16, dev)
        _need(out.shape == (T, n_heads, dh) and out.is_contiguous(), "out is [rows, n_heads, head_dim], contiguous")
    gate = qkv[:, : n_heads * 2 * dh].unflatten(1, (n_heads, 2, dh))[:, :, 1] if gated else None
    if T == 0:
        return out, gate
    args = cache._args(table, lens)
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().qmtp_paged_append(
            qkv.data_ptr(), _row_stride(qkv, width), T, _lib.ptr(cu), n_heads, int(gated), _lib.ptr(q_norm), _lib.ptr(k_norm),
            float(eps), _lib.ptr(cos), _lib.ptr(sin), 0 if cos is None else 2 * cos.shape[1],
            0 if cos is None else cos.shape[0], out.data_ptr(), ctypes.byref(args), _lib.stream()), "append_qkv")
    return out, gate


def _row_stride(t, width: int) -> int:
    """Elements between rows; a single row's stride says nothing, so it counts as dense."""
    return t.stride(0) if t.shape[0] > 1 else -(-width // 8) * 8


def _check_cu(cu, B: int, dev) -> None:
    if cu is not None:
        _tensor("cu", cu, torch.int32, dev)
        _need(cu.shape == (B + 1,) and cu.is_contiguous(), "cu is [sequences + 1], contiguous")


def _attention_args(q, cache: PagedCache, gate, scale, window, sinks, out):
    dev, dh = cache.k.device, cache.head_dim
    _tensor("q", q, BF16, dev)
    _need(q.dim() == 3 and q.shape[2] == dh, "q is [rows, heads, head_dim]")
    T, nq, _ = q.shape
    _need(nq >= 1 and q.stride(2) == 1 and (nq == 1 or q.stride(1) == dh), "a row of q needs to be contiguous")
    if out is None:
        out = torch.empty((T, nq * dh), dtype=BF16, device=dev)
    else:
        _tensor("out", out, BF16, dev)
        _need(out.shape == (T, nq * dh) and out.is_contiguous(), "out is [rows, heads * head_dim], contiguous")
    a = _lib.PagedArgs(q=q.data_ptr(), gate=None, out=out.data_ptr(), q_ld=_row_stride(q, nq * dh), gate_ld=0, gate_hs=0,
                       T=T, n_q=nq, scale=float(dh ** -0.5 if scale is None else scale), window=int(window),
                       sinks=int(sinks))
    if gate is not None:
        _tensor("gate", gate, BF16, dev)
        _need(gate.shape == q.shape and gate.stride(2) == 1, "gate has q's shape and contiguous heads")
        a.gate, a.gate_ld, a.gate_hs = gate.data_ptr(), gate.stride(0) if T > 1 else 0, gate.stride(1) if nq > 1 else 0
    return a, out


def attention(q, cache: PagedCache, table, lens, *, gate=None, scale: float | None = None, window: int = 0,
              sinks: int = 0, out=None):
    """Attention of the newest tokens: q bf16 [B * S, heads, head_dim], row b * S + s at position
    lens[b] - S + s of sequence b, S <= 8 -> bf16 [B * S, heads * head_dim].

    A query sees the keys at or before its position, with a window only those less than ``window`` back and
    the first ``sinks``; a query that sees none gives zeros.  scale: head_dim ** -0.5 by default.  gate (q's
    shape, any head and row strides): the result is multiplied by sigmoid(gate).  A token's result has the
    same bits whatever the batch, S and the page size are.  out must not overlap the inputs."""
    a, out = _attention_args(q, cache, gate, scale, window, sinks, out)
    if q.shape[0] == 0:
        return out
    c = cache._args(table, lens)
    L = _lib.lib()
    with torch.cuda.device(cache.k.device):
        n = L.qmtp_paged_attention_workspace(ctypes.byref(a), ctypes.byref(c))
        ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
        _lib.check(L.qmtp_paged_attention(ctypes.byref(a), ctypes.byref(c), _lib.ptr(ws), n, _lib.stream()),
                   "paged attention")
    return out


def prompt_attention(q, cache: PagedCache, table, lens, cu, *, gate=None, scale: float | None = None, window: int = 0,
                     sinks: int = 0, out=None):
    """Attention of a ragged batch of prompt chunks: rows cu[b] .. cu[b+1] of q bf16 [T, heads, head_dim] are the
    last tokens of sequence b -> bf16 [T, heads * head_dim].  Masks, scale and gate as in ``attention``; rows of
    no sequence are left as they were.  Any number of new tokens per sequence; ``attention`` is the one for a few."""
    a, out = _attention_args(q, cache, gate, scale, window, sinks, out)
    _check_cu(cu, table.shape[0], cache.k.device)
    if q.shape[0] == 0:
        return out
    c = cache._args(table, lens)
    L = _lib.lib()
    with torch.cuda.device(cache.k.device):
        n = L.qmtp_paged_prompt_workspace(ctypes.byref(a), ctypes.byref(c))
        ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
        _lib.check(L.qmtp_paged_prompt(ctypes.byref(a), cu.data_ptr(), ctypes.byref(c), _lib.ptr(ws), n, _lib.stream()),
                   "paged prompt attention")
    return out
