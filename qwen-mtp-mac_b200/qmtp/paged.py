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

import torch

from . import _lib

MAX_NEW = 8  # new tokens per sequence that ``attention`` takes
BF16 = torch.bfloat16
_INT_MAX = 2 ** 31 - 1


class PagedCache:
    """Key and value pages, bf16 [pages, n_kv, page, head_dim] each (head_dim 64, 128 or 256; page a power
    of two, 16 .. 256).  Handing pages to sequences, and taking them back, is the caller's."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        _need(k.dim() == 4 and k.shape == v.shape, "k and v are [pages, n_kv, page, head_dim], of one shape")
        self._k, self._v, self._index = k, v, k.get_device()
        for name, t in (("k", k), ("v", v)):
            _tensor(name, t, BF16, self._index)
        _lib.require_cuda(k, v)
        self.pages, self.n_kv, self.page, self.head_dim = k.shape
        self._k_ptr, self._v_ptr = k.data_ptr(), v.data_ptr()

    @classmethod
    def empty(cls, pages: int, n_kv: int, head_dim: int, page: int = 64, device="cuda") -> "PagedCache":
        """A pool of unset pages (a page may hold anything before its rows are appended)."""
        shape = (pages, n_kv, page, head_dim)
        return cls(torch.empty(shape, dtype=BF16, device=device), torch.empty(shape, dtype=BF16, device=device))

    @property
    def k(self) -> torch.Tensor:
        return self._k

    @property
    def v(self) -> torch.Tensor:
        return self._v

    def _args(self, table: torch.Tensor, lens: torch.Tensor) -> bytes:
        _tensor("table", table, torch.int32, self._index)
        _tensor("lens", lens, torch.int32, self._index)
        if table.dim() != 2:
            _need(False, "table is [sequences, pages of a sequence], lens [sequences]")
        (B, W), (ld, one) = table.shape, table.stride()
        if lens.shape != (B,) or W == 0 or (one != 1 and W > 1) or not lens.is_contiguous():
            _need(False, "table is [sequences, pages of a sequence] with contiguous rows, lens [sequences], contiguous")
        if W > _INT_MAX or B > _INT_MAX:
            _need(False, "table is too large")
        return _lib.PAGED_CACHE_ARGS.pack(self._k_ptr, self._v_ptr, table.data_ptr(), lens.data_ptr(), self.pages,
                                          ld if B > 1 else W, self.n_kv, self.page, self.head_dim, W, B)


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(f"qmtp.paged: {what}")


def _tensor(name: str, t: torch.Tensor, dtype, index: int) -> None:
    """t is a tensor of that type on the cache's device."""
    if t.dtype is dtype and t.get_device() == index >= 0:
        return
    if not t.is_cuda:
        raise RuntimeError("qmtp ops run on CUDA tensors only (no CPU fallback)")
    _need(t.dtype == dtype, f"{name} has type {t.dtype}, not {dtype}")
    _need(False, f"{name} is on {t.device}, the cache on cuda:{index}")


def _call(index: int, what: str, fn, *args) -> None:
    """fn(*args, stream) on the current stream of the tensors' device, whichever device is current."""
    if torch.cuda.current_device() == index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc, what)


def append_qkv(qkv, cache: PagedCache, table, lens, cu=None, *, n_heads: int, gated: bool = False, q_norm=None,
               k_norm=None, cos=None, sin=None, eps: float = 1e-6, out=None):
    """Splits projection rows into heads, norms and rotates q and k, writes k and v to their pages.

    qkv bf16 [T, >= width]: per row n_heads query heads (``gated``: (q, gate) pairs), then the key heads,
    then the value heads.  cu int32 [B + 1]: rows cu[b] .. cu[b+1] are sequence b's new tokens, the last
    ones of its lens[b]; None: the same number of rows for every sequence.  q_norm, k_norm bf16 [head_dim]
    or None, each by itself; cos, sin fp32 [positions, rotary / 2] or None (``qmtp.model.rope_tables``); the rotation turns
    the first 2 * cos.shape[1] dims.  Everything is computed in fp32 and rounded once.

    -> (q bf16 [T, n_heads, head_dim], gate: a view [T, n_heads, head_dim] of qkv, or None).  Rows of no
    sequence, and rows at a negative position (lens[b] below the row count), are left as they were.  Offsets
    that decrease or leave [0, T] hold no rows and set the device error word."""
    dev, dh = cache._index, cache.head_dim
    _tensor("qkv", qkv, BF16, dev)
    if qkv.dim() != 2:
        _need(False, "qkv is [rows, width] with contiguous rows")
    (T, w), (ld, one) = qkv.shape, qkv.stride()
    if one != 1:
        _need(False, "qkv is [rows, width] with contiguous rows")
    width = (n_heads * (2 if gated else 1) + 2 * cache.n_kv) * dh
    if n_heads < 1 or w < width:
        _need(False, f"a row of qkv needs {width} values")
    if cu is not None:
        _check_cu(cu, table.shape[0], dev)
    for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
        if w is not None:
            _tensor(name, w, BF16, dev)
            if w.shape != (dh,) or not w.is_contiguous():
                _need(False, f"{name} is [head_dim], contiguous")
    rotary = max_pos = 0
    if cos is not None or sin is not None:
        _need(cos is not None and sin is not None, "cos and sin go together")
        _tensor("cos", cos, torch.float32, dev)
        _tensor("sin", sin, torch.float32, dev)
        shape = cos.shape
        if len(shape) != 2 or sin.shape != shape or not (cos.is_contiguous() and sin.is_contiguous()):
            _need(False, "cos and sin are [positions, rotary / 2], contiguous")
        max_pos, rotary = shape[0], 2 * shape[1]
    if out is None:
        out = qkv.new_empty(T, n_heads, dh)
    else:
        _tensor("out", out, BF16, dev)
        _need(out.shape == (T, n_heads, dh) and out.is_contiguous(), "out is [rows, n_heads, head_dim], contiguous")
    gate = None
    if gated:
        gate = qkv.as_strided((T, n_heads, dh), (ld, 2 * dh, 1), qkv.storage_offset() + dh)
    if T:
        ptr = _lib.ptr
        _call(dev, "append_qkv", _lib.lib().qmtp_paged_append, qkv.data_ptr(), _row_stride(T, ld, width), T, ptr(cu), n_heads,
              1 if gated else 0, ptr(q_norm), ptr(k_norm), eps, ptr(cos), ptr(sin), rotary, max_pos, out.data_ptr(),
              cache._args(table, lens))
    return out, gate


def _row_stride(rows: int, ld: int, width: int) -> int:
    """Elements between rows; a single row's stride says nothing, so it counts as dense."""
    return ld if rows > 1 else -(-width // 8) * 8


def _check_cu(cu, B: int, dev: int) -> None:
    _tensor("cu", cu, torch.int32, dev)
    if cu.shape != (B + 1,) or not cu.is_contiguous():
        _need(False, "cu is [sequences + 1], contiguous")


def _attention_args(q, cache: PagedCache, gate, scale, window, sinks, out):
    dev, dh = cache._index, cache.head_dim
    _tensor("q", q, BF16, dev)
    if q.dim() != 3:
        _need(False, "q is [rows, heads, head_dim]")
    shape, (ld, hs, one) = q.shape, q.stride()
    T, nq, d = shape
    if d != dh:
        _need(False, "q is [rows, heads, head_dim]")
    width = nq * dh
    if nq < 1 or one != 1 or (hs != dh and nq > 1) or (ld < width and T > 1):
        _need(False, "a row of q needs to be contiguous, and rows apart")
    if window < 0 or sinks < 0:
        _need(False, "window and sinks count tokens")
    if scale is None:
        scale = dh ** -0.5
    elif not 0 < scale < 2.35e38:
        _need(False, "scale is positive, and scale * log2(e) finite in fp32")
    if T > _INT_MAX or nq > _INT_MAX:
        _need(False, "q is too large")
    if out is None:
        out = q.new_empty(T, width)
    else:
        _tensor("out", out, BF16, dev)
        _need(out.shape == (T, width) and out.is_contiguous(), "out is [rows, heads * head_dim], contiguous")
    gate_ptr = gate_ld = gate_hs = 0
    if gate is not None:
        _tensor("gate", gate, BF16, dev)
        if gate.shape != shape:
            _need(False, "gate has q's shape and contiguous heads")
        gate_ld, gate_hs, gate_one = gate.stride()
        if gate_one != 1:
            _need(False, "gate has q's shape and contiguous heads")
        gate_ptr, gate_ld, gate_hs = gate.data_ptr(), gate_ld if T > 1 else 0, gate_hs if nq > 1 else 0
    return _lib.PAGED_ARGS.pack(q.data_ptr(), gate_ptr, out.data_ptr(), _row_stride(T, ld, width), gate_ld, gate_hs, T, nq,
                                scale, min(window, _INT_MAX), min(sinks, _INT_MAX)), out


def _launch(cache, what, fn, workspace, a, c, q, *args):
    """Workspace and launch, both with the tensors' device as the current one: the launch's form goes by its SMs."""
    index = cache._index
    if torch.cuda.current_device() != index:
        with torch.cuda.device(index):
            return _launch(cache, what, fn, workspace, a, c, q, *args)
    n = workspace(a, c)
    ws = q.new_empty(n, dtype=torch.uint8) if n else None
    rc = fn(a, *args, c, _lib.ptr(ws), n, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc, what)


def attention(q, cache: PagedCache, table, lens, *, gate=None, scale: float | None = None, window: int = 0,
              sinks: int = 0, out=None):
    """Attention of the newest tokens: q bf16 [B * S, heads, head_dim], row b * S + s at position
    lens[b] - S + s of sequence b, S <= 8 -> bf16 [B * S, heads * head_dim].

    A query sees the keys at or before its position, with a window only those less than ``window`` back and
    the first ``sinks``; a query that sees none gives zeros.  scale: head_dim ** -0.5 by default.  gate (q's
    shape, any head and row strides): the result is multiplied by sigmoid(gate).  A token's result has the
    same bits whatever the batch, S and the page size are, as long as its sequence's keys and values are
    finite.  out must not overlap the inputs.  The workspace goes by the table's width, not by the lengths:
    a table much wider than its sequences costs memory, and a second launch where a short one needs one."""
    a, out = _attention_args(q, cache, gate, scale, window, sinks, out)
    if q.shape[0]:
        L = _lib.lib()
        _launch(cache, "paged attention", L.qmtp_paged_attention, L.qmtp_paged_attention_workspace, a,
                cache._args(table, lens), q)
    return out


def prompt_attention(q, cache: PagedCache, table, lens, cu, *, gate=None, scale: float | None = None, window: int = 0,
                     sinks: int = 0, out=None):
    """Attention of a ragged batch of prompt chunks: rows cu[b] .. cu[b+1] of q bf16 [T, heads, head_dim] are the
    last tokens of sequence b -> bf16 [T, heads * head_dim].  Masks, scale and gate as in ``attention``; rows of
    no sequence are left as they were.  Any number of new tokens per sequence; ``attention`` is the one for a few.
    Short prompts are fastest with a table as wide as the longest sequence (the keys are split by its width)."""
    a, out = _attention_args(q, cache, gate, scale, window, sinks, out)
    if cu is None:
        _need(False, "a prompt's rows are named by cu")
    _check_cu(cu, table.shape[0], cache._index)
    if q.shape[0]:
        L = _lib.lib()
        _launch(cache, "paged prompt attention", L.qmtp_paged_prompt, L.qmtp_paged_prompt_workspace, a,
                cache._args(table, lens), q, cu.data_ptr())
    return out
