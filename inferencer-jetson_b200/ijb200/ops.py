"""The stand-alone serving operators on torch tensors: the paged K/V cache
(write, read-back, attention of new tokens) and sampling from logits.

Thin calls of the C ABI (include/ijb200.h has each operator's definition):
tensors are passed by address, on the current stream of their device, and
nothing is allocated but outputs and the attention's workspace.  Arguments that
do not fit raise ValueError or IjbError; there is no fallback.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import lib as _L
from .lib import IjbError  # noqa: F401  (what the calls raise)

F32, F16 = 0, 1  # IJB_TYPE_F32, IJB_TYPE_F16
KV_F16, KV_E4M3 = 0, 2
_TYPE = {torch.float32: F32, torch.float16: F16}
_stream = torch._C._cuda_getCurrentRawStream


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _call(device: int, fn, *args) -> None:
    """One library call with `device` current, on its current stream."""
    if torch.cuda.current_device() == device:
        rc = fn(*args, _stream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _stream(device))
    if rc:
        _L.check(rc)


def _ptr(t, dtype, n: int, device: int, what: str):
    """Address of a contiguous vector of n values (None: NULL)."""
    if t is None:
        return None
    if t.dtype != dtype or t.numel() != n or t.get_device() != device or not t.is_contiguous():
        raise ValueError(f"{what}: expected {n} contiguous {dtype} values on cuda:{device}")
    return t.data_ptr()


def _rows(t, inner: int, device: int, what: str):
    """(address, stride in elements) of a [n, ..] tensor whose tokens are `inner` contiguous elements."""
    flat = t.dim() == 2 and t.stride(1) == 1 or t.dim() == 3 and t.stride(2) == 1 and t.stride(1) == t.shape[2]
    if t.get_device() != device or t.dtype not in _TYPE or not flat or t[0:1].numel() not in (0, inner):
        raise ValueError(f"{what}: expected [n, {inner}] fp32 or fp16 values on cuda:{device}, each token's contiguous")
    return t.data_ptr(), max(t.stride(0), inner) if t.shape[0] <= 1 else t.stride(0)


class PagedKV:
    """One paged K/V cache over the caller's tensors: ``data`` [pages, 2, kv_heads,
    page_size, head_dim] float16 or float8_e4m3fn, ``page_table`` [seqs, max_pages]
    int32, and for e4m3 ``scale`` [pages, 2, kv_heads, page_size] uint8 (a row's
    values are data * 2^(scale - 127)).  ``status``, if given, is one int32 or
    uint32 that collects the kernels' reports of indexes that name nothing."""

    def __init__(self, data, page_table, scale=None, status=None):
        _need(data.is_cuda and data.dim() == 5 and data.shape[1] == 2 and data.is_contiguous(),
              "data: expected a contiguous [pages, 2, kv_heads, page_size, head_dim] CUDA tensor")
        _need(data.dtype in (torch.float16, torch.float8_e4m3fn), "data: expected float16 or float8_e4m3fn")
        dev = data.get_device()
        _need(page_table.dim() == 2 and page_table.dtype == torch.int32 and page_table.is_contiguous() and
              page_table.get_device() == dev, "page_table: expected a contiguous [seqs, max_pages] int32 tensor beside data")
        e4m3 = data.dtype == torch.float8_e4m3fn
        _need(not e4m3 or scale is not None and scale.dtype == torch.uint8 and scale.shape == data.shape[:4] and
              scale.is_contiguous() and scale.get_device() == dev,
              "scale: an e4m3 cache needs contiguous uint8 [pages, 2, kv_heads, page_size] beside data")
        _need(status is None or status.element_size() == 4 and status.numel() == 1 and status.get_device() == dev,
              "status: expected one 32-bit word beside data")
        self.data, self.page_table, self.scale, self.status = data, page_table, scale if e4m3 else None, status
        self.device, self.kv_heads, self.head_dim = dev, data.shape[2], data.shape[4]
        self.row = self.kv_heads * self.head_dim
        self._lib = _L.load()
        self._view = _L.KvView(type=KV_E4M3 if e4m3 else KV_F16, kv_heads=self.kv_heads, head_dim=self.head_dim,
                               page_size=data.shape[3], num_pages=data.shape[0], data_dev=data.data_ptr(),
                               scale_dev=scale.data_ptr() if e4m3 else None, page_table_dev=page_table.data_ptr(),
                               n_seqs=page_table.shape[0], max_pages=page_table.shape[1])
        self._ref = ctypes.byref(self._view)
        self._status = status.data_ptr() if status is not None else None

    def append(self, k, v, seq, pos) -> None:
        """Writes rows k, v [n, kv_heads, head_dim] (fp32 or fp16) at positions pos [n] of sequences seq [n]."""
        n = k.shape[0]
        kp, stride = _rows(k, self.row, self.device, "k")
        vp, vstride = _rows(v, self.row, self.device, "v")
        _need(k.dtype == v.dtype and v.shape[0] == n and (vstride == stride or n <= 1),
              "k and v differ in type, length or stride")
        _call(self.device, self._lib.ijb_kv_append, self._ref, _TYPE[k.dtype], kp, vp, stride, n,
              _ptr(seq, torch.int32, n, self.device, "seq"), _ptr(pos, torch.int32, n, self.device, "pos"), self._status)

    def gather(self, seq, pos, dtype=torch.float32):
        """The rows at positions pos [n] of sequences seq [n]: (k, v), each [n, kv_heads, head_dim].
        Rows of entries that are skipped (a negative position) hold no meaning."""
        _need(dtype in _TYPE, "dtype must be float32 or float16")
        n = seq.numel()
        out = torch.empty((2, n, self.kv_heads, self.head_dim), dtype=dtype, device=self.data.device)
        k, v = out[0], out[1]
        _call(self.device, self._lib.ijb_kv_gather, self._ref, _TYPE[dtype], k.data_ptr(), v.data_ptr(), self.row, n,
              _ptr(seq, torch.int32, n, self.device, "seq"), _ptr(pos, torch.int32, n, self.device, "pos"), self._status)
        return k, v

    def attention(self, q, q_start, kv_len, seq=None, max_q: int = 0, scale: float | None = None, out=None):
        """Attention of new tokens: q [tokens, heads, head_dim] fp32 or fp16, entry e's tokens being rows
        q_start[e]..q_start[e + 1] and the last of the kv_len[e] positions of sequence seq[e] (default: e), which
        the cache already holds.  Each token sees the positions up to its own; a token before position 0 sees none and
        gets zeros.  ``max_q``: the most new tokens of any entry, if known.  Returns out (like q)."""
        _need(q.dim() == 3 and q.shape[2] == self.head_dim, "q: expected [tokens, heads, head_dim]")
        n, heads = q.shape[0], q.shape[1]
        qp, qs = _rows(q, heads * self.head_dim, self.device, "q")
        if out is None:
            out = torch.empty((n, heads, self.head_dim), dtype=q.dtype, device=q.device)
        _need(out.shape == q.shape and out.dtype == q.dtype, "out: expected the shape and type of q")
        op, os = _rows(out, heads * self.head_dim, self.device, "out")
        e = kv_len.numel()
        _need(e >= 1 and (seq is not None or e <= self.page_table.shape[0]), "kv_len: one length for each entry")
        size = self._lib.ijb_paged_attention_workspace(self._ref, heads, n, e)
        work = torch.empty((max(size, 16),), dtype=torch.uint8, device=q.device)
        _call(self.device, self._lib.ijb_paged_attention, self._ref, heads, _TYPE[q.dtype], qp, qs, op, os, n, e,
              _ptr(q_start, torch.int32, e + 1, self.device, "q_start"), _ptr(seq, torch.int32, e, self.device, "seq"),
              _ptr(kv_len, torch.int32, e, self.device, "kv_len"), max_q,
              1.0 / math.sqrt(self.head_dim) if scale is None else scale, work.data_ptr(), work.numel(), self._status)
        return out


def sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    """One token for each row of fp32 logits [n, vocab] from uniform numbers u [n] in [0, 1) and per-row settings
    (vectors of n values, or None): (tokens int32 [n], the probability each was drawn with, fp32 [n])."""
    _need(logits.is_cuda and logits.dim() == 2 and logits.dtype == torch.float32 and
          (logits.stride(1) == 1 or logits.shape[1] == 1), "logits: expected fp32 [n, vocab] with contiguous rows")
    n, vocab = logits.shape
    dev = logits.get_device()
    token = torch.empty((n,), dtype=torch.int32, device=logits.device)
    prob = torch.empty((n,), dtype=torch.float32, device=logits.device)
    _call(dev, _L.load().ijb_sample, logits.data_ptr(), max(logits.stride(0), vocab) if n <= 1 else logits.stride(0), n,
          vocab, _ptr(u, torch.float32, n, dev, "u"), _ptr(temperature, torch.float32, n, dev, "temperature"),
          _ptr(top_k, torch.int32, n, dev, "top_k"), _ptr(top_p, torch.float32, n, dev, "top_p"),
          _ptr(min_p, torch.float32, n, dev, "min_p"), token.data_ptr(), prob.data_ptr())
    return token, prob
