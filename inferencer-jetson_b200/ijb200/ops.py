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
_current = torch._C._cuda_getDevice
_empty = torch.empty


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _call(device: int, fn, *args) -> None:
    """One library call with `device` current, on its current stream."""
    if _current() == device:
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


def _rows(t, n: int, inner: int, device: int, what: str):
    """(address, stride in elements) of [n, ..] rows, each of `inner` contiguous elements."""
    if t.is_contiguous() and t.numel() == n * inner and t.get_device() == device:
        return t.data_ptr(), inner
    flat = t.dim() == 2 and t.stride(1) == 1 or t.dim() == 3 and t.stride(2) == 1 and t.stride(1) == t.shape[2]
    if t.get_device() != device or not flat or t.numel() != n * inner or t.stride(0) < inner and n > 1:
        raise ValueError(f"{what}: expected [{n}, {inner}] values on cuda:{device}, each row's contiguous")
    return t.data_ptr(), max(t.stride(0), inner)


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
        _need(status is None or status.dtype in (torch.int32, torch.uint32) and status.numel() == 1 and status.get_device() == dev,
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
        self._scale, self._seqs = 1.0 / math.sqrt(self.head_dim), page_table.shape[0]
        with torch.cuda.device(dev):
            self._work = self._lib.ijb_paged_attention_workspace(self._ref)

    def append(self, k, v, seq, pos) -> None:
        """Writes rows k, v [n, kv_heads, head_dim] (fp32 or fp16) at positions pos [n] of sequences seq [n]."""
        n, dev = k.shape[0], self.device
        kp, stride = _rows(k, n, self.row, dev, "k")
        vp, vstride = _rows(v, n, self.row, dev, "v")
        if k.dtype not in _TYPE or v.dtype != k.dtype or vstride != stride:
            raise ValueError("k and v: expected fp32 or fp16 rows of one type and stride")
        _call(dev, self._lib.ijb_kv_append, self._ref, _TYPE[k.dtype], kp, vp, stride, n,
              _ptr(seq, torch.int32, n, dev, "seq"), _ptr(pos, torch.int32, n, dev, "pos"), self._status)

    def gather(self, seq, pos, dtype=torch.float32):
        """The rows at positions pos [n] of sequences seq [n]: (k, v), each [n, kv_heads, head_dim].
        Rows of entries that are skipped (a negative position) hold no meaning."""
        _need(dtype in _TYPE, "dtype must be float32 or float16")
        n = seq.numel()
        k = _empty((n, self.kv_heads, self.head_dim), dtype=dtype, device=self.data.device)
        v = torch.empty_like(k)
        _call(self.device, self._lib.ijb_kv_gather, self._ref, _TYPE[dtype], k.data_ptr(), v.data_ptr(), self.row, n,
              _ptr(seq, torch.int32, n, self.device, "seq"), _ptr(pos, torch.int32, n, self.device, "pos"), self._status)
        return k, v

    def attention(self, q, q_start, kv_len, seq=None, max_q: int = 0, scale: float | None = None, out=None):
        """Attention of new tokens: q [tokens, heads, head_dim] fp32 or fp16, entry e's tokens being rows
        q_start[e]..q_start[e + 1] and the last of the kv_len[e] positions of sequence seq[e] (default: e), which
        the cache already holds.  Each token sees the positions up to its own; a token before position 0 sees none and
        gets zeros.  ``max_q``: the most new tokens of any entry, if known.  Returns out (like q)."""
        if q.dim() != 3 or q.shape[2] != self.head_dim or q.dtype not in _TYPE:
            raise ValueError("q: expected [tokens, heads, head_dim], fp32 or fp16")
        n, heads, _ = q.shape
        dev, row = self.device, heads * self.head_dim
        qp, qs = _rows(q, n, row, dev, "q")
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
            op, os = out.data_ptr(), row
        else:
            _need(out.shape == q.shape and out.dtype == q.dtype, "out: expected the shape and type of q")
            op, os = _rows(out, n, row, dev, "out")
        e = kv_len.numel()
        _need(e >= 1 and (seq is not None or e <= self._seqs), "kv_len: one length for each entry")
        work = _empty(self._work, dtype=torch.uint8, device=q.device)
        _call(dev, self._lib.ijb_paged_attention, self._ref, heads, _TYPE[q.dtype], qp, qs, op, os, n, e,
              _ptr(q_start, torch.int32, e + 1, dev, "q_start"), _ptr(seq, torch.int32, e, dev, "seq"),
              _ptr(kv_len, torch.int32, e, dev, "kv_len"), max_q, self._scale if scale is None else scale,
              work.data_ptr(), self._work, self._status)
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
