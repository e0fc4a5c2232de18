"""Paged key/value cache: ragged batches, prompts of any length, shared prefixes.

``PagedKVCache`` wraps the two page pools of one layer and ``PagedBatch`` the
device tensors that say which rows each sequence owns; the three operators run
``libcbq``'s kernels (``cbq_paged_*`` in ``include/cbq.h``) on the caller's
current stream:

* ``append_rope`` -- q/k RMSNorm and rotary embedding of the new tokens, keys
  and values written to their rows;
* ``attend_decode`` -- one new token per sequence over its group's prefix
  (computed once for the whole group) and its own rows;
* ``attend_extend`` -- any number of new tokens per sequence, causally.

Lengths and tables stay on the device and may be updated in place between
calls, so a step can be captured in a CUDA graph.  No counterpart in the
reference, which uses HF's cache and attention.
"""
from __future__ import annotations

import ctypes as ct
import struct
from typing import Optional

import torch

from . import _lib

__all__ = ["PagedKVCache", "PagedBatch"]

# Zero-filled scratch of the attention calls, one growing buffer per stream: calls
# on one stream do not overlap (the library keeps a call's launches together,
# whatever other host threads do), and each leaves its arrival counters zero.
_WORKSPACES = {}

_F32 = torch.float32
_FUNCTIONS = {}

_CODES = {torch.float32: _lib.CBQ_F32, torch.bfloat16: _lib.CBQ_BF16}


def _run(name: str, *args) -> None:
    """A libcbq call, its function looked up once (these calls are short)."""
    f = _FUNCTIONS.get(name)
    if f is None:
        f = _FUNCTIONS[name] = getattr(_lib.lib(), name)
    rc = f(*args)
    if rc != _lib.CBQ_OK:
        raise _lib.CbqError(name, rc)


# torch.cuda.current_stream builds a Stream object; the raw handle is all that is passed on
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)
_capturing = torch.cuda.is_current_stream_capturing
_current = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _ints(t: Optional[torch.Tensor], name: str, ndim: int, device: torch.device) -> Optional[torch.Tensor]:
    if t is None:
        return None
    _need(isinstance(t, torch.Tensor) and t.dtype == torch.int32 and t.dim() == ndim,
          f"{name}: int32 tensor of {ndim} dimension(s) expected")
    _need(t.device == device, f"{name}: on {t.device}, expected {device}")
    _need(t.shape[-1] <= 1 or t.stride(-1) == 1, f"{name}: last dimension must be contiguous")
    return t


def _row_stride(t: torch.Tensor, name: str) -> int:
    """Entries from row to row of a table (a single row has none to step to).
    Rows that overlap (an expanded row has stride 0) are not a layout the kernels take."""
    n, width = t.shape
    if n <= 1:
        return width
    _need(t.stride(0) >= width, f"{name}: rows {t.stride(0)} entries apart overlap ({width} wide); make it contiguous")
    return t.stride(0)


class _Held:
    """The kernels read the tensors by the addresses that they had when the
    object was made: an attribute cannot be set to another tensor later."""

    def __setattr__(self, name: str, value) -> None:
        if name in self.__dict__ and self.__dict__[name] is not value:      # ``b.kv_lens += 1`` sets the same one
            raise AttributeError(f"{name} is read by its address: write into it in place, or make a new object")
        object.__setattr__(self, name, value)


class PagedBatch(_Held):
    """The sequences of a step.

    ``page_table`` int32 [seqs, width], ``kv_lens`` int32 [seqs] (rows of each
    sequence, its new tokens included); ``cu_tokens`` int32 [seqs + 1]: where
    each sequence's new tokens begin (None: one token each); tokens outside
    ``cu_tokens[0] .. cu_tokens[-1] - 1`` belong to no sequence (a captured
    step may hold fewer than it was captured for).  Shared prefixes:
    group g holds the sequences ``group_starts[g] .. group_starts[g+1] - 1``
    and its prefix the first ``prefix_lens[g]`` rows of the pages in
    ``prefix_table[g]``; a sequence in no group has none.  ``max_kv_len`` / ``max_prefix_len`` bound the values
    the two length tensors will ever hold (default: what the tables can name).
    ``status`` int32 [4]: what calls record there, see :func:`check_status`
    (None: one of the batch's own; :meth:`check` reads it).
    The tensors are kept, not copied: write new values into them in place."""

    def __init__(self, page_table: torch.Tensor, kv_lens: torch.Tensor, cu_tokens: Optional[torch.Tensor] = None,
                 group_starts: Optional[torch.Tensor] = None, prefix_lens: Optional[torch.Tensor] = None,
                 prefix_table: Optional[torch.Tensor] = None, max_kv_len: Optional[int] = None,
                 max_prefix_len: Optional[int] = None, status: Optional[torch.Tensor] = None):
        dev = page_table.device
        self.device = dev
        self.page_table = _ints(page_table, "page_table", 2, dev)
        self.kv_lens = _ints(kv_lens, "kv_lens", 1, dev)
        self.cu_tokens = _ints(cu_tokens, "cu_tokens", 1, dev)
        self.group_starts = _ints(group_starts, "group_starts", 1, dev)
        self.prefix_lens = _ints(prefix_lens, "prefix_lens", 1, dev)
        self.prefix_table = _ints(prefix_table, "prefix_table", 2, dev)
        _ints(status, "status", 1, dev)
        self.seqs = n = kv_lens.shape[0]
        _need(page_table.shape[0] == n, f"page_table has {page_table.shape[0]} rows for {n} sequences")
        _need(cu_tokens is None or cu_tokens.shape[0] == n + 1, "cu_tokens must have one entry more than kv_lens")
        shared = (group_starts is None, prefix_lens is None, prefix_table is None)
        _need(len(set(shared)) == 1, "group_starts, prefix_lens and prefix_table come together")
        groups = 0
        if prefix_lens is not None:
            groups = prefix_lens.shape[0]
            _need(group_starts.shape[0] == groups + 1 and prefix_table.shape[0] == groups,
                  "group_starts needs one entry more than prefix_lens, prefix_table one row for each")
        _need(status is None or status.shape[0] == 4, "status must have four entries")
        self.status = status = self.new_status(dev) if status is None else status
        self.groups = groups
        ptr = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
        big = 0x7fffff00
        raw = struct.pack(
            "<qqqqqqqqqqqqqqq", n, ptr(cu_tokens), ptr(kv_lens), ptr(page_table), page_table.shape[1],
            _row_stride(page_table, "page_table"), big if max_kv_len is None else int(max_kv_len), groups,
            ptr(group_starts), ptr(prefix_lens), ptr(prefix_table), prefix_table.shape[1] if groups else 0,
            _row_stride(prefix_table, "prefix_table") if groups else 0,
            big if max_prefix_len is None else int(max_prefix_len), ptr(status))
        self._desc = ct.create_string_buffer(raw, len(raw))
        self._addr = ct.addressof(self._desc)
        self._ws = {}                      # (cache layout, tokens, heads, extend) -> workspace bytes

    @staticmethod
    def new_status(device) -> torch.Tensor:
        """A status word for ``status=``: flags, first row, count, spare."""
        s = torch.zeros(4, dtype=torch.int32, device=device)
        s[1] = -1
        return s

    def check(self) -> None:
        """:func:`check_status` of this batch's calls (reads the device)."""
        check_status(self.status)


def check_status(status: torch.Tensor) -> None:
    """Raise if a call recorded a device-side wait that ran out (its result is
    not to be used) or lengths or pages outside the tables (reads the device)."""
    flags = int(status[0].item())
    if flags & _lib.FLAG_TIMEOUT:
        raise _lib.CbqError("paged cache", _lib.CBQ_ERR_TIMEOUT)
    if flags:
        raise _lib.CbqError("paged cache", _lib.CBQ_ERR_CORRUPT)


class PagedKVCache(_Held):
    """One layer's keys and values: ``k_pages``, ``v_pages`` [pages, kv_heads,
    page_size, head_dim] (fp32 or bf16, head_dim contiguous, equal strides; a
    pool stored as [pages, page_size, kv_heads, head_dim] is passed transposed)."""

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor):
        if not k_pages.is_cuda:
            raise RuntimeError("the paged cache lives on a CUDA device; there is no CPU fallback")
        _need(k_pages.dim() == 4, "pools are [pages, kv_heads, page_size, head_dim]")
        _need(k_pages.dtype in _CODES, f"cache dtype {k_pages.dtype}: float32 or bfloat16 expected")
        _need(v_pages.shape == k_pages.shape and v_pages.dtype == k_pages.dtype and
              v_pages.stride() == k_pages.stride() and v_pages.device == k_pages.device,
              "k_pages and v_pages must agree in shape, strides, dtype and device")
        _need(k_pages.stride(3) == 1, "head_dim must be contiguous")
        self.k_pages, self.v_pages = k_pages, v_pages
        self.device, self.dtype = k_pages.device, k_pages.dtype
        self.pages, self.kv_heads, self.page_size, self.head_dim = k_pages.shape
        st = k_pages.stride()
        raw = struct.pack("<qqqqqqqqqq", k_pages.data_ptr(), v_pages.data_ptr(), *k_pages.shape, st[0], st[1], st[2],
                          _CODES[k_pages.dtype])
        self._desc = ct.create_string_buffer(raw, len(raw))
        self._addr = ct.addressof(self._desc)
        self._key = (tuple(k_pages.shape), st, self.dtype)      # what a plan depends on
        self._index = k_pages.get_device()

    def _batch(self, batch: PagedBatch) -> None:
        """The kernels dereference the batch's addresses: they have to be this device's."""
        if batch.device != self.device:
            raise ValueError(f"the batch is on {batch.device}, the cache on {self.device}")

    def _rows(self, t: torch.Tensor, name: str, heads: int) -> int:
        """Checks [tokens, heads, head_dim] of the cache's dtype, heads and
        head_dim contiguous; the stride from token to token."""
        n, h, d = t.shape
        st = t.stride()
        if d != self.head_dim or h != heads:
            raise ValueError(f"{name}: [tokens, {heads}, {self.head_dim}] expected, got {tuple(t.shape)}")
        if t.dtype is not self.dtype or t.get_device() != self._index:
            raise ValueError(f"{name}: {t.dtype} on {t.device}, the cache is {self.dtype} on {self.device}")
        if st[2] != 1 or (st[1] != d and h != 1):
            raise ValueError(f"{name}: the heads of a token must be contiguous")
        return st[0] if n > 1 else h * d

    def append_rope(self, batch: PagedBatch, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor,
                    sin: torch.Tensor, eps: float = 1e-6, q_weight: Optional[torch.Tensor] = None,
                    k_weight: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Normalise and rotate q [tokens, heads, d] and k [tokens, kv_heads, d]
        at the tokens' positions, write k and v to the cache, return the rotated
        q.  ``eps`` < 0: no RMSNorm; weights fp32 [d] or None (ones); cos / sin
        fp32 [positions, d] (``qwen3_decode.rope_tables``)."""
        if _current() != self._index:                  # the library launches on the current device
            with torch.cuda.device(self._index):
                return self.append_rope(batch, q, k, v, cos, sin, eps, q_weight, k_weight, out)
        self._batch(batch)
        tokens, heads, d = q.shape
        qs, ks, vs = self._rows(q, "q", heads), self._rows(k, "k", self.kv_heads), self._rows(v, "v", self.kv_heads)
        if k.shape[0] != tokens or v.shape[0] != tokens:
            raise ValueError("q, k and v must have the same tokens")
        length = cos.shape[0]
        for t in (cos, sin):
            if t.shape != (length, d) or t.dtype is not _F32 or not t.is_contiguous() or t.get_device() != self._index:
                raise ValueError(f"cos and sin: contiguous float32 [positions, {d}] on {self.device} expected")
        for w in (q_weight, k_weight):
            if w is not None and (w.shape != (d,) or w.dtype is not _F32 or not w.is_contiguous() or
                                  w.get_device() != self._index):
                raise ValueError(f"q_weight and k_weight: contiguous float32 [{d}] on {self.device} expected")
        if out is None:
            out = q.new_empty((tokens, heads, d))
        else:
            self._out(out, tokens, heads)
        _run("cbq_paged_append_rope", self._addr, batch._addr, tokens, q.data_ptr(), qs, k.data_ptr(),
             ks, v.data_ptr(), vs, heads, eps, None if q_weight is None else q_weight.data_ptr(),
             None if k_weight is None else k_weight.data_ptr(), cos.data_ptr(), sin.data_ptr(), length, out.data_ptr(),
             _stream(self._index))
        return out

    def _out(self, out: torch.Tensor, tokens: int, heads: int) -> None:
        _need(out.shape == (tokens, heads, self.head_dim) and out.dtype == self.dtype and out.is_contiguous() and
              out.device == self.device, f"out: contiguous [{tokens}, {heads}, {self.head_dim}] of the cache's dtype")

    def workspace_bytes(self, batch: PagedBatch, tokens: int, heads: int, extend: bool) -> int:
        """Bytes of the zero-filled scratch one attention call needs; a
        ``workspace=`` tensor may serve calls of any shape that do not overlap."""
        if _current() != self._index:
            with torch.cuda.device(self._index):
                return self.workspace_bytes(batch, tokens, heads, extend)
        self._batch(batch)
        key = (self._key, tokens, heads, extend)
        n = batch._ws.get(key)
        if n is None:
            n = _lib.query("cbq_paged_attn_workspace_bytes", self._addr, batch._addr, tokens, heads, int(extend))
            batch._ws[key] = n
        return n

    def _attend(self, name: str, extend: bool, batch: PagedBatch, q: torch.Tensor, scale: Optional[float],
                out: Optional[torch.Tensor], workspace: Optional[torch.Tensor]) -> torch.Tensor:
        if _current() != self._index:
            with torch.cuda.device(self._index):
                return self._attend(name, extend, batch, q, scale, out, workspace)
        self._batch(batch)
        tokens, heads, d = q.shape
        stride = self._rows(q, "q", heads)
        if out is None:
            out = q.new_empty((tokens, heads, d))
        else:
            self._out(out, tokens, heads)
        stream = _stream(self._index)
        if workspace is None:
            workspace = self._scratch(stream, self.workspace_bytes(batch, tokens, heads, extend))
        elif (workspace.device != self.device or workspace.dtype is not torch.uint8 or
              not workspace.is_contiguous()):
            raise ValueError(f"workspace: contiguous uint8 on {self.device} expected")
        _run(name, self._addr, batch._addr, tokens, q.data_ptr(), stride, heads, d ** -0.5 if scale is None else scale,
             out.data_ptr(), workspace.data_ptr(), workspace.numel(), stream)
        return out

    def _scratch(self, stream: int, need: int) -> torch.Tensor:
        """Zero-filled scratch for calls on ``stream``; inside a graph capture a
        buffer of the graph's own, which its replays clear."""
        if _capturing():
            return torch.zeros(need, dtype=torch.uint8, device=self.device)
        key = (self._index, stream)
        ws = _WORKSPACES.get(key)
        if ws is None or ws.numel() < need:
            ws = _WORKSPACES[key] = torch.zeros(need + need // 2, dtype=torch.uint8, device=self.device)
        return ws

    def attend_decode(self, batch: PagedBatch, q: torch.Tensor, scale: Optional[float] = None,
                      out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
        """q [seqs, heads, d], one token per sequence (``cu_tokens`` is not
        read) -> [seqs, heads, d]: softmax(q k^T scale) v over the group's
        prefix and the sequence's rows (``scale`` None: d^-1/2); zeros where
        there is nothing to read."""
        return self._attend("cbq_paged_attn_decode", False, batch, q, scale, out, workspace)

    def attend_extend(self, batch: PagedBatch, q: torch.Tensor, scale: Optional[float] = None,
                      out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
        """q [tokens, heads, d], the sequences' new tokens one after the other
        (``cu_tokens``) -> [tokens, heads, d]; token i of sequence s sees the
        prefix and the rows up to its own; tokens of no sequence give zeros."""
        return self._attend("cbq_paged_attn_extend", True, batch, q, scale, out, workspace)
