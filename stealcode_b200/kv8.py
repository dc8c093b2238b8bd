"""A paged 8-bit key/value cache on the device, and attention over it.

``KvCache8`` holds the keys and values of many sequences in int8 with one f32
scale per block of tokens and kv head, in pages that sequences can share
(C ABI: ``sc_kv8_*``).  One step of some sequences is::

    cache.reserve(counts)                      # pages for the new tokens; lengths grow
    for layer in range(n_layers):
        cache.append(layer, k, v, n=1)         # quantise their keys and values
        out = cache.attend(layer, q, n=1)      # attention over their whole past
    cache.slide(window, sinks)                 # give back what left the window

``append``, ``attend`` and ``rows`` work on the last tokens of each sequence.
Their rows are packed: ``n`` rows for each sequence, or, with ``cu`` (int32
CUDA tensor [m + 1]), rows ``cu[i] .. cu[i + 1]`` for the i-th, at most ``n``
each.  Rows before ``cu[0]`` and from ``cu[m]`` on belong to no sequence: they
are not touched, and hold anything in an output that the call allocates.  ``seqs`` (int32 CUDA tensor [m]) names the sequences; None means
sequences 0, 1, ...

Everything runs on the current torch stream (or ``stream``) without a copy to
the host; failures that only the device sees (too few free pages) are read with
``check()``.  Calls can be captured in a CUDA graph once the same kind of call
has run on that stream: the first one makes the stream's workspace.  A graph
keeps the workspace of the stream that it was captured on: wherever it is
replayed, the replay has to be ordered against every other call and replay that
uses that workspace (capture on a stream of its own for graphs that overlap).
"""
from __future__ import annotations

import ctypes
from ctypes import c_int32, c_int64, c_void_p

import torch

from . import _lib
from ._lib import SC_ERR_ALLOC, SC_ERR_INVALID, SC_ERR_TIMEOUT, ScError, check, lib

POOL_FULL, TABLE_FULL, BAD_SEQUENCE, BAD_PAGE, WAIT_TIMEOUT, BAD_ROWS = 1, 2, 4, 8, 16, 32

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_FAILURES = (
    (POOL_FULL, SC_ERR_ALLOC, "too few free pages"),
    (TABLE_FULL, SC_ERR_ALLOC, "a sequence is longer than its table row"),
    (BAD_SEQUENCE, SC_ERR_INVALID, "a sequence id outside the cache or named twice, or a negative count"),
    (BAD_PAGE, SC_ERR_INVALID, "a page id outside the cache, or an append without a reserved page"),
    (BAD_ROWS, SC_ERR_INVALID, "cu gives an entry more than n rows, fewer than 0, or rows outside the packed ones"),
    (WAIT_TIMEOUT, SC_ERR_TIMEOUT, "a bounded device-side wait gave up"),
)


# The current stream's handle without building a torch.cuda.Stream (5 us of a 10 us call).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


class _Cache(ctypes.Structure):
    _fields_ = [(x, c_void_p) for x in ("k", "v", "k_scale", "v_scale", "table", "length", "refs", "status")] + \
               [(x, c_int64) for x in ("n_layers", "n_pages", "n_seqs", "max_pages")] + \
               [(x, c_int32) for x in ("n_kv_heads", "head_dim", "page", "block")]


class _Batch(ctypes.Structure):
    _fields_ = [("seqs", c_void_p), ("cu", c_void_p), ("m", c_int64), ("n", c_int64), ("total", c_int64)]


class KvCache8:
    """The cache's tensors (see the module's text) and the calls on them.

    ``k``, ``v`` int8 [n_layers, n_pages, n_kv_heads, page, head_dim]; ``k_scale``, ``v_scale``
    f32 [n_layers, n_pages, n_kv_heads, page // block]; ``table`` int32 [n_seqs, max_pages];
    ``length`` int32 [n_seqs]; ``refs`` int32 [n_pages]; ``status`` int32 [1]."""

    def __init__(self, n_layers: int, n_pages: int, n_kv_heads: int, head_dim: int, n_seqs: int, max_pages: int, *,
                 page: int = 64, block: int = 32, device=None):
        if page < 1 or block < 1 or page % block:
            raise ValueError(f"page {page} has to be a multiple of block {block}")
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        codes = (n_layers, n_pages, n_kv_heads, page, head_dim)
        scales = (n_layers, n_pages, n_kv_heads, page // block)
        i32 = dict(dtype=torch.int32, device=dev)
        self._take(torch.empty(codes, dtype=torch.int8, device=dev), torch.empty(codes, dtype=torch.int8, device=dev),
                   torch.empty(scales, dtype=torch.float32, device=dev),
                   torch.empty(scales, dtype=torch.float32, device=dev),
                   torch.full((n_seqs, max_pages), -1, **i32), torch.zeros(n_seqs, **i32), torch.zeros(n_pages, **i32))

    @classmethod
    def wrap(cls, k, v, k_scale, v_scale, table, length, refs) -> "KvCache8":
        """A cache over tensors that the caller holds (their contents as they are)."""
        self = cls.__new__(cls)
        self._take(k, v, k_scale, v_scale, table, length, refs)
        return self

    def _take(self, k, v, k_scale, v_scale, table, length, refs):
        if k.dim() != 5 or k.shape != v.shape or k_scale.dim() != 4 or k_scale.shape != v_scale.shape or \
                k_scale.shape[:3] != k.shape[:3]:
            raise ValueError("k, v: [layers, pages, kv heads, page, head_dim]; scales: [layers, pages, kv heads, blocks]")
        if k_scale.shape[3] < 1 or k.shape[3] % k_scale.shape[3]:
            raise ValueError(f"{k_scale.shape[3]} scales do not divide a page of {k.shape[3]} tokens")
        if table.dim() != 2 or length.shape != table.shape[:1] or refs.shape != k.shape[1:2]:
            raise ValueError("table [seqs, max_pages], length [seqs], refs [pages]")
        for t, dt in ((k, torch.int8), (v, torch.int8), (k_scale, torch.float32), (v_scale, torch.float32),
                      (table, torch.int32), (length, torch.int32), (refs, torch.int32)):
            if t.dtype != dt or not t.is_contiguous() or t.device != k.device or not t.is_cuda:
                raise ValueError("the cache's tensors have to be contiguous CUDA tensors of one device: int8 codes, "
                                 "f32 scales, int32 table, length and refs")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.table, self.length, self.refs = table, length, refs
        self.device = k.device
        self._index = k.device.index
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self.n_layers, self.n_pages, self.n_kv_heads, self.page, self.head_dim = k.shape
        self.block = self.page // k_scale.shape[3]
        self.n_seqs, self.max_pages = table.shape
        self._c = _Cache(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), table.data_ptr(),
                         length.data_ptr(), refs.data_ptr(), self.status.data_ptr(), self.n_layers, self.n_pages,
                         self.n_seqs, self.max_pages, self.n_kv_heads, self.head_dim, self.page, self.block)
        self._p = ctypes.addressof(self._c)
        self._ws = {}  # (kind, stream) -> workspace: calls on two streams share none, replays see the module's text
        self._named = set()  # streams that calls have named

    # ---- arguments ----------------------------------------------------------------

    def _stream(self, stream, *used) -> int:
        """The call's stream.  A stream that the call names reads the cache and the tensors ``used``: their
        memory is not given out again before that work is done."""
        if _current_device() != self._index:
            raise ValueError(f"the cache lives on {self.device}, the current device is {_current_device()}")
        if stream is None:
            return _raw_stream(self._index)
        st = stream.cuda_stream
        if st not in self._named:
            for t in (self.k, self.v, self.k_scale, self.v_scale, self.table, self.length, self.refs, self.status):
                t.record_stream(stream)
            self._named.add(st)
        for t in used:
            if t is not None:
                t.record_stream(stream)
        return st

    def _ids(self, t, name: str) -> int:
        if t is None:
            return 0
        if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous() or t.device != self.device:
            raise ValueError(f"{name} has to be a contiguous int32 tensor [m] on {self.device}")
        return t.data_ptr()

    def _workspace(self, kind: str, st: int, stream, need) -> tuple:
        """(address, bytes) of this stream's workspace, zeroed when it is made."""
        ws = self._ws.get((kind, st))
        if ws is None:
            with torch.cuda.stream(torch.cuda.current_stream() if stream is None else stream):
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("kv8: make one such call on this stream before a graph capture (the workspace "
                                       "would belong to the graph)")
                n = need()
                check(min(n, 0))
                buf = torch.zeros(n, dtype=torch.uint8, device=self.device)
            ws = self._ws[(kind, st)] = (buf.data_ptr(), n, buf)
        return ws

    def _batch(self, seqs, cu, n, total):
        if n is None:
            raise ValueError("n (the rows of a sequence, or with cu the most) is needed")
        if cu is not None:
            m = cu.shape[0] - 1
            if m < 0:
                raise ValueError("cu has one entry more than there are sequences")
        elif seqs is not None:
            m = seqs.shape[0]
        else:
            m = total // n if total is not None and n else self.n_seqs
        if seqs is not None and seqs.shape[0] != m:
            raise ValueError(f"{seqs.shape[0]} sequences for {m} entries of cu")
        if total is None:
            if cu is not None:
                raise ValueError("total (the packed rows) is needed with cu")
            total = m * n
        return _Batch(self._ids(seqs, "seqs"), self._ids(cu, "cu"), m, n, total)

    def _rows_in(self, t, heads: int, name: str):
        """The strides of a checked row tensor."""
        shape, strides = t.shape, t.stride()
        if len(shape) != 3 or shape[1] != heads or shape[2] != self.head_dim or t.dtype not in _DTYPES or \
                t.device != self.device or (strides[2] != 1 and t.numel()):
            raise ValueError(f"{name} has to be [rows, {heads}, {self.head_dim}] f32, f16 or bf16 on {self.device}, "
                             "dense in its last dimension")
        return strides

    # ---- rows ---------------------------------------------------------------------

    def append(self, layer: int, k, v, *, seqs=None, cu=None, n=None, stream=None) -> None:
        """Quantise k, v [rows, n_kv_heads, head_dim] into the sequences' last tokens.

        An append that fails on the device (see ``check``) leaves these tokens undefined until they are
        appended again."""
        ks, vs = self._rows_in(k, self.n_kv_heads, "k"), self._rows_in(v, self.n_kv_heads, "v")
        if k.dtype != v.dtype or k.shape != v.shape:
            raise ValueError("k and v differ in type or shape")
        b = self._batch(seqs, cu, n, k.shape[0])
        rc = lib.sc_kv8_append(self._p, layer, ctypes.byref(b), k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1],
                               _DTYPES[k.dtype], self._stream(stream, k, v, seqs, cu))
        if rc:
            check(rc)

    def rows(self, layer: int, *, seqs=None, cu=None, n=None, total=None, dtype=torch.float32, stream=None):
        """The stored values (k, v), each [rows, n_kv_heads, head_dim], of the sequences' last tokens; with
        ``cu``, ``total`` says how many rows it packs."""
        b = self._batch(seqs, cu, n, total)
        if dtype not in _DTYPES:
            raise ValueError("dtype has to be f32, f16 or bf16")
        st = self._stream(stream, seqs, cu)
        shape = (b.total, self.n_kv_heads, self.head_dim)
        if stream is None:
            k = self.k_scale.new_empty(shape, dtype=dtype)
            v = torch.empty_like(k)
        else:  # allocations belong to the stream that uses them
            with torch.cuda.stream(stream):
                k = self.k_scale.new_empty(shape, dtype=dtype)
                v = torch.empty_like(k)
        rc = lib.sc_kv8_rows(self._p, layer, ctypes.byref(b), k.data_ptr(), v.data_ptr(), _DTYPES[dtype], st)
        if rc:
            check(rc)
        return k, v

    def attend(self, layer: int, q, *, seqs=None, cu=None, n=None, max_len: int = 0, window: int = 0, sinks: int = 0,
               scale=None, out=None, return_lse: bool = False, stream=None):
        """Attention of the sequences' last tokens, q [rows, n_heads, head_dim], over the sequences.

        A query at position p sees the tokens t <= p that still have a page and, with a window,
        t > p - window or t < sinks.  Returns out (q's type and shape), and with ``return_lse`` also the
        log-sum-exp of the scores, f32 [rows, n_heads].  A query that sees nothing: 0, -inf.
        ``max_len``: no sequence is longer (sizes the launch).  ``scale``: head_dim ** -0.5 if None.
        An 8-bit cache serves and is not trained through: the result carries no gradient, whatever q does."""
        if q.dim() != 3 or q.shape[1] < 1:
            raise ValueError("q has to be [rows, n_heads, head_dim]")
        rows, heads = q.shape[:2]
        qs = self._rows_in(q, heads, "q")
        b = self._batch(seqs, cu, n, rows)
        st = self._stream(stream, q, seqs, cu)
        if out is not None:
            os_ = self._rows_in(out, heads, "out")
            if out.dtype != q.dtype or out.shape != q.shape:
                raise ValueError("out has to have q's type and shape")
            if stream is not None:
                out.record_stream(stream)
        lse = None
        if stream is None:
            if out is None:
                out = torch.empty_like(q, memory_format=torch.contiguous_format)
                os_ = out.stride()
            if return_lse:
                lse = self.k_scale.new_empty((rows, heads))
        else:  # allocations belong to the stream that uses them
            with torch.cuda.stream(stream):
                if out is None:
                    out = torch.empty_like(q, memory_format=torch.contiguous_format)
                    os_ = out.stride()
                if return_lse:
                    lse = self.k_scale.new_empty((rows, heads))
        ws = self._ws.get(("attend", st)) or self._workspace("attend", st, stream, lib.sc_kv8_attend_workspace_bytes)
        rc = lib.sc_kv8_attend(self._p, layer, ctypes.byref(b), q.data_ptr(), qs[0], qs[1], heads,
                               self.head_dim ** -0.5 if scale is None else scale, window, sinks, max_len,
                               out.data_ptr(), os_[0], os_[1], lse.data_ptr() if return_lse else None,
                               _DTYPES[q.dtype], ws[0], ws[1], st)
        if rc:
            check(rc)
        return (out, lse) if return_lse else out

    # ---- pages --------------------------------------------------------------------

    def _page_ws(self, st: int, stream):
        return self._workspace("pages", st, stream, lambda: lib.sc_kv8_page_workspace_bytes(self._p))

    def reserve(self, counts, *, seqs=None, stream=None) -> None:
        """Pages for counts[i] more tokens (int32 CUDA tensor [m]) of each sequence; the lengths grow."""
        p = self._ids(counts, "counts")
        if seqs is not None and seqs.shape != counts.shape:
            raise ValueError("seqs and counts differ in length")
        s = self._ids(seqs, "seqs")
        st = self._stream(stream, counts, seqs)
        ws = self._page_ws(st, stream)
        check(lib.sc_kv8_reserve(self._p, s, p, counts.shape[0], ws[0], ws[1], st))

    def fork(self, parents, children, *, stream=None) -> None:
        """children[i] becomes a copy of parents[i] (int32 CUDA tensors [m]; all pairs at once, so a parent
        may be a child too): full pages are shared, a partly filled last page is copied, and what a child
        held before is released."""
        a, b = self._ids(parents, "parents"), self._ids(children, "children")
        if parents.shape != children.shape:
            raise ValueError("parents and children differ in length")
        st = self._stream(stream, parents, children)
        ws = self._page_ws(st, stream)
        check(lib.sc_kv8_fork(self._p, a, b, parents.shape[0], ws[0], ws[1], st))

    def release(self, seqs=None, *, stream=None) -> None:
        """Give back the sequences' pages; their lengths become 0.  None: all sequences."""
        m = self.n_seqs if seqs is None else seqs.shape[0]
        check(lib.sc_kv8_release(self._p, self._ids(seqs, "seqs"), m, self._stream(stream, seqs)))

    def slide(self, window: int, sinks: int = 0, *, seqs=None, stream=None) -> None:
        """Give back the pages that no later query can see under this window and these sinks."""
        m = self.n_seqs if seqs is None else seqs.shape[0]
        check(lib.sc_kv8_slide(self._p, self._ids(seqs, "seqs"), m, window, sinks, self._stream(stream, seqs)))

    def compact(self, *, stream=None) -> None:
        """Move the pages in use to the lowest ids; the tables follow."""
        st = self._stream(stream)
        ws = self._page_ws(st, stream)
        check(lib.sc_kv8_compact(self._p, ws[0], ws[1], st))

    def check(self) -> None:
        """Raise ScError if a call failed on the device (synchronises); ``clear_status`` forgets it."""
        bits = int(self.status.item())
        for bit, code, text in _FAILURES:
            if bits & bit:
                raise ScError(code, f"kv8: {text} (status {bits:#x})")

    def clear_status(self) -> None:
        self.status.zero_()


__all__ = ["KvCache8"]
