"""A paged KV cache held in 4 bits, its attention, and its pages on the device.

``Int4PagedCache`` holds the K / V of many sequences in 4-bit codes with one
fp16 (scale, zero) pair per token and channel group, quantised when a token
arrives (the reference's INT4 tier, akv/fused_attention.py:213-317, is
quantised in bulk and dequantised to be read).  Every layer has its own pool
of pages (32 tokens x all KV heads); one page table serves all layers.

A serving step is

    granted = cache.reserve(rows, n_new)        # pages, lengths
    for layer in ...:
        cache.append(layer, k, v, rows, granted)
        out = cache.attend(layer, q, rows, granted)
    cache.truncate(rows, kept_lengths)          # rejected drafts

and ``fork`` / ``free`` / ``compact`` manage whole sequences.  Page tables,
lengths and reference counts live on the device and every call is a few
launches on the current stream: nothing waits for the host, so accepted
counts that only the device knows drive the next step, and a step can be
captured in a CUDA graph.  Errors found on the device (a bad row, an exhausted
pool) go to ``cache.status``; ``check()`` reads it.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from . import _C

BLOCK = _C.BLOCK_TOKENS
_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_ROWS_PER_CALL = 1024  # requests one reserve plan holds


def _half_dtype(*tensors) -> int:
    d = tensors[0].dtype
    if d not in (torch.float16, torch.bfloat16) or any(t.dtype != d for t in tensors):
        raise TypeError(f"fp16 or bf16 tensors of one type wanted (got {[str(t.dtype) for t in tensors]})")
    return _DTYPES[d]


class Int4PagedCache:
    """``n_layers`` pools of ``n_pages`` pages for ``max_seqs`` sequences of up to ``max_blocks`` pages.

    ``group_size`` channels share a scale and zero: head_dim (default),
    head_dim / 2 or head_dim / 4; head_dim 64, 128 or 256."""

    def __init__(self, n_layers: int, n_pages: int, kv_heads: int, head_dim: int, group_size: Optional[int] = None,
                 max_seqs: int = 64, max_blocks: int = 1024, device="cuda"):
        group_size = head_dim if group_size is None else group_size
        self.layout = _C.int4_layout(head_dim, group_size)
        if min(n_layers, n_pages, kv_heads, max_seqs, max_blocks) <= 0:
            raise ValueError("layers, pages, heads, sequences and blocks must be positive")
        self.n_layers, self.n_pages, self.H, self.D, self.group = n_layers, n_pages, kv_heads, head_dim, group_size
        self.max_seqs, self.max_blocks = max_seqs, max_blocks
        self.rec = self.layout.bytes
        self.buf = torch.zeros(n_layers, n_pages, kv_heads, self.rec, dtype=torch.uint8, device=device)
        # the bookkeeping in one buffer, so that it is saved and restored by one copy
        words = (n_pages + 31) // 32
        sizes = (max_seqs * max_blocks, max_seqs, n_pages, words)
        self._state = torch.zeros(sum(sizes), dtype=torch.int32, device=device)
        t, self.lens, self.refs, self.free_bits = self._state.split(sizes)
        self.table = t.view(max_seqs, max_blocks)
        self.table.fill_(-1)
        self._rebuild_free()
        self.status = torch.zeros(1, dtype=torch.int32, device=device)
        self._pt = _C.PageTable(self.table.data_ptr(), max_blocks, self.lens.data_ptr(), self.refs.data_ptr(),
                                self.free_bits.data_ptr(), max_seqs, max_blocks, n_pages)
        self._ws: dict = {}
        self._views = [self._view(layer) for layer in range(n_layers)]

    # ------------------------------------------------------------------ state
    @property
    def device(self):
        return self.buf.device

    def _view(self, layer: int) -> "_C.Int4Cache":
        return _C.Int4Cache(self.buf[layer].data_ptr(), self.buf.stride(1), self.buf.stride(2), self.n_pages,
                            self.table.data_ptr(), self.max_blocks, self.lens.data_ptr(), self.max_seqs,
                            self.max_blocks, self.H, self.D, self.group)

    def _rebuild_free(self) -> None:
        free = torch.zeros(self.free_bits.numel() * 32, dtype=torch.int64, device=self.device)
        free[:self.n_pages] = (self.refs == 0).long()
        w = (free.view(-1, 32) << torch.arange(32, device=self.device)).sum(1)
        self.free_bits.copy_(torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32))

    def page_state(self) -> torch.Tensor:
        """A copy of the bookkeeping (tables, lengths, reference counts, free pages)."""
        return self._state.clone()

    def set_page_state(self, state: torch.Tensor) -> None:
        """The bookkeeping put back as ``page_state`` returned it (the pages' bytes are not touched)."""
        self._state.copy_(state)

    def load_state(self, buf: torch.Tensor, table: torch.Tensor, lens: torch.Tensor) -> None:
        """Take over pages, table and lengths (a checkpoint's ``buf``, ``table``, ``lens``); the reference
        counts follow from the table."""
        if buf.shape != self.buf.shape or table.shape != self.table.shape or lens.shape != self.lens.shape:
            raise ValueError("the state's shapes do not match the cache")
        t = table.to(self.device)
        used = torch.arange(self.max_blocks, device=self.device)[None, :] < \
            ((lens.to(self.device).long() + BLOCK - 1) // BLOCK)[:, None]
        pages = t[used].long()
        if pages.numel() and (int(pages.min()) < 0 or int(pages.max()) >= self.n_pages):
            raise ValueError("the table names a page outside the pool")
        self.buf.copy_(buf)
        self.table.copy_(torch.where(used, t, -1))
        self.lens.copy_(lens)
        self.refs.zero_()
        self.refs.index_add_(0, pages, torch.ones_like(pages, dtype=torch.int32))
        self._rebuild_free()

    def check(self) -> None:
        """Wait for the device and raise if an operation reported an error since the last check."""
        code = int(self.status.item())
        if code:
            self.status.zero_()
            raise RuntimeError(f"int4 cache: {_C.ERRORS.get(code, code)} ({_C.strerror(code)})")

    def free_pages(self) -> int:
        """Pages without a holder (waits for the device)."""
        return int((self.refs == 0).sum())

    def resident_bytes(self) -> int:
        return self.buf.numel()

    # ------------------------------------------------------------------ arguments
    def _ints(self, x, what: str, n: Optional[int] = None) -> Optional[torch.Tensor]:
        """A contiguous int32 vector on the cache's device (lists are copied over)."""
        if x is None:
            return None
        if not torch.is_tensor(x):
            x = torch.tensor(x, dtype=torch.int32, device=self.device)
        if x.device != self.device:
            raise ValueError(f"{what} must be on {self.device}")
        if x.dtype != torch.int32 or x.dim() != 1:
            raise ValueError(f"{what} must be an int32 vector")
        if n is not None and x.numel() != n:
            raise ValueError(f"{what} needs {n} entries (got {x.numel()})")
        return x if x.is_contiguous() else x.contiguous()

    def _layer(self, layer: int) -> "_C.Int4Cache":
        if not 0 <= layer < self.n_layers:
            raise ValueError(f"layer {layer} of {self.n_layers}")
        return self._views[layer]

    def _count(self, rows, n: int) -> None:
        if rows is None and n > self.max_seqs:
            raise ValueError(f"{n} rows, but the cache holds {self.max_seqs} sequences")

    def _workspace(self, need: int, stream: int) -> torch.Tensor:
        """Zeroed scratch for attention on a stream: kept per stream (calls on two streams may overlap), its own
        for each call of a captured graph (replays may overlap eager calls)."""
        if torch.cuda.is_current_stream_capturing():
            return torch.zeros(need, dtype=torch.uint8, device=self.device)
        ws = self._ws.get(stream)
        if ws is None or ws.numel() < need:
            ws = self._ws[stream] = torch.zeros(max(need, 1 << 20), dtype=torch.uint8, device=self.device)
        return ws

    # ------------------------------------------------------------------ pages
    def reserve(self, rows, n_new) -> torch.Tensor:
        """Room for ``n_new`` (int32 vector, or one number for all) more tokens in each of ``rows`` (None: all,
        in order), the lengths advanced.  Returns the tokens granted per row, n_new or 0 where the request was
        refused: pass it to ``append`` and ``attend`` as their ``n_new``."""
        lib = _C.load()
        rows = self._ints(rows, "rows")
        n = self.max_seqs if rows is None else rows.numel()
        one = isinstance(n_new, int)
        if one and n_new < 0:
            raise ValueError("n_new is negative")
        if rows is None and n > _ROWS_PER_CALL:
            rows = torch.arange(n, dtype=torch.int32, device=self.device)
        counts = None if one else self._ints(n_new, "n_new", n)
        granted = torch.empty(n, dtype=torch.int32, device=self.device)
        need = _C.workspace_bytes("akv_pages_workspace_bytes", self.n_pages, min(n, _ROWS_PER_CALL))
        ws = torch.empty(need, dtype=torch.uint8, device=self.device)
        for a in range(0, n, _ROWS_PER_CALL):
            b = min(n, a + _ROWS_PER_CALL)
            rc = lib.akv_pages_reserve(
                ctypes.byref(self._pt), None if rows is None else rows.data_ptr() + 4 * a,
                None if one else counts.data_ptr() + 4 * a, n_new if one else 0, b - a, granted.data_ptr() + 4 * a,
                self.buf.data_ptr(), self.n_layers, self.buf.stride(0), self.buf.stride(1), ws.data_ptr(), need,
                self.status.data_ptr(), _C.stream_of(self.buf))
            _C.check(rc, "akv_pages_reserve")
        return granted

    def fork(self, parents, children) -> None:
        """Row ``children[i]`` (empty) continues row ``parents[i]``: it shares the parent's pages, and whichever
        of them next writes into a shared, partly filled page gets its own copy (``reserve``)."""
        parents = self._ints(parents, "parents")
        children = self._ints(children, "children", parents.numel())
        _C.check(_C.load().akv_pages_fork(ctypes.byref(self._pt), parents.data_ptr(), children.data_ptr(),
                                          parents.numel(), self.status.data_ptr(), _C.stream_of(self.buf)),
                 "akv_pages_fork")

    def truncate(self, rows, new_lens) -> None:
        """Rows shortened to ``new_lens`` tokens (int32 vector); pages beyond go back to the pool."""
        rows = self._ints(rows, "rows")
        n = self.max_seqs if rows is None else rows.numel()
        new_lens = self._ints(new_lens, "new_lens", n)
        _C.check(_C.load().akv_pages_truncate(ctypes.byref(self._pt), _C.ptr(rows), _C.ptr(new_lens), n,
                                              self.status.data_ptr(), _C.stream_of(self.buf)), "akv_pages_truncate")

    def free(self, rows) -> None:
        """The sequences' pages given back, their rows empty."""
        rows = self._ints(rows, "rows")
        n = self.max_seqs if rows is None else rows.numel()
        _C.check(_C.load().akv_pages_truncate(ctypes.byref(self._pt), _C.ptr(rows), None, n, self.status.data_ptr(),
                                              _C.stream_of(self.buf)), "akv_pages_truncate")

    def compact(self) -> torch.Tensor:
        """Live pages moved to the low end of the pool, tables following.  Returns their number (int32, device)."""
        live = torch.empty(1, dtype=torch.int32, device=self.device)
        need = _C.workspace_bytes("akv_pages_workspace_bytes", self.n_pages, 0)
        ws = torch.empty(need, dtype=torch.uint8, device=self.device)
        rc = _C.load().akv_pages_compact(ctypes.byref(self._pt), self.buf.data_ptr(), self.n_layers,
                                         self.buf.stride(0), self.buf.stride(1), live.data_ptr(), ws.data_ptr(), need,
                                         self.status.data_ptr(), _C.stream_of(self.buf))
        _C.check(rc, "akv_pages_compact")
        return live

    def copy_pages(self, src, dst) -> None:
        """The bytes of pages ``src`` copied over pages ``dst`` in every layer (no page in both)."""
        src = self._ints(src, "src")
        dst = self._ints(dst, "dst", src.numel())
        _C.check(_C.load().akv_pages_copy(self.buf.data_ptr(), self.n_layers, self.buf.stride(0), self.buf.stride(1),
                                          self.n_pages, src.data_ptr(), dst.data_ptr(), src.numel(),
                                          self.status.data_ptr(), _C.stream_of(self.buf)), "akv_pages_copy")

    # ------------------------------------------------------------------ tokens
    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, rows=None, n_new=None) -> None:
        """Quantise the newest tokens of each row into its pages (``reserve`` made the room).

        k, v (R, kv_heads, M, head_dim) fp16 or bf16, any strides: row i's last ``n_new[i]`` tokens (None: M)
        are k[i, :, :n_new[i]]."""
        view = self._layer(layer)
        _C.require_cuda(k, v)
        dt = _half_dtype(k, v)
        if k.shape != v.shape or k.dim() != 4 or k.shape[1] != self.H or k.shape[3] != self.D:
            raise ValueError(f"k and v must be (rows, {self.H}, tokens, {self.D})")
        k = k if k.stride(-1) == 1 else k.contiguous()
        v = v if v.stride(-1) == 1 else v.contiguous()
        R, _, M, _ = k.shape
        rows, n_new = self._ints(rows, "rows", R), self._ints(n_new, "n_new", R)
        self._count(rows, R)
        rc = _C.load().akv_int4_append(ctypes.byref(view), _C.ptr(rows), _C.ptr(n_new), R, M,
                                       k.data_ptr(), k.stride(0), k.stride(1), k.stride(2),
                                       v.data_ptr(), v.stride(0), v.stride(1), v.stride(2), dt,
                                       self.status.data_ptr(), _C.stream_of(k))
        _C.check(rc, "akv_int4_append")

    def read(self, layer: int, n_tokens: int, rows=None, start=None, n_new=None, dtype=torch.float16):
        """The K and V values the cache stands for, (R, kv_heads, n_tokens, head_dim) in ``dtype``: tokens
        ``start[i]`` onwards of each row, or with ``start`` None its last ``n_new[i]`` (None: n_tokens); 0 past
        the row's end."""
        view = self._layer(layer)
        if dtype not in (torch.float16, torch.bfloat16):
            raise TypeError(f"dtype must be fp16 or bf16 (got {dtype})")
        if n_tokens < 0:
            raise ValueError("n_tokens is negative")
        rows = self._ints(rows, "rows")
        given = [x for x in (rows, start, n_new) if x is not None]
        R = len(given[0]) if given else self.max_seqs
        start, n_new = self._ints(start, "start", R), self._ints(n_new, "n_new", R)
        self._count(rows, R)
        k = torch.empty(R, self.H, n_tokens, self.D, dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        rc = _C.load().akv_int4_read(ctypes.byref(view), _C.ptr(rows), _C.ptr(start), _C.ptr(n_new), R, n_tokens,
                                     k.data_ptr(), k.stride(0), k.stride(1), k.stride(2),
                                     v.data_ptr(), v.stride(0), v.stride(1), v.stride(2), _DTYPES[dtype],
                                     self.status.data_ptr(), _C.stream_of(self.buf))
        _C.check(rc, "akv_int4_read")
        return k, v

    def attend(self, layer: int, query: torch.Tensor, rows=None, n_new=None, sm_scale: Optional[float] = None,
               out: Optional[torch.Tensor] = None, return_lse: bool = False):
        """softmax(q K^T * sm_scale) V of each row's newest tokens over its sequence, causal by position.

        query (R, Hq, M, head_dim), or (R, Hq, head_dim) for one token, fp16 or bf16, any strides: query m of
        row i is its token lens - n_new[i] + m (``n_new`` None: M) and sees the tokens up to itself.  Queries
        past n_new[i] give zero rows.  Returns the output in the query's shape and type, and with
        ``return_lse`` the natural-log LSE (R, Hq, M) fp32."""
        view = self._layer(layer)
        _C.require_cuda(query)
        dt = _half_dtype(query)
        q = query.unsqueeze(2) if query.dim() == 3 else query
        if q.dim() != 4 or q.shape[3] != self.D or q.shape[1] % self.H:
            raise ValueError(f"query must be (rows, a multiple of {self.H} heads, tokens, {self.D})")
        q = q if q.stride(-1) == 1 else q.contiguous()
        R, Hq, M, D = q.shape
        rows, n_new = self._ints(rows, "rows", R), self._ints(n_new, "n_new", R)
        self._count(rows, R)
        if out is None:
            o = torch.empty(R, Hq, M, D, dtype=q.dtype, device=q.device)
        else:
            o = out.unsqueeze(2) if out.dim() == 3 else out
            if o.shape != q.shape or o.dtype != q.dtype or o.stride(-1) != 1 or o.device != q.device:
                raise ValueError("out must have the query's shape, type and device, its last dim contiguous")
        lse = torch.empty(R, Hq, M, dtype=torch.float32, device=q.device) if return_lse else None
        lib = _C.load()
        need = _C.workspace_bytes("akv_int4_attention_workspace_bytes", R, M, Hq, self.H, D, self.max_blocks)
        stream = _C.stream_of(q)
        ws = self._workspace(need, stream)
        rc = lib.akv_int4_attention(ctypes.byref(view), _C.ptr(rows), _C.ptr(n_new), R, M, Hq,
                                    q.data_ptr(), q.stride(0), q.stride(1), q.stride(2),
                                    1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale),
                                    o.data_ptr(), o.stride(0), o.stride(1), o.stride(2), _C.ptr(lse), dt,
                                    ws.data_ptr(), need, self.status.data_ptr(), stream)
        _C.check(rc, "akv_int4_attention")
        res = o.squeeze(2) if query.dim() == 3 else o
        return (res, lse) if return_lse else res
