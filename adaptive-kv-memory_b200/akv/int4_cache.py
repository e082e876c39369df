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
captured in a CUDA graph.  A call runs on the cache's GPU, whichever is current,
on that GPU's current stream.  Errors found on the device (a bad row, an exhausted
pool) go to ``cache.status``; ``check()`` reads it.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from . import _C

BLOCK = _C.BLOCK_TOKENS
_REQUESTS = 1024  # requests that a call may hold however few the sequences


_HALF = {torch.float16: 0, torch.bfloat16: 1}


def _half_dtype(t: torch.Tensor) -> int:
    d = _HALF.get(t.dtype)
    if d is None:
        raise TypeError(f"fp16 or bf16 wanted (got {t.dtype})")
    return d


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
        self._lib = _C.load()
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
        self._dev = self.buf.device
        # the default stream's handle, 0, does not say whose it is: every call makes this GPU current to launch
        self._dev_index = self._dev.index if self._dev.index is not None else torch.cuda.current_device()
        self._status_ptr = self.status.data_ptr()
        self._pt = _C.PageTable(self.table.data_ptr(), max_blocks, self.lens.data_ptr(), self.refs.data_ptr(),
                                self.free_bits.data_ptr(), max_seqs, max_blocks, n_pages)
        self._ws: dict = {}
        self._ws_need: dict = {}
        self._scale = 1.0 / math.sqrt(head_dim)
        self._pt_ref = ctypes.byref(self._pt)
        # the page operations of one cache follow one another (they change one table), so they share a workspace
        self._most_requests = max(_REQUESTS, max_seqs)
        self._page_ws_bytes = int(self._lib.akv_pages_workspace_bytes(n_pages, self._most_requests))
        self._page_ws = torch.empty(self._page_ws_bytes, dtype=torch.uint8, device=device)
        self._page_ws_ptr = self._page_ws.data_ptr()
        self._pool_ptr, self._layer_bytes, self._page_bytes = self.buf.data_ptr(), self.buf.stride(0), self.buf.stride(1)
        self._views = [self._view(layer) for layer in range(n_layers)]
        self._view_ptrs = [ctypes.addressof(v) for v in self._views]

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
        if state.shape != self._state.shape or state.dtype is not torch.int32:
            raise ValueError("the state does not match the cache")
        self._state.copy_(state)

    def load_state(self, buf: torch.Tensor, table: torch.Tensor, lens: torch.Tensor) -> None:
        """Take over pages, table and lengths (a checkpoint's ``buf``, ``table``, ``lens``); the reference
        counts follow from the table."""
        if buf.shape != self.buf.shape or table.shape != self.table.shape or lens.shape != self.lens.shape:
            raise ValueError("the state's shapes do not match the cache")
        if int(lens.min()) < 0 or int(lens.max()) > self.max_blocks * BLOCK:
            raise ValueError(f"a length is outside 0 to {self.max_blocks * BLOCK}")
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
        if not isinstance(x, torch.Tensor):
            x = torch.tensor(x, dtype=torch.int32, device=self._dev)
        shape = x.shape
        if x.dtype is not torch.int32 or len(shape) != 1:
            raise ValueError(f"{what} must be an int32 vector")
        if x.device != self._dev:
            raise ValueError(f"{what} must be on {self._dev}")
        if n is not None and shape[0] != n:
            raise ValueError(f"{what} needs {n} entries (got {shape[0]})")
        return x if x.is_contiguous() else x.contiguous()

    def _layer(self, layer: int) -> int:
        if not 0 <= layer < self.n_layers:
            raise ValueError(f"layer {layer} of {self.n_layers}")
        return self._view_ptrs[layer]

    def _rows(self, rows, n_new, R: int) -> tuple:
        """The row and count vectors of a call over R rows, and their pointers (0: none)."""
        if rows is not None:
            rows = self._ints(rows, "rows", R)
        elif R > self.max_seqs:
            raise ValueError(f"{R} rows, but the cache holds {self.max_seqs} sequences")
        if n_new is not None:
            n_new = self._ints(n_new, "n_new", R)
        return (rows, n_new, 0 if rows is None else rows.data_ptr(), 0 if n_new is None else n_new.data_ptr())

    def _workspace(self, need: int, stream: int) -> torch.Tensor:
        """Zeroed scratch for attention on a stream: kept per stream (calls on two streams may overlap), its own
        for each call of a captured graph (replays may overlap eager calls)."""
        if torch.cuda.is_current_stream_capturing():
            return torch.zeros(need, dtype=torch.uint8, device=self._dev)
        ws = self._ws.get(stream)
        if ws is None or ws.numel() < need:
            ws = self._ws[stream] = torch.zeros(max(need, 1 << 20), dtype=torch.uint8, device=self._dev)
        return ws

    # ------------------------------------------------------------------ pages
    def reserve(self, rows, n_new) -> torch.Tensor:
        """Room for ``n_new`` (int32 vector, or one number for all) more tokens in each of ``rows`` (None: all,
        in order), the lengths advanced.  Returns the tokens granted per row, n_new or 0 where the request was
        refused: pass it to ``append`` and ``attend`` as their ``n_new``.  When the pool runs out, that request and
        all after it are refused; so is a row that was already asked for in the call."""
        if _C.current_device() != self._dev_index:
            with torch.cuda.device(self._dev_index):
                return self.reserve(rows, n_new)
        rows = self._ints(rows, "rows")
        n = self.max_seqs if rows is None else rows.shape[0]
        counts = None
        if isinstance(n_new, int):
            if not 0 <= n_new < 1 << 31:
                raise ValueError(f"n_new must be 0 to 2^31 - 1 (got {n_new})")
        else:
            counts = self._ints(n_new, "n_new", n)
            n_new = 0
        if n > self._most_requests:
            raise ValueError(f"{n} requests for {self.max_seqs} sequences")
        granted = torch.empty_strided((n,), (1,), dtype=torch.int32, device=self._dev)
        rc = self._lib.akv_pages_reserve_many(
            self._pt_ref, _C.ptr(rows), _C.ptr(counts), n_new, n, granted.data_ptr(), self._pool_ptr, self.n_layers,
            self._layer_bytes, self._page_bytes, self._page_ws_ptr, self._page_ws_bytes, self._status_ptr,
            _C.raw_stream(self._dev_index))
        if rc:
            _C.check(rc, "akv_pages_reserve_many")
        return granted

    def fork(self, parents, children) -> None:
        """Row ``children[i]`` (empty) continues row ``parents[i]``: it shares the parent's pages, and whichever
        of them next writes into a shared, partly filled page gets its own copy (``reserve``)."""
        if _C.current_device() != self._dev_index:
            with torch.cuda.device(self._dev_index):
                return self.fork(parents, children)
        parents = self._ints(parents, "parents")
        n = parents.shape[0]
        children = self._ints(children, "children", n)
        rc = self._lib.akv_pages_fork(self._pt_ref, parents.data_ptr(), children.data_ptr(), n, self._status_ptr,
                                      _C.raw_stream(self._dev_index))
        if rc:
            _C.check(rc, "akv_pages_fork")

    def _truncate(self, rows, n: int, new_lens) -> None:
        if _C.current_device() != self._dev_index:
            with torch.cuda.device(self._dev_index):
                return self._truncate(rows, n, new_lens)
        rc = self._lib.akv_pages_truncate(self._pt_ref, _C.ptr(rows), _C.ptr(new_lens), n, self._status_ptr,
                                          _C.raw_stream(self._dev_index))
        if rc:
            _C.check(rc, "akv_pages_truncate")

    def truncate(self, rows, new_lens) -> None:
        """Rows shortened to ``new_lens`` tokens (int32 vector); pages beyond go back to the pool."""
        if new_lens is None:
            raise ValueError("new_lens is missing (free() empties rows)")
        rows = self._ints(rows, "rows")
        n = self.max_seqs if rows is None else rows.shape[0]
        self._truncate(rows, n, self._ints(new_lens, "new_lens", n))

    def free(self, rows) -> None:
        """The sequences' pages given back, their rows empty."""
        rows = self._ints(rows, "rows")
        self._truncate(rows, self.max_seqs if rows is None else rows.shape[0], None)

    def compact(self) -> torch.Tensor:
        """Live pages moved to the low end of the pool, tables following.  Returns their number (int32, device)."""
        if _C.current_device() != self._dev_index:
            with torch.cuda.device(self._dev_index):
                return self.compact()
        live = torch.empty_strided((1,), (1,), dtype=torch.int32, device=self._dev)
        rc = self._lib.akv_pages_compact(self._pt_ref, self._pool_ptr, self.n_layers, self._layer_bytes,
                                         self._page_bytes, live.data_ptr(), self._page_ws_ptr, self._page_ws_bytes,
                                         self._status_ptr, _C.raw_stream(self._dev_index))
        if rc:
            _C.check(rc, "akv_pages_compact")
        return live

    def copy_pages(self, src, dst) -> None:
        """The bytes of pages ``src`` copied over pages ``dst`` in every layer (no page in both)."""
        if _C.current_device() != self._dev_index:
            with torch.cuda.device(self._dev_index):
                return self.copy_pages(src, dst)
        src = self._ints(src, "src")
        n = src.shape[0]
        dst = self._ints(dst, "dst", n)
        rc = self._lib.akv_pages_copy(self._pool_ptr, self.n_layers, self._layer_bytes, self._page_bytes, self.n_pages,
                                      src.data_ptr(), dst.data_ptr(), n, self._status_ptr,
                                      _C.raw_stream(self._dev_index))
        if rc:
            _C.check(rc, "akv_pages_copy")

    # ------------------------------------------------------------------ tokens
    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, rows=None, n_new=None) -> None:
        """Quantise the newest tokens of each row into its pages (``reserve`` made the room).

        k, v (R, kv_heads, M, head_dim) fp16 or bf16, any strides: row i's last ``n_new[i]`` tokens (None: M)
        are k[i, :, :n_new[i]]."""
        if _C.current_device() != self._dev_index:
            with torch.cuda.device(self._dev_index):
                return self.append(layer, k, v, rows, n_new)
        view = self._layer(layer)
        dt = _half_dtype(k)
        if v.dtype is not k.dtype:
            raise TypeError(f"k and v must be of one type (got {k.dtype}, {v.dtype})")
        shape = k.shape
        if len(shape) != 4 or v.shape != shape or shape[1] != self.H or shape[3] != self.D:
            raise ValueError(f"k and v must be (rows, {self.H}, tokens, {self.D})")
        if k.device != self._dev or v.device != self._dev:
            raise RuntimeError(f"akv: k and v must be on {self._dev} (no CPU fallback)")
        ks, vs = k.stride(), v.stride()
        if ks[3] != 1:
            k = k.contiguous()
            ks = k.stride()
        if vs[3] != 1:
            v = v.contiguous()
            vs = v.stride()
        R, M = shape[0], shape[2]
        rows, n_new, rp, np_ = self._rows(rows, n_new, R)
        rc = self._lib.akv_int4_append(
            _C.IO_ARGS.pack(view, rp, np_, 0, k.data_ptr(), ks[0], ks[1], ks[2], v.data_ptr(), vs[0], vs[1], vs[2],
                            self._status_ptr, R, M, dt, 0), _C.raw_stream(self._dev_index))
        if rc:
            _C.check(rc, "akv_int4_append")

    def read(self, layer: int, n_tokens: int, rows=None, start=None, n_new=None, dtype=torch.float16):
        """The K and V values the cache stands for, (R, kv_heads, n_tokens, head_dim) in ``dtype``: tokens
        ``start[i]`` onwards of each row, or with ``start`` None its last ``n_new[i]`` (None: n_tokens); 0 past
        the row's end."""
        if _C.current_device() != self._dev_index:
            with torch.cuda.device(self._dev_index):
                return self.read(layer, n_tokens, rows, start, n_new, dtype)
        view = self._layer(layer)
        dt = _HALF.get(dtype)
        if dt is None:
            raise TypeError(f"dtype must be fp16 or bf16 (got {dtype})")
        if n_tokens < 0:
            raise ValueError("n_tokens is negative")
        given = rows if rows is not None else (start if start is not None else n_new)
        R = self.max_seqs if given is None else len(given)
        rows, n_new, rp, np_ = self._rows(rows, n_new, R)
        start = self._ints(start, "start", R)
        shape = (R, self.H, n_tokens, self.D)
        sm = self.D
        sh = sm * n_tokens
        sr = sh * self.H
        # empty_strided: 1.5 us of host time, torch.empty with its keywords 2.3
        k = torch.empty_strided(shape, (sr, sh, sm, 1), dtype=dtype, device=self._dev)
        v = torch.empty_strided(shape, (sr, sh, sm, 1), dtype=dtype, device=self._dev)
        rc = self._lib.akv_int4_read(
            _C.IO_ARGS.pack(view, rp, np_, 0 if start is None else start.data_ptr(), k.data_ptr(), sr, sh, sm,
                            v.data_ptr(), sr, sh, sm, self._status_ptr, R, n_tokens, dt, 0),
            _C.raw_stream(self._dev_index))
        if rc:
            _C.check(rc, "akv_int4_read")
        return k, v

    def attend(self, layer: int, query: torch.Tensor, rows=None, n_new=None, sm_scale: Optional[float] = None,
               out: Optional[torch.Tensor] = None, return_lse: bool = False):
        """softmax(q K^T * sm_scale) V of each row's newest tokens over its sequence, causal by position.

        query (R, Hq, M, head_dim), or (R, Hq, head_dim) for one token, fp16 or bf16, any strides: query m of
        row i is its token lens - n_new[i] + m (``n_new`` None: M) and sees the tokens up to itself.  Queries
        past n_new[i] give zero rows, queries with NaN or infinities rows of NaN.  Returns the output in the
        query's shape, type and (where it is dense) layout, and with ``return_lse`` the natural-log LSE (R, Hq, M)
        fp32."""
        if _C.current_device() != self._dev_index:
            with torch.cuda.device(self._dev_index):
                return self.attend(layer, query, rows, n_new, sm_scale, out, return_lse)
        view = self._layer(layer)
        dt = _half_dtype(query)
        one = query.dim() == 3
        q = query.unsqueeze(2) if one else query
        shape = q.shape
        if len(shape) != 4 or shape[3] != self.D or shape[1] % self.H or not shape[1]:
            raise ValueError(f"query must be (rows, a multiple of {self.H} heads, tokens, {self.D})")
        if q.device != self._dev:
            raise RuntimeError(f"akv: the query must be on {self._dev} (no CPU fallback)")
        R, Hq, M, D = shape
        qs = q.stride()
        if qs[3] != 1:
            q = q.contiguous()
            qs = q.stride()
        rows, n_new, rp, np_ = self._rows(rows, n_new, R)
        if out is None:
            o = torch.empty_like(q)
            os_ = o.stride()
            if os_[3] != 1:  # a query whose layout does not carry over
                o = torch.empty(shape, dtype=q.dtype, device=self._dev)
                os_ = o.stride()
        else:
            o = out.unsqueeze(2) if out.dim() == 3 else out
            os_ = o.stride()
            if o.shape != shape or o.dtype is not q.dtype or os_[-1] != 1 or o.device != self._dev:
                raise ValueError("out must have the query's shape, type and device, its last dim contiguous")
        lse = torch.empty_strided((R, Hq, M), (Hq * M, M, 1), dtype=torch.float32,
                                  device=self._dev) if return_lse else None
        stream = _C.raw_stream(self._dev_index)
        key = (R, M, Hq)
        need = self._ws_need.get(key)
        if need is None:
            need = self._ws_need[key] = int(self._lib.akv_int4_attention_workspace_bytes(R, M, Hq, self.H, D,
                                                                                         self.max_blocks))
            if need == 0:
                raise ValueError(f"unsupported attention shape: {M} tokens of {Hq} heads")
        ws = self._workspace(need, stream)
        rc = self._lib.akv_int4_attention(
            _C.ATTENTION_ARGS.pack(view, rp, np_, q.data_ptr(), qs[0], qs[1], qs[2], o.data_ptr(), os_[0], os_[1],
                                   os_[2], 0 if lse is None else lse.data_ptr(), ws.data_ptr(), need,
                                   self._status_ptr, R, M, Hq, dt,
                                   self._scale if sm_scale is None else float(sm_scale), 0), stream)
        if rc:
            _C.check(rc, "akv_int4_attention")
        res = o.squeeze(2) if one else o
        return (res, lse) if return_lse else res
