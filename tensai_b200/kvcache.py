"""Paged 8-bit key/value cache (C ABI tq_kv_*): block tables and slots from
request lengths, the store of new keys and values, and the attention over
them, for a process that serves several requests at once.

    cache = KVCache(n_layer=28, n_kv=4, hd=128, page=64, n_pages=4096)
    cache.plan(cached, added, table, free_pages, free_count, starts, lens, slots)
    for layer in range(28):
        ...                                     # this layer's q, k, v of the new tokens
        cache.store(layer, k, v, slots)
        out = cache.attention(layer, q, starts, lens, table)

Arguments are CUDA tensors on the cache's device; lengths, tables and counts
are int32, slots int64. Every call is asynchronous, allocates no device memory
in the library and can be captured into a CUDA graph. `stream`: a
torch.cuda.Stream, by default torch's current one on the cache's device.
Wrong shapes and types raise at the call; what only the device can see (a full
pool, a bad page id) is skipped there and raised by check().
"""
from __future__ import annotations

import ctypes
import struct

from . import _lib
from ._lib import TensaiError

_MESSAGES = ((_lib.TQ_KV_STATUS_POOL, "not enough free pages, or a full free list"),
             (_lib.TQ_KV_STATUS_TABLE, "a request longer than its table row"),
             (_lib.TQ_KV_STATUS_SLOTS, "more new tokens than slots, or slots of a page out of order"),
             (_lib.TQ_KV_STATUS_LENGTH, "a negative length or count, or starts that do not ascend"),
             (_lib.TQ_KV_STATUS_PAGE, "a page id or slot outside the cache"),
             (_lib.TQ_KV_STATUS_TIMEOUT, "a kernel gave up a bounded wait"))


# The argument structs of include/tensai_cuda.h, packed: cheaper than a ctypes
# Structure for each call of a decode step.
_PLAN = struct.Struct("5i4x9Q").pack
_RELEASE = struct.Struct("4i6Q").pack
_ATTENTION = struct.Struct("2Q4i2q3Q2if4x2Q").pack


def _refuse(msg: str):
    raise ValueError("tensai: " + msg)


class KVCache:
    """n_pages pages of `page` tokens (16, 32, 64 or 128) for n_layer layers of
    n_kv KV heads of size hd (a multiple of 8 up to 256), on the thread's
    device (tq_set_device). Codes are int8, with one float32 scale for the keys
    and one for the values of each page and head."""

    def __init__(self, n_layer: int, n_kv: int, hd: int, page: int, n_pages: int):
        import torch
        self._h = 0
        self._L = _lib.load()
        c = _lib.KvConfig(n_layer, n_kv, hd, page, n_pages)
        h = ctypes.c_uint64()
        _lib.check(self._L.tq_kv_create(ctypes.byref(c), ctypes.byref(h)))
        self._h = h.value
        self.n_layer, self.n_kv, self.hd, self.page, self.n_pages = n_layer, n_kv, hd, page, n_pages
        dev = ctypes.c_int()
        _lib.check(self._L.tq_kv_info(self._h, None, ctypes.byref(dev)))
        self.device = torch.device("cuda", dev.value)
        self._index = dev.value
        self._i32, self._i64 = torch.int32, torch.int64
        self._raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        size = ctypes.c_size_t()
        _lib.check(self._L.tq_kv_attention_workspace(self._h, ctypes.byref(size)))
        self.workspace_bytes = size.value
        self._spaces = {}
        self._torch = torch
        self._kinds = {torch.float32: _lib.TQ_LINEAR_F32, torch.float16: _lib.TQ_LINEAR_F16,
                       torch.bfloat16: _lib.TQ_LINEAR_BF16}

    # ---- arguments ----
    def _stream(self, stream) -> int:
        if stream is not None:
            return stream.cuda_stream
        if self._raw_stream is not None:
            return self._raw_stream(self._index)
        return self._torch.cuda.current_stream(self.device).cuda_stream

    def _capturing(self, stream) -> bool:
        """Whether the call's stream is being captured, which need not be the current one."""
        cuda = self._torch.cuda
        if stream is None and cuda.current_device() == self._index:
            return cuda.is_current_stream_capturing()
        with cuda.stream(cuda.current_stream(self.device) if stream is None else stream):
            return cuda.is_current_stream_capturing()

    def _array(self, name, t, dtype, numel=None):
        if t.dtype is not dtype or not t.is_cuda or t.get_device() != self._index or not t.is_contiguous():
            _refuse(f"{name}: a contiguous {dtype} tensor on {self.device} is required")
        if numel is not None and t.numel() != numel:
            _refuse(f"{name}: {t.numel()} elements, expected {numel}")
        return t.data_ptr()

    def _table(self, t, n):
        if t.dtype is self._i32 and t.is_cuda and t.get_device() == self._index and t.dim() == 2:
            rows, cols = t.shape
            if rows == n:
                if t.is_contiguous():
                    return t.data_ptr(), cols, cols
                down, along = t.stride()
                if (cols <= 1 or along == 1) and (n <= 1 or down >= cols):
                    return t.data_ptr(), (down if n > 1 else cols), cols
        _refuse(f"table: an int32 tensor [{n}][pages of a request] on {self.device} is required")

    def _rows(self, name, t, heads):
        """(address, elements between tokens) of [tokens][heads][hd] with dense rows."""
        if t.dtype not in self._kinds or not t.is_cuda or t.get_device() != self._index:
            _refuse(f"{name}: a float32, float16 or bfloat16 tensor on {self.device} is required")
        shape, hd = t.shape, self.hd
        if len(shape) != 3 or (heads is not None and shape[1] != heads) or shape[2] != hd:
            _refuse(f"{name}: shape {tuple(shape)}, expected [tokens][{heads or 'heads'}][{hd}]")
        row = shape[1] * hd
        if t.is_contiguous():
            return t.data_ptr(), row
        s0, s1, s2 = t.stride()
        if s2 != 1 or (shape[1] > 1 and s1 != hd) or (shape[0] > 1 and s0 < row):
            _refuse(f"{name}: heads and dimensions must be dense within a token")
        return t.data_ptr(), (s0 if shape[0] > 1 else row)

    def _pages(self, pages):
        return self._array("pages", pages, self._torch.int32), pages.numel()

    # ---- bookkeeping ----
    def plan(self, cached, added, table, free_pages, free_count, starts, lens, slots, free_left=None,
             stream=None) -> None:
        """The pages that the step needs from the free list into `table`, and
        starts [n + 1], lens [n] (may be `cached`) and slots of the new tokens
        (tq_kv_plan_dev). free_left: where the remaining count goes (free_count
        itself when None)."""
        n, i32, array = cached.numel(), self._i32, self._array
        tp, ts, tc = self._table(table, n)
        a = _PLAN(n, ts, tc, free_pages.numel(), slots.numel(), array("cached", cached, i32), array("added", added, i32, n),
                  tp, array("free_pages", free_pages, i32), array("free_count", free_count, i32, 1),
                  array("starts", starts, i32, n + 1), array("lens", lens, i32, n), array("slots", slots, self._i64),
                  array("free_left", free_count if free_left is None else free_left, i32, 1))
        _lib.check(self._L.tq_kv_plan_dev(self._h, a, self._stream(stream)))

    def release(self, done, lens, table, free_pages, free_count, free_left=None, stream=None) -> None:
        """Puts the pages of the requests with done != 0 (int32) back on the
        free list and sets their lens to 0 (tq_kv_release_dev)."""
        n, i32, array = lens.numel(), self._i32, self._array
        tp, ts, tc = self._table(table, n)
        a = _RELEASE(n, ts, tc, free_pages.numel(), array("done", done, i32, n), array("lens", lens, i32), tp,
                     array("free_pages", free_pages, i32), array("free_count", free_count, i32, 1),
                     array("free_left", free_count if free_left is None else free_left, i32, 1))
        _lib.check(self._L.tq_kv_release_dev(self._h, a, self._stream(stream)))

    # ---- store and attention ----
    def store(self, layer: int, k, v, slots, stream=None) -> None:
        """New keys and values [tokens][n_kv][hd] (float32, float16 or bfloat16;
        tokens may be strided) into their slots (tq_kv_store_dev)."""
        kp, ks = self._rows("k", k, self.n_kv)
        vp, vs = self._rows("v", v, self.n_kv)
        n = k.shape[0]
        if v.shape[0] != n or v.dtype != k.dtype:
            _refuse("k and v must have the same tokens and type")
        _lib.check(self._L.tq_kv_store_dev(self._h, layer, kp, vp, self._kinds[k.dtype], ks, vs,
                                           self._array("slots", slots, self._torch.int64, n), n, self._stream(stream)))

    def attention(self, layer: int, q, starts, lens, table, out=None, scale=None, workspace=None, stream=None):
        """softmax(scale q . k) v of the new tokens' queries [tokens][heads][hd]
        over their sequences' cached positions, causal (tq_kv_attention_dev).
        scale: hd ** -0.5 by default. out: a tensor like q; rows behind
        starts[n] are not written. A table wider than the step's longest
        sequence needs can cost time (the header says when). workspace: self.workspace() by default, one
        for each stream, or one for each call while a graph is captured, so
        that graphs never share one."""
        torch = self._torch
        qp, qs = self._rows("q", q, None)
        if out is None:
            out = self._empty(q.shape, q.dtype, stream)
        elif out.dtype != q.dtype or out.shape != q.shape:
            _refuse("out must have the shape and type of q")
        op, os = self._rows("out", out, None)
        n = lens.numel()
        tp, ts, tc = self._table(table, n)
        st = self._stream(stream)
        if workspace is None:
            if self._capturing(stream):
                workspace = self.workspace(stream)
            else:
                workspace = self._spaces.get(st)
                if workspace is None:
                    workspace = self._spaces[st] = self.workspace(stream)
        a = _ATTENTION(qp, op, self._kinds[q.dtype], q.shape[1], q.shape[0], n, qs, os,
                       self._array("starts", starts, self._i32, n + 1), self._array("lens", lens, self._i32), tp, ts, tc,
                       self.hd ** -0.5 if scale is None else scale,
                       self._array("workspace", workspace, torch.uint8), workspace.numel())
        _lib.check(self._L.tq_kv_attention_dev(self._h, layer, a, st))
        return out

    def workspace(self, stream=None):
        """A workspace for attention(): never shared by calls that may overlap."""
        torch = self._torch
        with torch.cuda.stream(stream):  # None: the current one
            w = torch.empty(self.workspace_bytes, dtype=torch.uint8, device=self.device)
            w[:_lib.TQ_KV_WORKSPACE_HEAD].zero_()
        return w

    def _empty(self, shape, dtype, stream):
        """An output of a call on `stream`: memory of that stream, so that it can be dropped any time."""
        if stream is None:
            return self._torch.empty(shape, dtype=dtype, device=self.device)
        with self._torch.cuda.stream(stream):
            return self._torch.empty(shape, dtype=dtype, device=self.device)

    # ---- pages in and out ----
    def load(self, layer: int, pages, k, v, kscale, vscale, stream=None) -> None:
        """Codes [pages][page][n_kv][hd] int8 and scales [pages][n_kv] float32
        into the listed pages (int32, each once)."""
        torch = self._torch
        pp, n = self._pages(pages)
        m = n * self.n_kv
        _lib.check(self._L.tq_kv_load_dev(
            self._h, layer, pp, n, self._array("k", k, torch.int8, m * self.page * self.hd),
            self._array("v", v, torch.int8, m * self.page * self.hd), self._array("kscale", kscale, torch.float32, m),
            self._array("vscale", vscale, torch.float32, m), self._stream(stream)))

    def save(self, layer: int, pages, stream=None):
        """(k, v, kscale, vscale) of the listed pages, as load takes them."""
        torch = self._torch
        pp, n = self._pages(pages)
        shape = (n, self.page, self.n_kv, self.hd)
        k, v = (self._empty(shape, torch.int8, stream) for _ in range(2))
        ks, vs = (self._empty((n, self.n_kv), torch.float32, stream) for _ in range(2))
        _lib.check(self._L.tq_kv_save_dev(self._h, layer, pp, n, k.data_ptr(), v.data_ptr(), ks.data_ptr(),
                                          vs.data_ptr(), self._stream(stream)))
        return k, v, ks, vs

    def read(self, layer: int, pages, stream=None):
        """The values (code * scale) of the listed pages: k and v
        [pages][page][n_kv][hd] float32."""
        torch = self._torch
        pp, n = self._pages(pages)
        shape = (n, self.page, self.n_kv, self.hd)
        k, v = (self._empty(shape, torch.float32, stream) for _ in range(2))
        _lib.check(self._L.tq_kv_read_dev(self._h, layer, pp, n, k.data_ptr(), v.data_ptr(), self._stream(stream)))
        return k, v

    # ---- state ----
    def status(self) -> int:
        """TQ_KV_STATUS_* bits since the last look (waits for the device)."""
        bits = ctypes.c_uint()
        _lib.check(self._L.tq_kv_status(self._h, ctypes.byref(bits)))
        return bits.value

    def check(self) -> None:
        """Raises TensaiError when a call since the last look could not do its work."""
        bits = self.status()
        if bits:
            what = "; ".join(m for b, m in _MESSAGES if bits & b)
            raise TensaiError(_lib.TQ_ERR_TIMEOUT if bits & _lib.TQ_KV_STATUS_TIMEOUT else _lib.TQ_ERR_SHAPE,
                              f"tensai: cache: {what}")

    def free(self) -> None:
        """Releases the pages (idempotent)."""
        if self._h:
            self._L.tq_kv_free(self._h)
            self._h = 0
            self._spaces.clear()

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.free()
