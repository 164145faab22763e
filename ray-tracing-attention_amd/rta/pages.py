"""Paged history over librta.so's rta_pages_* and rta_paged_* entry points: the keys and
values of many sequences in one pool of pages that are handed out, shared between forked
sequences, copied on write and closed up on the device, and the attention that reads them.

PyTorch only provides device memory and the current stream.  No call synchronises or reads
a length back, so a loop of them can be captured in a HIP graph; what only the device can
know (a bad sequence or page, a pool that has run out) raises DEVERR_PAGES in the device
error word (ops.device_error).
"""
import ctypes

import torch

from . import _lib
from ._lib import BF16, F16, Q8_ROW, check
from .ops import _rows, _rs

WHOLE = 2**31 - 1   # a `last` past every length


def page_bytes(fmt, kv_heads, head_dim, page):
    """Bytes of one page of one layer (a multiple of 128)."""
    n = int(_lib.load().rta_page_bytes(fmt, kv_heads, head_dim, page))
    if n < 0:
        raise ValueError(f"no pages of format {fmt} with {kv_heads} heads of {head_dim} and {page} positions")
    return n


class PagedCache:
    """A paged history and its operators.

    Either sizes (n_pages, max_seqs, max_pages per sequence, layers, device), and the pool and
    an empty book are allocated, or the four tensors of a caller that keeps them: pool uint8
    [layers, n_pages, page_bytes], table int32 [max_seqs, max_pages], lengths int32 [max_seqs],
    refs int32 [n_pages], all of them on one device and contiguous.

    List arguments are int32 device tensors: seqs (None: the sequences 0, 1, ..) names a
    sequence per entry; cu_rows (n + 1 offsets, None: one row per entry) gives each entry its
    rows, which are its sequence's newest positions."""

    def __init__(self, fmt, kv_heads, head_dim, page, n_pages=None, max_seqs=None, max_pages=None, layers=1,
                 device="cuda:0", pool=None, table=None, lengths=None, refs=None):
        self.lib = _lib.load()
        pb = page_bytes(fmt, kv_heads, head_dim, page)
        given = (pool, table, lengths, refs)
        fresh = all(t is None for t in given)
        if fresh:
            if None in (n_pages, max_seqs, max_pages):
                raise ValueError("n_pages, max_seqs and max_pages, or pool, table, lengths and refs")
            ints = lambda *shape: torch.empty(*shape, dtype=torch.int32, device=device)  # noqa: E731
            pool = torch.empty(layers, n_pages, pb, dtype=torch.uint8, device=device)
            table, lengths, refs = ints(max_seqs, max_pages), ints(max_seqs), ints(n_pages)
        elif any(t is None for t in given):
            raise ValueError("pool, table, lengths and refs come together")
        for t, name, dtype, dim in ((pool, "pool", torch.uint8, 3), (table, "table", torch.int32, 2),
                                    (lengths, "lengths", torch.int32, 1), (refs, "refs", torch.int32, 1)):
            if not isinstance(t, torch.Tensor) or not t.is_cuda:
                raise TypeError(f"{name} must be a CUDA (HIP) tensor")
            if t.dtype != dtype or t.dim() != dim or not t.is_contiguous() or t.device != pool.device:
                raise ValueError(f"{name} must be a contiguous {dim}-D {dtype} tensor on the pool's device")
        if pool.shape[2] != pb or refs.shape[0] != pool.shape[1] or lengths.shape[0] != table.shape[0]:
            raise ValueError(f"pool [layers, n_pages, {pb}], table [max_seqs, max_pages], lengths [max_seqs], "
                             "refs [n_pages]")
        self.fmt, self.kv_heads, self.head_dim, self.page = fmt, kv_heads, head_dim, page
        self.pool, self.table, self.lengths, self.refs = pool, table, lengths, refs
        self.device = pool.device
        self._c = _lib.Pages(fmt, kv_heads, head_dim, page, pool.shape[0], pool.shape[1], table.shape[0],
                             table.shape[1], pool.data_ptr(), table.data_ptr(), lengths.data_ptr(), refs.data_ptr())
        self._at = ctypes.byref(self._c)
        if fresh:
            self.reset()

    # ------------------------------------------------------------------ helpers ----
    def _call(self, name, *args):
        """One entry point on the current stream of the pool's device."""
        fn, index = getattr(self.lib, name), self.device.index
        # (the raw handle: building a Stream object takes 3 us, as long as a launch)
        stream = torch._C._cuda_getCurrentRawStream(index)
        if torch.cuda.current_device() == index:
            status = fn(self._at, *args, stream)
        else:
            with torch.cuda.device(index):
                status = fn(self._at, *args, stream)
        if status:
            check(status, name)

    def _scratch(self, need, given):
        """(pointer, bytes) of a call's workspace; the tensor comes third, to outlive the launch."""
        if given is None:
            if not need:
                return None, 0, None
            given = torch.empty(need, dtype=torch.uint8, device=self.device)
        elif not isinstance(given, torch.Tensor) or given.device != self.device:
            raise TypeError(f"workspace must be a tensor on {self.device}")
        elif not given.is_contiguous():
            raise ValueError("workspace must be contiguous")
        return given.data_ptr(), given.numel() * given.element_size(), given

    def _ints(self, t, name, n=None):
        if t is None:
            return None
        if not isinstance(t, torch.Tensor) or t.device != self.device or t.dtype != torch.int32:
            raise TypeError(f"{name} must be an int32 tensor on {self.device}")
        if t.dim() != 1 or not t.is_contiguous() or (n is not None and t.shape[0] != n):
            raise ValueError(f"{name} must be contiguous and 1-D" + (f" of {n} values" if n is not None else ""))
        return t.data_ptr()

    def _check_floats(self, t, name, shape):
        if not isinstance(t, torch.Tensor) or t.device != self.device or t.dtype != torch.float32:
            raise TypeError(f"{name} must be a float32 tensor on {self.device}")
        if tuple(t.shape) != shape or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous of shape {shape}")

    def _list(self, rows, seqs, cu_rows):
        """(seqs pointer, cu_rows pointer, entries) of a row list over `rows` rows."""
        if cu_rows is not None:
            cu = self._ints(cu_rows, "cu_rows")
            n = cu_rows.shape[0] - 1
        else:
            cu, n = None, rows
        if seqs is None and n > self.table.shape[0]:
            raise ValueError(f"{n} entries for {self.table.shape[0]} sequences")
        return self._ints(seqs, "seqs", n), cu, n

    def _entries(self, seqs, n):
        if seqs is not None:
            self._ints(seqs, "seqs")
            return seqs.shape[0]
        return self.table.shape[0] if n is None else n

    # ------------------------------------------------------------------ the book ----
    def reset(self):
        """Every sequence empty, every page free."""
        self._call("rta_pages_init")

    def workspace_bytes(self, n=1):
        return int(self.lib.rta_pages_workspace_bytes(self._at, n))

    def extend(self, seqs=None, add=None, n=None, workspace=None):
        """lengths[seqs] += add (None: one position each) with pages for the new positions; a last
        page shared with another sequence is copied first.  seqs None: the first n sequences."""
        n = self._entries(seqs, n)
        sp, ap = self._ints(seqs, "seqs", n), self._ints(add, "add", n)
        ws, size, _keep = self._scratch(self.workspace_bytes(n), workspace)
        self._call("rta_pages_extend", sp, ap, n, ws, size)

    def fork(self, src, dst):
        """The empty sequences dst become copies of src that share their pages."""
        if src is None or dst is None:
            raise TypeError("src and dst must be tensors")
        sp = self._ints(src, "src")
        n = src.shape[0]
        self._call("rta_pages_fork", sp, self._ints(dst, "dst", n), n)

    def free(self, seqs=None, first=None, last=None, n=None):
        """Gives up the pages of seqs whose positions lie in [first, last) (None: all of them); with
        last at or past its length a sequence ends at first."""
        n = self._entries(seqs, n)
        self._call("rta_pages_free", self._ints(seqs, "seqs", n), self._ints(first, "first", n),
                   self._ints(last, "last", n), n)

    def compact(self, used=None, workspace=None):
        """Moves the used pages to the front of the pool; returns their number, int32 [1] on the device."""
        if used is None:
            used = torch.empty(1, dtype=torch.int32, device=self.device)
        up = self._ints(used, "used", 1)
        ws, size, _keep = self._scratch(self.workspace_bytes(), workspace)
        self._call("rta_pages_compact", up, ws, size)
        return used

    # ------------------------------------------------------------------ rows ----
    def _strided(self, t, name, rows):
        _rows(t, name)
        if t.device != self.device or t.dtype != torch.float32:
            raise TypeError(f"{name} must be a float32 tensor on {self.device}")
        if t.shape != (rows, self.kv_heads * self.head_dim):
            raise ValueError(f"{name} must be [{rows}, {self.kv_heads * self.head_dim}]")
        return t.data_ptr(), _rs(t)

    def append(self, k, v, layer=0, seqs=None, cu_rows=None):
        """Keys and values [rows, kv_heads * head_dim] fp32 (rows may be strided) of the sequences'
        newest positions into the pages of `layer`.  Call it after extend."""
        rows = _rows(k, "k").shape[0]
        sp, cu, n = self._list(rows, seqs, cu_rows)
        self._call("rta_paged_append", layer, *self._strided(k, "k", rows), *self._strided(v, "v", rows), rows, sp, cu,
                   n)

    def read(self, rows, layer=0, seqs=None, cu_rows=None, k=None, v=None):
        """The keys and values of those rows as fp32: (k, v), each [rows, kv_heads * head_dim].
        Rows that no entry lists are left as they were in k and v, and mean nothing in tensors
        made here."""
        sp, cu, n = self._list(rows, seqs, cu_rows)
        shape = (rows, self.kv_heads * self.head_dim)
        k = torch.empty(shape, dtype=torch.float32, device=self.device) if k is None else k
        v = torch.empty(shape, dtype=torch.float32, device=self.device) if v is None else v
        self._call("rta_paged_read", layer, rows, sp, cu, n, *self._strided(k, "k", rows), *self._strided(v, "v", rows))
        return k, v

    # ------------------------------------------------------------------ attention ----
    def attention_workspace_bytes(self, hq, rows, n=None, max_rows=1, max_len=0, window=0, sinks=0):
        return int(self.lib.rta_paged_attention_workspace_bytes(self._at, hq, rows, rows if n is None else n, max_rows,
                                                                max_len or 0, window, sinks))

    def attention(self, q, layer=0, seqs=None, cu_rows=None, max_rows=None, max_len=0, window=0, sinks=0, gate=None,
                  out=None, m=None, z=None, workspace=None):
        """Causal attention of the rows q [rows, hq, head_dim] fp32 (rows may be strided) over
        their sequences' pages; with window > 0 a row sees its last `window` positions and the
        first `sinks`.  Returns (out [rows, hq, head_dim], m [rows, hq], z [rows, hq]).

        max_rows: the most rows of an entry (None: one without cu_rows, else all of them), which
        decides the kernel for all entries: prompts and single rows are faster in calls of their own;
        max_len: the longest sequence (0: max_pages * page).  Rows that no entry lists are left as
        they were in out, m and z, and mean nothing in tensors made here."""
        if not isinstance(q, torch.Tensor) or q.device != self.device or q.dtype != torch.float32:
            raise TypeError(f"q must be a float32 tensor on {self.device}")
        if q.dim() != 3 or q.shape[2] != self.head_dim or q.stride(2) != 1 or \
                (q.shape[1] > 1 and q.stride(1) != self.head_dim):
            raise ValueError(f"q must be [rows, heads, {self.head_dim}] with contiguous rows")
        rows, hq, hd = q.shape
        sp, cu, n = self._list(rows, seqs, cu_rows)
        if max_rows is None:
            max_rows = 1 if cu_rows is None else rows
        for t, name, shape in ((gate, "gate", (rows, hq, hd)), (out, "out", (rows, hq, hd)), (m, "m", (rows, hq)),
                               (z, "z", (rows, hq))):
            if t is not None:
                self._check_floats(t, name, shape)
        if out is None:
            out = torch.empty(rows, hq, hd, dtype=torch.float32, device=self.device)
        if m is None:
            m = torch.empty(rows, hq, dtype=torch.float32, device=self.device)
        if z is None:
            z = torch.empty(rows, hq, dtype=torch.float32, device=self.device)
        max_len = max_len or 0
        need = self.lib.rta_paged_attention_workspace_bytes(self._at, hq, rows, n, max_rows, max_len, window, sinks)
        ws, size, _keep = self._scratch(need, workspace)
        stride = q.stride(0) if rows > 1 else max(q.stride(0), hq * hd)
        self._call("rta_paged_attention", layer, q.data_ptr(), stride, rows, hq, sp, cu, n, max_rows, max_len, window,
                   sinks, None if gate is None else gate.data_ptr(), out.data_ptr(), m.data_ptr(), z.data_ptr(), ws,
                   size)
        return out, m, z


__all__ = ["BF16", "F16", "Q8_ROW", "PagedCache", "WHOLE", "page_bytes"]
