"""Key/value rows held in 4 bits: ctypes binding of include/homcomp_cache.h.

    from tirocinio_triennale_amd import cache          (after __graft_entry__.load_package())
    c = cache.Cache(pages, kv_heads, head_dim, page_tokens)     # pages: cache.new_pages(...)
    c.store(k, v, table, lengths, starts)                # the new rows, quantised into their slots
    c.attend(q, out, table, lengths, starts)             # attention of the same rows over all slots

Like the rest of the package: torch supplies device memory and streams, the HIP kernels do the work, and without the library or
a GPU every call raises.  Arguments that the library cannot see (shapes, types, devices) are checked here; a
refusal is a ValueError or a TypeError, and nothing has been enqueued then.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import struct

from . import _check, lib as _package_lib

EXPORTS = ("homcomp_cache_page_bytes", "homcomp_cache_store", "homcomp_cache_load", "homcomp_cache_attend_scratch",
           "homcomp_cache_attend", "homcomp_cache_evict")

BF16, F16, F32 = 0, 1, 2


# The argument structures of the header, packed by hand: a call's cost in Python is a good part of a small call's.
_CACHE = struct.Struct("@P N iiii P N P")         # homcomp_cache
_ATTENTION = struct.Struct("@P N N P N N ii P N N N f i N P P P N P N")   # homcomp_attention
_EVICTION = struct.Struct("@P N N N N N P N P P P")                      # homcomp_eviction


_lib = None


def lib() -> C.CDLL:
    """The library with this header's signatures; raises if it has not been built (no fallback)."""
    global _lib
    if _lib is None:
        L = _package_lib()
        vp, sz = C.c_void_p, C.c_size_t   # (packed structures are bytes, which a void pointer takes)
        L.homcomp_cache_page_bytes.argtypes = [C.c_int, C.c_int, C.c_int]
        L.homcomp_cache_page_bytes.restype = sz
        for name in ("homcomp_cache_store", "homcomp_cache_load"):
            getattr(L, name).argtypes = [vp, vp, vp, C.c_int, sz, sz, vp, sz, vp]
        L.homcomp_cache_attend_scratch.argtypes = [vp, vp]
        L.homcomp_cache_attend_scratch.restype = sz
        L.homcomp_cache_attend.argtypes = [vp, vp, vp]
        L.homcomp_cache_evict.argtypes = [vp, vp, vp]
        _lib = L
    return _lib


def page_bytes(kv_heads: int, head_dim: int, page_tokens: int) -> int:
    """Bytes of a page; raises where the shape is not supported."""
    n = int(lib().homcomp_cache_page_bytes(kv_heads, head_dim, page_tokens))
    if n == 0:
        raise ValueError(f"no cache of {kv_heads} heads of {head_dim} values in pages of {page_tokens}: heads 1..1024, "
                         "values 64, 128 or 256, page a power of two from 32 to 65536")
    return n


def new_pages(n_pages: int, kv_heads: int, head_dim: int, page_tokens: int, device="cuda"):
    """Room for n_pages pages, [n_pages, page bytes] uint8 (what it holds does not matter before it is stored to)."""
    import torch
    return torch.empty(n_pages, page_bytes(kv_heads, head_dim, page_tokens), dtype=torch.uint8, device=device)


def _stream_of(device, stream) -> int:
    import torch
    if device.type != "cuda":
        raise ValueError("the cache's pages lie in a GPU's memory")
    if stream is None:   # the handle alone, without the object around it: a tenth of the time
        return torch._C._cuda_getCurrentRawStream(device.index)
    if stream.device != device:
        raise ValueError("stream: of the pages' device")
    return int(stream.cuda_stream)


def _allocating(stream):
    """New memory belongs to the stream that the call runs on: what another stream freed may still be in use there."""
    if stream is None:
        return _NOTHING
    import torch
    return torch.cuda.stream(stream)


_NOTHING = contextlib.nullcontext()


def _share_memory(rows, row, heads, head, d):
    """Whether of the runs of d elements at i * row + j * head two have one in common."""
    if rows > 1 and row < d or heads > 1 and head < d:
        return True
    if rows < 2 or heads < 2 or row >= (heads - 1) * head + d or head >= (rows - 1) * row + d:
        return False                      # (one inside the other: nearly every layout)
    for j in range(1, heads):             # j heads on and the rows next to there
        i = j * head // row
        if i < rows and j * head - i * row < d or i + 1 < rows and (i + 1) * row - j * head < d:
            return True
    return False


def _meet(offset, rows, row, heads, head, d):
    """Whether the runs of two such arrays, the second `offset` elements behind the first, have an element in common."""
    offset = abs(offset)
    if offset >= (rows - 1) * row + (heads - 1) * head + d:
        return False
    row, head = row if rows > 1 else 0, head if heads > 1 else 0
    for j in range(1 - heads, heads):     # offset + j * head against the rows next to there, of either sign
        at = offset + j * head
        i = at // row if row else 0
        if min(abs(at - max(1 - rows, min(rows - 1, x)) * row) for x in (i, i + 1)) < d:
            return True
    return False


class Cache:
    """Pages of a cache and their shape.  The tables and lengths that say whose slots they are belong to the calls:

    table    int32 [sequences, pages of a sequence]   page numbers
    lengths  int32 [sequences]                        slots held, the new rows among them
    starts   int32 [sequences + 1]                    packed rows of sequence s: starts[s] .. starts[s + 1] - 1, its last slots

    all on the pages' device.  What the numbers in them may be is said in include/homcomp_cache.h.
    """

    def __init__(self, pages, kv_heads: int, head_dim: int, page_tokens: int = 64):
        import torch
        self.page_bytes = page_bytes(kv_heads, head_dim, page_tokens)
        if pages.dtype != torch.uint8 or not pages.is_contiguous() or pages.numel() % self.page_bytes:
            raise ValueError(f"pages: contiguous uint8, a multiple of {self.page_bytes} bytes")
        self.pages, self.kv_heads, self.head_dim, self.page_tokens = pages, kv_heads, head_dim, page_tokens
        self.n_pages = pages.numel() // self.page_bytes
        self._device = pages.device
        self._types = {torch.bfloat16: BF16, torch.float16: F16, torch.float32: F32}
        self._int32, self._float32 = torch.int32, torch.float32
        self._current_device = torch.cuda.current_device if pages.is_cuda else lambda: self._device.index

    # -- argument checks --------------------------------------------------------------------
    def _call(self, name, function, *args):
        """The call, with the pages' device as the current one (the library launches there)."""
        if self._device.index == self._current_device():
            status = function(*args)
        else:
            import torch
            with torch.cuda.device(self._device):
                status = function(*args)
        if status:
            _check(status, name)

    def _ints(self, name, t, dims):
        if t.dtype is not self._int32 or t.dim() != dims or t.device != self._device or not (t.is_contiguous() or not t.numel()):
            raise ValueError(f"{name}: int32, {dims}-dimensional, contiguous, on the pages' device")
        return t.data_ptr()

    def _args(self, table, lengths):
        """The cache's structure for these sequences, how many they are and the pages that one can have."""
        at, n_at = self._ints("table", table, 2), self._ints("lengths", lengths, 1)
        n, width = table.shape
        if lengths.shape[0] != n:
            raise ValueError("table: a row for every sequence")
        return _CACHE.pack(self.pages.data_ptr(), self.n_pages, self.kv_heads, self.head_dim, self.page_tokens, n, at, width, n_at), n, width

    def _starts(self, starts, n):
        at = self._ints("starts", starts, 1)
        if starts.shape[0] != n + 1:
            raise ValueError("starts: one number more than sequences")
        return at

    def _numbers(self, name, t, heads):
        """Strides of rows and heads."""
        if t.dtype not in self._types:
            raise TypeError(f"{name}: bfloat16, float16 or float32")
        shape = t.shape
        if len(shape) != 3 or shape[1] != heads or shape[2] != self.head_dim or t.device != self._device:
            raise ValueError(f"{name}: [rows, {heads}, {self.head_dim}] on the pages' device")
        row, head, one = t.stride()
        if one != 1 and t.numel():
            raise ValueError(f"{name}: the values of a row and head adjacent")
        return row, head

    def _own_memory(self, name, t, row, head):
        """Written tensors: no row or head of which shares another's memory."""
        heads, d = t.shape[1], self.head_dim
        if (head < d or row < (heads - 1) * head + d) and t.numel() and _share_memory(t.shape[0], row, heads, head, d):   # (seldom looked at)
            raise ValueError(f"{name}: rows and heads of its own memory")

    def _whole(self, name, t, shape, dtype):
        if t.dtype is not dtype or t.shape != shape or not t.is_contiguous() or t.device != self._device:
            raise ValueError(f"{name}: contiguous {dtype} {list(shape)} on the pages' device")
        return t.data_ptr()

    def _rows(self, name, what, written, k, v, table, lengths, starts, stream):
        row, head = self._numbers("k", k, self.kv_heads)
        if self._numbers("v", v, self.kv_heads) != (row, head) or k.dtype is not v.dtype or k.shape != v.shape:
            raise ValueError("k and v: of one type, shape and layout")
        at_k, at_v, rows, type_ = k.data_ptr(), v.data_ptr(), k.shape[0], self._types[k.dtype]
        if written:
            self._own_memory("k and v", k, row, head)
            if rows and _meet((at_v - at_k) // (4 if type_ == F32 else 2), rows, row, self.kv_heads, head, self.head_dim):
                raise ValueError("k and v: each of its own memory")
        args, n, _ = self._args(table, lengths)
        self._call(name, what, args, at_k, at_v, type_, row, head, self._starts(starts, n), rows, _stream_of(self._device, stream))

    # -- the operators ----------------------------------------------------------------------
    def store(self, k, v, table, lengths, starts, stream=None) -> None:
        """Quantises the rows of k and v ([rows, kv_heads, head_dim]) into their slots."""
        self._rows("cache_store", lib().homcomp_cache_store, False, k, v, table, lengths, starts, stream)

    def load(self, k, v, table, lengths, starts, stream=None) -> None:
        """Fills k and v with the rows that the slots stand for (of every sequence the last starts[s + 1] - starts[s] ones)."""
        self._rows("cache_load", lib().homcomp_cache_load, True, k, v, table, lengths, starts, stream)

    def attend(self, q, out, table, lengths, starts, scale: float | None = None, causal: bool = True, window: int = 0,
               max_rows: int | None = None, max_length: int | None = None, lse=None, weights=None, prior=None, scratch=None,
               stream=None) -> None:
        """Attention of the rows of q ([rows, heads, head_dim], heads a multiple of kv_heads) over the slots their sequences hold.

        scale       of the scores, default head_dim ** -0.5
        window      a row sees at most that many slots back, itself among them (0: all); after an eviction: of the slots left
        max_rows    no sequence has more rows (default: the rows of q), max_length: holds more slots (default: what the table can hold);
                    tighter numbers than the defaults make the launch smaller
        lse         float32 [rows, heads]: the log of the sum of the exponentials
        weights     float32 [sequences, kv_heads, at least max_length]: prior (same shape, may be weights, default 0) + the attention
                    that the slots received in this call
        scratch     at least scratch_bytes(...) bytes of contiguous memory, not shared by calls that may overlap; by default memory of
                    torch's allocator, taken for this call
        """
        rows, heads = q.shape[0], q.shape[1] if q.dim() == 3 else 0
        if heads < 1 or heads % self.kv_heads:
            raise ValueError(f"q: [rows, a multiple of {self.kv_heads}, {self.head_dim}]")
        q_row, q_head = self._numbers("q", q, heads)
        out_row, out_head = self._numbers("out", out, heads)
        if out.dtype is not q.dtype or out.shape != q.shape:
            raise ValueError("out: of q's type and shape")
        self._own_memory("out", out, out_row, out_head)
        args, n, width = self._args(table, lengths)
        first = self._starts(starts, n)
        most = width * self.page_tokens
        max_length = most if max_length is None or max_length > most else max_length
        max_rows = rows if max_rows is None or max_rows > rows else max_rows
        if max_length < 0 or max_rows < 0 or window < 0:
            raise ValueError("max_rows, max_length and window are not negative")
        at_lse = self._whole("lse", lse, (rows, heads), self._float32) if lse is not None else None
        at_weights = at_prior = None
        stride = 0
        if weights is not None:
            stride = weights.shape[2] if weights.dim() == 3 else -1
            if stride < max_length:
                raise ValueError(f"weights: [sequences, kv_heads, at least max_length = {max_length}]")
            at_weights = self._whole("weights", weights, (n, self.kv_heads, stride), self._float32)
            if prior is not None:
                at_prior = self._whole("prior", prior, (n, self.kv_heads, stride), self._float32)
        elif prior is not None:
            raise ValueError("prior goes with weights")
        L = lib()

        def packed(memory, size):
            return _ATTENTION.pack(q.data_ptr(), q_row, q_head, out.data_ptr(), out_row, out_head, self._types[q.dtype], heads, first, rows,
                                   max_rows, max_length, self.head_dim ** -0.5 if scale is None else scale, 1 if causal else 0, window,
                                   at_lse or 0, at_prior or 0, at_weights or 0, stride, memory, size)

        t = packed(0, 0)
        need = L.homcomp_cache_attend_scratch(args, t)
        if need:
            if scratch is None:
                with _allocating(stream):
                    scratch = q.new_empty((need + 3) // 4, dtype=self._float32)
            elif scratch.device != self._device or not scratch.is_contiguous():
                raise ValueError("scratch: contiguous, on the pages' device")
            t = packed(scratch.data_ptr(), scratch.numel() * scratch.element_size())
        self._call("cache_attend", L.homcomp_cache_attend, args, t, _stream_of(self._device, stream))

    def scratch_bytes(self, rows: int, heads: int, sequences: int, table_pages: int, dtype, window: int = 0, max_rows: int | None = None,
                      max_length: int | None = None, weights: bool = False, lse: bool = False) -> int:
        """Bytes of scratch memory that attend needs for these shapes."""
        most = table_pages * self.page_tokens
        args = _CACHE.pack(0, self.n_pages, self.kv_heads, self.head_dim, self.page_tokens, sequences, 0, table_pages, 0)
        # (pointers are looked at for being there alone)
        t = _ATTENTION.pack(0, 0, 0, 0, 0, 0, self._types[dtype], heads, 0, rows, rows if max_rows is None else min(max_rows, rows),
                            most if max_length is None else min(max_length, most), 1.0, 1, window, 16 if lse else 0, 0, 16 if weights else 0,
                            most if weights else 0, 0, 0)
        return int(lib().homcomp_cache_attend_scratch(args, t))

    def evict(self, weights, table, lengths, keep: int, to_table, to_lengths, first: int = 0, recent: int = 0,
              max_length: int | None = None, to_weights=None, kept=None, stream=None):
        """Cuts every longer sequence to `keep` rows a head, those of the largest weights among them, on other pages of this cache;
        returns (to_weights, kept).

        weights               float32 [sequences, kv_heads, at least max_length], as attend gathers them
        first, recent         slots at the front and at the back that stay whatever their weight
        to_table, to_lengths  where the rows go (the table is the caller's, its pages nobody's), and how many there are then
        to_weights, kept      [sequences, kv_heads, keep] float32 and int32: weights and old slots of the rows that stay; by default new
                              memory of the call's stream
        """
        args, n, width = self._args(table, lengths)
        at_table = self._ints("to_table", to_table, 2)
        if to_table.shape[0] != n:
            raise ValueError("to_table: a row for every sequence")
        most = width * self.page_tokens
        max_length = most if max_length is None or max_length > most else max_length
        if keep < 1 or first < 0 or recent < 0 or first + recent > keep or max_length < 0:
            raise ValueError("keep is positive, first and recent are not negative and together at most keep")
        if keep > to_table.shape[1] * self.page_tokens:
            raise ValueError("to_table has no room for keep rows")
        stride = weights.shape[2] if weights.dim() == 3 else -1
        if stride < max_length:
            raise ValueError(f"weights: [sequences, kv_heads, at least max_length = {max_length}]")
        shape = (n, self.kv_heads, keep)
        with _allocating(stream):
            to_weights = weights.new_empty(shape) if to_weights is None else to_weights
            kept = weights.new_empty(shape, dtype=self._int32) if kept is None else kept
        t = _EVICTION.pack(self._whole("weights", weights, (n, self.kv_heads, stride), self._float32), stride, max_length, keep, first, recent, at_table,
                           to_table.shape[1], self._whole("to_lengths", to_lengths, (n,), self._int32),
                           self._whole("to_weights", to_weights, shape, self._float32), self._whole("kept", kept, shape, self._int32))
        self._call("cache_evict", lib().homcomp_cache_evict, args, t, _stream_of(self._device, stream))
        return to_weights, kept
