"""The paged key/value cache of the full-attention blocks and the attention
over it, on CUDA tensors (``include/moe_b200.h``, section 3).

Beside ``NativeDelta`` (the DeltaNet mixer's step) this is the other mixer of
the hybrid model: a serving loop writes each call's new keys and values and
attends over the cache, for prompts, chunks of prompts, drafted tokens and
single tokens alike::

    cache = PagedKVCache.empty(num_pages, page_size, kv_heads, head_dim, Q8_0, device)
    batch = KVBatch(q_start, kv_lens, page_table)   # int32 CUDA tensors
    cache.write(batch, k, v)                        # [tokens, kv_heads, head_dim]
    out = cache.attend(batch, q)                    # [tokens, q_heads, head_dim]
    k, v = cache.read(batch, dtype=torch.float16)   # the same rows, dequantised

Rows ``q_start[b] .. q_start[b+1]-1`` of the tokens belong to sequence b;
``kv_lens[b]`` counts its cached tokens, the new ones included.  All calls are
asynchronous on torch's current stream of the cache's device (or ``stream``),
read the batch on the device, and can be captured in a CUDA graph.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from .formats import BF16, F16, F32, Q8_0

TYPE_IDS = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
_BYTES = {torch.float32: 4, torch.float16: 2, torch.bfloat16: 2}
BLOCK_VALUES = 32   # values that share one scale of a Q8_0 cache


class KVBatch:
    """The sequences of a call: ``q_start`` [B + 1], ``kv_lens`` [B] and
    ``page_table`` [B, max_pages], int32 CUDA tensors.  Their contents may
    change between calls (a captured graph reads the current ones)."""

    def __init__(self, q_start: torch.Tensor, kv_lens: torch.Tensor, page_table: torch.Tensor):
        for t, dim in ((q_start, 1), (kv_lens, 1), (page_table, 2)):
            if t.dtype != torch.int32 or t.dim() != dim or not t.is_cuda:
                raise ValueError("KVBatch needs int32 CUDA tensors q_start [B + 1], kv_lens [B], "
                                 "page_table [B, max_pages]")
        n = kv_lens.shape[0]
        if q_start.shape[0] != n + 1 or page_table.shape[0] != n:
            raise ValueError("KVBatch shapes do not agree on the number of sequences")
        if not (q_start.device == kv_lens.device == page_table.device):
            raise ValueError("KVBatch tensors must be on one device")
        if not q_start.is_contiguous() or not kv_lens.is_contiguous() or (
                page_table.numel() and page_table.stride(1) != 1):
            raise ValueError("KVBatch tensors must have contiguous rows")
        if n > 1 and page_table.stride(0) < page_table.shape[1]:
            raise ValueError("KVBatch page table rows must not overlap")
        self.q_start, self.kv_lens, self.page_table = q_start, kv_lens, page_table
        self.device = q_start.device
        self.index = q_start.get_device()
        self.sequences = n
        self.max_pages = page_table.shape[1]
        self._structs: dict[int, _lib.KVBatchStruct] = {}

    def struct(self, tokens: int) -> _lib.KVBatchStruct:
        s = self._structs.get(tokens)
        if s is None:
            if len(self._structs) > 64:
                self._structs.clear()
            stride = max(self.page_table.stride(0), self.max_pages)
            s = self._structs[tokens] = _lib.KVBatchStruct(
                self.sequences, tokens, self.max_pages, 0, stride, self.q_start.data_ptr(),
                self.kv_lens.data_ptr(), self.page_table.data_ptr())
        return s


def _raw_stream(index: int) -> int:
    """Handle of torch's current stream of a device."""
    return torch.cuda.current_stream(index).cuda_stream


# the same without building a Stream object (about 2 us of a call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _raw_stream)


def _overlap(n: int, ns: int, m: int, ms: int, length: int) -> bool:
    """Whether two of the n x m rows of ``length`` values at i ns + j ms share
    a value."""
    if n <= 1 or m <= 1:
        return (n > 1 and ns < length) or (m > 1 and ms < length)
    if ns < length or ms < length:
        return True
    if ns >= (m - 1) * ms + length or ms >= (n - 1) * ns + length:
        return False
    # neither axis lies within a step of the other: rows j apart meet rows i or
    # i + 1 apart
    return any((i < n and r < length) or (i + 1 < n and ns - r < length)
               for i, r in (divmod(j * ms, ns) for j in range(1, m)))


class PagedKVCache:
    """Keys and values [num_pages, kv_heads, page_size, head_dim]: fp16, bf16,
    or int8 codes with binary16 scales [..., head_dim / 32] (Q8_0 arithmetic:
    a value is scale * code).  The tensors are the caller's and are used in
    place."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scales: torch.Tensor | None = None,
                 v_scales: torch.Tensor | None = None):
        self.lib = _lib.load()
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError("cache k and v must be [num_pages, kv_heads, page_size, head_dim] "
                             "of one shape and dtype")
        pages, heads, page_size, dim = k.shape
        tensors = [k, v]
        if k.dtype == torch.int8:
            self.type = Q8_0
            shape = (pages, heads, page_size, dim // BLOCK_VALUES)
            for s in (k_scales, v_scales):
                if s is None or s.dtype != torch.float16 or tuple(s.shape) != shape:
                    raise ValueError(f"a Q8_0 cache needs fp16 scales of shape {shape}")
            tensors += [k_scales, v_scales]
        elif k.dtype in (torch.float16, torch.bfloat16):
            self.type = TYPE_IDS[k.dtype]
            if k_scales is not None or v_scales is not None:
                raise ValueError("only a Q8_0 cache has scales")
        else:
            raise ValueError("cache dtype must be fp16, bf16 or int8 (Q8_0)")
        if dim % BLOCK_VALUES or not 32 <= dim <= 256:
            raise ValueError("head_dim must be a multiple of 32 between 32 and 256")
        if page_size & (page_size - 1) or not 16 <= page_size <= 256:
            raise ValueError("page_size must be a power of two between 16 and 256")
        if pages < 1 or heads < 1 or heads > 1024 or pages * heads > 0x7fffffff:
            raise ValueError("the cache needs at least one page and 1 to 1024 heads, and fewer "
                             "than 2^31 pages * heads")
        for t in tensors:
            if not t.is_cuda or t.device != k.device or not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError("cache tensors must be contiguous, 16-byte aligned CUDA tensors "
                                 "on one device")
        self.k, self.v, self.k_scales, self.v_scales = k, v, k_scales, v_scales
        self.device = k.device
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = pages, heads, page_size, dim
        ptr = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
        self._struct = _lib.KVCacheStruct(self.type, pages, page_size, heads, dim, 0, ptr(k),
                                          ptr(v), ptr(k_scales), ptr(v_scales))
        self._ref = C.byref(self._struct)
        self._ws_bytes: dict[tuple, int] = {}
        self._index = k.get_device()
        self._q_dtypes = ((torch.float16, torch.bfloat16) if self.type == Q8_0 else (k.dtype,))

    @classmethod
    def empty(cls, num_pages: int, page_size: int, kv_heads: int, head_dim: int, type_id: int,
              device) -> "PagedKVCache":
        """A cache of ``type_id`` F16, BF16 or Q8_0 (``formats``) with
        uninitialised pages."""
        dtype = {F16: torch.float16, BF16: torch.bfloat16, Q8_0: torch.int8}.get(type_id)
        if dtype is None:
            raise ValueError("cache type must be F16, BF16 or Q8_0")
        shape = (num_pages, kv_heads, page_size, head_dim)
        k, v = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))
        if dtype != torch.int8:
            return cls(k, v)
        scales = (*shape[:3], head_dim // BLOCK_VALUES)
        return cls(k, v, *(torch.empty(scales, dtype=torch.float16, device=device)
                           for _ in range(2)))

    # ---------------------------------------------------------------- checks

    def _elsewhere(self, stream):
        """A context that makes `stream` current (and the cache's device), or
        None when the call can run as it is."""
        if stream is None:
            if torch.cuda.current_device() == self._index:
                return None
            return torch.cuda.device(self.device)
        if stream.device != self.device:
            raise ValueError("the stream must belong to the cache's device")
        return torch.cuda.stream(stream)

    def _rows(self, t, heads, dtypes, what, output=False):
        """Address and token / head strides of `t` [tokens, heads, head_dim]
        with contiguous, 16-byte aligned head rows, and the tensor that holds
        them: `t`, or a contiguous copy of an input that is not aligned.  The
        stride along an axis of one entry, which torch leaves arbitrary, is
        0."""
        shape = t.shape
        if (len(shape) != 3 or shape[1] != heads or shape[2] != self.head_dim
                or t.dtype not in dtypes or t.get_device() != self._index):
            raise ValueError(f"{what} must be a [tokens, {heads}, {self.head_dim}] CUDA tensor on "
                             f"the cache's device, dtype one of {[str(d) for d in dtypes]}")
        ts, hs, ds = t.stride()
        if shape[0] <= 1:
            ts = 0
        if heads == 1:
            hs = 0
        ptr = t.data_ptr()
        if output and _overlap(shape[0], ts, heads, hs, self.head_dim):
            raise ValueError(f"{what} must have rows that do not overlap")
        if ds != 1 or (ptr | ts * _BYTES[t.dtype] | hs * _BYTES[t.dtype]) & 15:
            if output:
                raise ValueError(f"{what} must have contiguous, 16-byte aligned head rows")
            t = t.clone(memory_format=torch.contiguous_format)
            return t.data_ptr(), heads * self.head_dim, self.head_dim, t
        return ptr, ts, hs, t

    def _status(self, status):
        if status is None:
            return None
        if (status.dtype != torch.int32 or status.numel() < 1
                or status.get_device() != self._index):
            raise ValueError("status must be an int32 tensor on the cache's device")
        return status.data_ptr()

    # ----------------------------------------------------------------- calls

    def write(self, batch: KVBatch, k: torch.Tensor, v: torch.Tensor, status=None,
              stream=None) -> None:
        """Store new rows k, v [tokens, kv_heads, head_dim] (fp32, fp16 or
        bf16, any strides) in the batch's pages (``moe_b200_kv_write``).
        ``status`` (int32 CUDA tensor, optional) receives 0 or a sum of
        ``_lib.KV_*`` bits."""
        other = self._elsewhere(stream)
        if other is not None:
            with other:
                return self.write(batch, k, v, status)
        kp, kts, khs, k = self._rows(k, self.kv_heads, TYPE_IDS, "k")
        vp, vts, vhs, v = self._rows(v, self.kv_heads, (k.dtype,), "v")
        tokens = k.shape[0]
        if tokens != v.shape[0] or batch.index != self._index:
            raise ValueError("k, v and the batch must agree in tokens and device")
        st = self.lib.moe_b200_kv_write(
            self._ref, batch.struct(tokens), TYPE_IDS[k.dtype], kp, kts, khs, vp, vts, vhs,
            self._status(status), _raw_stream(self._index))
        if st:
            _lib.check(st, "moe_b200_kv_write")

    def read(self, batch: KVBatch, tokens: int | None = None, dtype: torch.dtype | None = None,
             out: tuple[torch.Tensor, torch.Tensor] | None = None, status=None, stream=None):
        """The cached (k, v) at the batch's rows, [tokens, kv_heads, head_dim]
        of ``dtype`` (``moe_b200_kv_read``): with ``q_start`` the running sum
        of ``kv_lens``, whole sequences.  Give ``out``, or ``tokens`` and
        ``dtype`` (default: fp16 for a Q8_0 cache, else the cache's dtype);
        rows behind the last sequence are left as they are (uninitialised
        without ``out``)."""
        other = self._elsewhere(stream)
        if other is not None:
            with other:
                return self.read(batch, tokens, dtype, out, status)
        if out is None:
            if tokens is None or tokens < 0:
                raise ValueError("read needs out, or the number of tokens")
            if dtype is None:
                dtype = torch.float16 if self.type == Q8_0 else self.k.dtype
            shape = (2, tokens, self.kv_heads, self.head_dim)
            k, v = self.k.new_empty(shape, dtype=dtype).unbind(0)
        else:
            k, v = out
        kp, kts, khs, _ = self._rows(k, self.kv_heads, TYPE_IDS, "out k", output=True)
        vp, vts, vhs, _ = self._rows(v, self.kv_heads, (k.dtype,), "out v", output=True)
        tokens = k.shape[0]
        if tokens != v.shape[0] or batch.index != self._index:
            raise ValueError("out and the batch must agree in tokens and device")
        st = self.lib.moe_b200_kv_read(
            self._ref, batch.struct(tokens), TYPE_IDS[k.dtype], kp, kts, khs, vp, vts, vhs,
            self._status(status), _raw_stream(self._index))
        if st:
            _lib.check(st, "moe_b200_kv_read")
        return k, v

    def attend(self, batch: KVBatch, q: torch.Tensor, out: torch.Tensor | None = None,
               lse: torch.Tensor | None = None, scale: float | None = None, causal: bool = True,
               window: int = 0, status=None, stream=None) -> torch.Tensor:
        """Attention of the batch's rows q [tokens, q_heads, head_dim] (fp16
        or bf16, the cache's own dtype unless it is Q8_0) over their cached
        tokens (``moe_b200_attend``).  ``scale`` defaults to
        head_dim ** -0.5; ``window`` > 0 keeps a causal row's last ``window``
        tokens; ``lse`` (fp32 [tokens, q_heads], contiguous) receives the
        logarithm of the softmax sum.  Rows without a token get zeros and
        -inf; rows behind the last sequence are left as they are (``out`` is
        allocated uninitialised when not given).  ``out`` may be ``q``; no
        gradient is recorded."""
        other = self._elsewhere(stream)
        if other is not None:
            with other:
                return self.attend(batch, q, out, lse, scale, causal, window, status)
        shape = q.shape
        heads = shape[1] if len(shape) == 3 else 0
        if heads < 1 or heads % self.kv_heads:
            raise ValueError("q must be [tokens, q_heads, head_dim], q_heads a multiple of "
                             "kv_heads")
        qp, qts, qhs, q = self._rows(q, heads, self._q_dtypes, "q")
        if batch.index != self._index:
            raise ValueError("q and the batch must be on the cache's device")
        if window < 0 or (window and not causal):
            raise ValueError("window must be positive, and needs causal")
        window = min(window, 0x7fffffff)   # wider than any sequence: no limit
        tokens = shape[0]
        if out is None:
            out = q.new_empty(shape)
            op, ots, ohs = out.data_ptr(), heads * self.head_dim, self.head_dim
        else:
            op, ots, ohs, _ = self._rows(out, heads, (q.dtype,), "out", output=True)
            if out.shape[0] != tokens:
                raise ValueError("out must have q's shape")
        if lse is not None and (lse.dtype != torch.float32 or tuple(lse.shape) != (tokens, heads)
                                or not lse.is_contiguous() or lse.device != self.device):
            raise ValueError("lse must be a contiguous fp32 [tokens, q_heads] tensor on the "
                             "cache's device")
        bs = batch.struct(tokens)
        key = (tokens, heads, batch.sequences, batch.max_pages)
        need = self._ws_bytes.get(key)
        if need is None:
            n = C.c_size_t(0)
            _lib.check(self.lib.moe_b200_attend_workspace(self._ref, bs, heads, C.byref(n)),
                       "moe_b200_attend_workspace")
            if len(self._ws_bytes) > 4096:
                self._ws_bytes.clear()
            need = self._ws_bytes[key] = n.value
        # a workspace of the call's own: torch's allocator hands it to the next
        # call on this stream, or keeps it with the graph that captured it
        ws = q.new_empty(max(need, 256), dtype=torch.uint8)
        st = self.lib.moe_b200_attend(
            self._ref, bs, TYPE_IDS[q.dtype], qp, qts, qhs, heads, op, ots, ohs,
            lse.data_ptr() if lse is not None else None,
            self.head_dim ** -0.5 if scale is None else scale, 1 if causal else 0, window,
            ws.data_ptr(), max(need, 256), self._status(status), _raw_stream(self._index))
        if st:
            _lib.check(st, "moe_b200_attend")
        return out
