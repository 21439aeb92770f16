"""A paged key/value cache in 4 bits on the GPU, with the attention that reads it and the eviction that shortens it: the
host side of the ``t3_op_kv4_*`` / ``t3_op_attn_kv4`` entry points of ``lib/libt3hip.so`` (include/t3_hip.h).

It stands beside the engine's bf16 pool (which the reference leaves to vLLM, src/chatterbox_vllm/tts.py:130-140) and has no
counterpart in the reference: 4.25 bits a value, 3.76 times less to store and to read per decode step.

    cache = KV4Cache(num_kv_heads=16, head_dim=64, num_pages=4096, num_streams=64, max_pages=16)
    cache.block_table[s, i] = page                               # page allocation is the caller's
    batch = cache.batch(seq_start, streams, ctx, rows=R, max_rows=1, max_ctx=n)      # one object for the calls of a step
    cache.append(k, v, batch)
    out = cache.attend(q, batch, weights=weights[0])             # weights: cache.new_weights(), where eviction is wanted
    new_ctx, kept = cache.evict(src, dst, ctx, keep=256, sink=34, recent=64, weights=weights)

All work is enqueued on torch's current stream of the cache's device; nothing synchronises, so the calls can be captured into a
graph.  torch carries device memory only.  Loading fails loudly when the library is missing (there is no CPU fallback)."""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Tuple

import torch
from torch._C import _cuda_getCurrentRawStream as _raw_stream, _cuda_getDevice as _current_device    # (a Stream object costs 2 us a call)

from . import _capi

PAGE = 64
_DTYPES = {torch.bfloat16: 0, torch.float16: 1}


def page_bytes(num_kv_heads: int, head_dim: int) -> int:
    """Bytes of one page (64 tokens, all key/value heads, K and V)."""
    n = _capi.load().t3_op_kv4_page_bytes(num_kv_heads, head_dim)
    if n <= 0:
        raise ValueError(f"no 4-bit cache for {num_kv_heads} heads of {head_dim} dims: head_dim must be 64 or 128, 1..1024 heads")
    return n


class KV4Batch:
    """The rows of a call: sequence i owns rows ``seq_start[i] .. seq_start[i + 1] - 1`` of the row tensors, which are entries
    ``ctx[i] - n_i .. ctx[i] - 1`` of stream ``streams[i]`` (< 0: skipped).  The three tensors (int32, on the cache's device) are
    read when the kernels run, so a captured graph follows what is written into them; ``rows``, ``max_rows`` and ``max_ctx`` are
    the host's bounds for them, by default the loosest ones (all rows in one sequence, the whole block table).  Grids and the work
    buffer of ``attend`` follow the bounds: what is known to be less is worth giving."""

    def __init__(self, cache: "KV4Cache", seq_start: torch.Tensor, streams: torch.Tensor, ctx: torch.Tensor, rows: int,
                 max_rows: Optional[int] = None, max_ctx: Optional[int] = None):
        n = streams.numel()
        for name, t, size in (("seq_start", seq_start, n + 1), ("streams", streams, n), ("ctx", ctx, n)):
            cache._int32(name, t, size)
        self.cache, self.n_seqs, self.rows = cache, n, rows
        self.max_rows = rows if max_rows is None else max_rows
        self.max_ctx = cache.max_pages * PAGE if max_ctx is None else max_ctx
        self._tensors = (seq_start, streams, ctx)                # keeps the addresses below alive
        self._c = _capi.T3Kv4Batch(seq_start.data_ptr(), streams.data_ptr(), ctx.data_ptr(), n, rows, self.max_rows, self.max_ctx)
        self._ref = C.byref(self._c)
        self._work = {}                                          # heads (negative: with weights) -> bytes of the work buffer


class KV4Cache:
    """``pool`` (uint8 [layers, pages, page_bytes], or None with ``num_pages`` and ``num_layers``: allocated, cleared) and
    ``block_table`` (int32 [streams, max_pages], or None with ``num_streams`` and ``max_pages``: allocated, all -1)."""

    def __init__(self, num_kv_heads: int, head_dim: int, pool: Optional[torch.Tensor] = None,
                 block_table: Optional[torch.Tensor] = None, num_pages: int = 0, num_layers: int = 1, num_streams: int = 0,
                 max_pages: int = 0, device: int = 0):
        self._lib = _capi.load()
        size = page_bytes(num_kv_heads, head_dim)
        if pool is None:
            if num_pages < 1 or num_layers < 1:
                raise ValueError("give a pool, or num_pages and num_layers")
            pool = torch.zeros(num_layers, num_pages, size, dtype=torch.uint8, device=torch.device("cuda", device))
        if block_table is None:
            if num_streams < 1 or max_pages < 1:
                raise ValueError("give a block_table, or num_streams and max_pages")
            block_table = torch.full((num_streams, max_pages), -1, dtype=torch.int32, device=pool.device)
        if pool.dtype != torch.uint8 or pool.dim() != 3 or pool.shape[2] != size:
            raise ValueError(f"pool must be uint8 [layers, pages, {size}], got {pool.dtype} {tuple(pool.shape)}")
        if pool.stride(2) != 1 or pool.stride(1) != size or min(pool.shape) < 1:
            raise ValueError("the pages of a layer must lie one behind the other")
        if pool.device.type != "cuda":
            raise ValueError(f"the pool must be on the GPU, got {pool.device}")
        self.device, self._index = pool.device, pool.device.index
        if block_table.dim() != 2 or block_table.numel() < 1:
            raise ValueError("block_table must be [streams, max_pages]")
        self._int32("block_table", block_table, block_table.numel())
        self._scale = 1.0 / math.sqrt(head_dim)
        self.num_kv_heads, self.head_dim, self.pool, self.block_table = num_kv_heads, head_dim, pool, block_table
        self.num_layers, self.num_pages = pool.shape[0], pool.shape[1]
        self.num_streams, self.max_pages = block_table.shape
        self._c = _capi.T3Kv4Cache(pool.data_ptr(), block_table.data_ptr(), pool.stride(0), self.num_layers, self.num_pages,
                                   self.num_streams, self.max_pages, num_kv_heads, head_dim)
        self._ref = C.byref(self._c)

    # -- bookkeeping -------------------------------------------------------------------------------------------------
    def batch(self, seq_start: torch.Tensor, streams: torch.Tensor, ctx: torch.Tensor, rows: int,
              max_rows: Optional[int] = None, max_ctx: Optional[int] = None) -> KV4Batch:
        return KV4Batch(self, seq_start, streams, ctx, rows, max_rows, max_ctx)

    def new_weights(self) -> torch.Tensor:
        """Accumulated attention weights of every entry, zero: fp32 [layers, streams, kv_heads, max_pages * 64]."""
        return torch.zeros(self.num_layers, self.num_streams, self.num_kv_heads, self.max_pages * PAGE, dtype=torch.float32,
                           device=self.device)

    # -- operators ---------------------------------------------------------------------------------------------------
    def append(self, k: torch.Tensor, v: torch.Tensor, batch: KV4Batch, layer: int = 0) -> None:
        """Quantises K and V rows [rows, kv_heads, head_dim] (bf16 or fp16; views with any row stride) into the cache."""
        dtype, k_stride = self._rows("k", k, batch, self.num_kv_heads)
        v_dtype, v_stride = self._rows("v", v, batch, self.num_kv_heads)
        if v_dtype != dtype:
            raise ValueError("k and v must have one type")
        self._run(self._lib.t3_op_kv4_append, self._ref, batch._ref, k.data_ptr(), v.data_ptr(), k_stride, v_stride, dtype, layer)

    def attend(self, q: torch.Tensor, batch: KV4Batch, scale: Optional[float] = None, layer: int = 0,
               weights: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Causal attention of rows q [rows, heads, head_dim] over their streams' entries, appended rows among them; heads is a
        multiple of kv_heads.  ``scale`` defaults to head_dim ** -0.5.  ``weights`` (fp32 [streams, kv_heads, width], one layer of
        ``new_weights()``): the softmax weights of every entry are added to it.  Returns ``out``, by default a new tensor in which
        rows of no sequence are undefined."""
        heads = q.shape[1] if q.dim() == 3 else 0
        if heads == 0 or heads % self.num_kv_heads:
            raise ValueError(f"q must be [rows, heads, {self.head_dim}] with heads a multiple of {self.num_kv_heads}, got {tuple(q.shape)}")
        dtype, q_stride = self._rows("q", q, batch, heads)
        if out is None:
            out = torch.empty_like(q)                            # dense, or q's own row stride where q is
            out_stride = out.stride(0) if batch.rows > 1 else heads * self.head_dim
        else:
            out_dtype, out_stride = self._rows("out", out, batch, heads)
            if out_dtype != dtype:
                raise ValueError("out must have q's type")
        w_ptr, w_stride = None, 0
        if weights is not None:
            self._weights(weights, 3)
            w_ptr, w_stride = weights.data_ptr(), weights.shape[2]       # (a contiguous tensor's stride of a single head may be any)
        size = batch._work.get(heads if weights is None else -heads)
        if size is None:
            size = self._lib.t3_op_attn_kv4_work_bytes(self._ref, batch._ref, heads, int(weights is not None))
            if size < 0:
                _capi.check(self._lib, 1)
            batch._work[heads if weights is None else -heads] = size
        # a buffer of this call's own: calls on other streams and captured graphs get others
        work = torch.empty_strided((size,), (1,), dtype=torch.uint8, device=self.device) if size else None
        self._run(self._lib.t3_op_attn_kv4, self._ref, batch._ref, q.data_ptr(), q_stride, out.data_ptr(), out_stride, heads,
                  dtype, self._scale if scale is None else scale, w_ptr, w_stride,
                  work.data_ptr() if size else None, size, layer)
        return out

    def read(self, batch: KV4Batch, layer: int = 0, n_layers: Optional[int] = None,
             dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
        """The batch's rows as the cache holds them: K and V [rows, kv_heads, head_dim], or, with ``n_layers``, those of layers
        layer .. layer + n_layers - 1: [n_layers, rows, kv_heads, head_dim].  Rows of no sequence are undefined."""
        if dtype not in _DTYPES:
            raise ValueError(f"dtype must be bfloat16 or float16, got {dtype}")
        self._batch(batch)
        layers = 1 if n_layers is None else n_layers
        if layers < 1:
            raise ValueError("n_layers must be at least 1")
        rows, kv, hd = batch.rows, self.num_kv_heads, self.head_dim
        if n_layers is None:                                     # (strides given: torch.empty takes 0.4 us longer)
            k = torch.empty_strided((rows, kv, hd), (kv * hd, hd, 1), dtype=dtype, device=self.device)
        else:
            k = torch.empty_strided((layers, rows, kv, hd), (rows * kv * hd, kv * hd, hd, 1), dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        self._run(self._lib.t3_op_kv4_read, self._ref, batch._ref, k.data_ptr(), v.data_ptr(), _DTYPES[dtype], layer, layers)
        return k, v

    def evict(self, src: torch.Tensor, dst: torch.Tensor, ctx: torch.Tensor, keep: int, sink: int, recent: int,
              weights: torch.Tensor, max_ctx: Optional[int] = None, layer: int = 0,
              n_layers: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """Moves stream src[i] (ctx[i] entries) into the pages of stream dst[i], shortened to its first ``sink``, its last
        ``recent`` and its most attended other entries, ``keep`` in all; per layer and key head by ``weights`` (fp32
        [n_layers, streams, kv_heads, width], as ``new_weights()`` makes it; dst's rows are rewritten).  Covers layers
        layer .. layer + n_layers - 1, by default all from ``layer`` on.  src keeps its pages.  Returns the new lengths, as ctx (-1: the
        entry was refused, see include/t3_hip.h) and the old index of every kept entry [n_layers, n, kv_heads, keep] (-1 behind
        the last)."""
        n = src.numel()
        for name, t in (("src", src), ("dst", dst), ("ctx", ctx)):
            self._int32(name, t, n)
        layers = self.num_layers - layer if n_layers is None else n_layers
        if layers < 1 or keep < 1:
            raise ValueError("n_layers and keep must be at least 1")
        self._weights(weights, 4)
        if weights.shape[0] != layers:
            raise ValueError(f"weights must have {layers} layers, got {weights.shape[0]}")
        new_ctx = torch.empty_like(ctx)
        kv = self.num_kv_heads
        kept = torch.empty_strided((layers, n, kv, keep), (n * kv * keep, kv * keep, keep, 1), dtype=torch.int32, device=self.device)
        width = weights.shape[3]
        d = _capi.T3Kv4EvictDesc(src.data_ptr(), dst.data_ptr(), ctx.data_ptr(), weights.data_ptr(), width, new_ctx.data_ptr(),
                                 kept.data_ptr(), n, min(width, self.max_pages * PAGE) if max_ctx is None else max_ctx, keep, sink, recent,
                                 layer, layers)
        self._run(self._lib.t3_op_kv4_evict, self._ref, C.byref(d))
        return new_ctx, kept

    # -- checks ------------------------------------------------------------------------------------------------------
    def _run(self, fn, *args) -> None:
        if _current_device() != self._index:
            with torch.cuda.device(self._index):
                return self._run(fn, *args)
        status = fn(*args, _raw_stream(self._index))
        if status:
            _capi.check(self._lib, status)

    def _int32(self, name: str, t: torch.Tensor, size: int) -> None:
        if t.dtype != torch.int32 or t.numel() != size or size < 1 or not t.is_contiguous() or t.get_device() != self._index:
            raise ValueError(f"{name} must be {size} contiguous int32 values on {self.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")

    def _batch(self, batch: KV4Batch) -> None:
        if batch.cache is not self:
            raise ValueError("the batch belongs to another cache")

    def _rows(self, name: str, t: torch.Tensor, batch: KV4Batch, heads: int) -> Tuple[int, int]:
        """Checks rows [batch.rows, heads, head_dim]; the type's number and the row stride."""
        if batch.cache is not self:
            self._batch(batch)
        dtype = _DTYPES.get(t.dtype)
        if dtype is None or t.shape != (batch.rows, heads, self.head_dim) or t.get_device() != self._index:
            raise ValueError(f"{name} must be bfloat16 or float16 [{batch.rows}, {heads}, {self.head_dim}] on {self.device}, "
                             f"got {t.dtype} {tuple(t.shape)} on {t.device}")
        row, head, dim = t.stride()
        if dim != 1 or (head != self.head_dim and heads != 1):   # (along one row or head a tensor's stride may be any number)
            raise ValueError(f"the heads of a row of {name} must lie one behind the other, strides are {t.stride()}")
        return dtype, row if batch.rows > 1 else heads * self.head_dim

    def _weights(self, w: torch.Tensor, dims: int) -> None:
        if w.dtype != torch.float32 or w.get_device() != self._index or w.dim() != dims or not w.is_contiguous() \
                or w.shape[-3:-1] != (self.num_streams, self.num_kv_heads):
            raise ValueError(f"weights must be contiguous fp32 [{'layers, ' if dims == 4 else ''}{self.num_streams}, {self.num_kv_heads}, width] "
                             f"on {self.device}, got {w.dtype} {tuple(w.shape)} on {w.device}")
