"""A paged cache of keys and values shared by many sequences, and the attention of new positions over it.

The reference configures a streaming recogniser whose chunks look back into cached frames
(/root/reference/voice-service/app/services/voice_interface.py:651-653, the call at :1753-1809 is commented out); it has no
cache of its own.  ``PagedKvCache`` is what a streaming or autoregressive model keeps next to ``SANMEncoder`` and
``ParaformerHead``: pages of ``page_size`` positions in one pool, a table of page numbers per sequence, 16-bit storage or
e4m3 bytes with a power-of-two scale per position and head.  One step is ``append`` (the new positions' keys and values go
into their pages) and ``attend`` (the new queries attend to everything their sequence holds); ``read`` gives dense copies
back.  Everything runs on the device through libasrfe; there is no CPU path.  An e4m3 value takes part as what the
queries' type has of it: exactly in bfloat16, in float16 rounded below 2 ** -14 and kept inside +-65504.

A batch is described by three int32 device tensors: ``cu_q`` [B + 1] (rows of the packed new tokens), ``kv_lens`` [B] (positions
of every sequence, the new ones included: they are its last) and ``block_table`` [B, n] (page numbers; -1 where there is no
page).
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _lib

_DT = {torch.float16: _lib.DT_F16, torch.bfloat16: _lib.DT_BF16}
PAGE_SIZES = (16, 32, 64, 128, 256)
HEAD_DIMS = (64, 128)


def _rows_apart(n, heads, dim, ts, hs):
    """Whether no two of the n x heads rows of ``dim`` elements at t * ts + h * hs share an element."""
    if (n > 1 and ts < dim) or (heads > 1 and hs < dim):
        return False
    if n == 1 or heads == 1 or ts >= (heads - 1) * hs + dim or hs >= (n - 1) * ts + dim:  # (one stride spans the other's rows)
        return True
    return all(abs(h * hs - t * ts) >= dim for h in range(1, heads) for t in (min(h * hs // ts, n - 1), min(h * hs // ts + 1, n - 1)))


class PagedKvCache:
    def __init__(self, ctx: _lib.Context, k: torch.Tensor, v: torch.Tensor, k_exp: torch.Tensor | None = None,
                 v_exp: torch.Tensor | None = None):
        """k, v [n_pages, n_heads, page_size, head_dim] of float16, bfloat16 or float8_e4m3fn; for float8_e4m3fn also k_exp,
        v_exp [n_pages, n_heads, page_size] uint8 (a stored value is code * 2 ** (exp - 127), exp 0 .. 254).  The buffers stay the
        caller's; see ``allocate`` for new ones."""
        e4m3 = k.dtype == torch.float8_e4m3fn
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or not (e4m3 or k.dtype in _DT):
            raise ValueError("PagedKvCache: k and v must have one shape [n_pages, n_heads, page_size, head_dim] and one type, "
                             "float16, bfloat16 or float8_e4m3fn")
        if k.shape[2] not in PAGE_SIZES or k.shape[3] not in HEAD_DIMS or k.shape[0] < 1 or not 1 <= k.shape[1] <= 256:
            raise ValueError(f"PagedKvCache: page_size in {PAGE_SIZES}, head_dim in {HEAD_DIMS}, 1 to 256 heads, at least one page")
        if e4m3 != (k_exp is not None) or e4m3 != (v_exp is not None):
            raise ValueError("PagedKvCache: k_exp and v_exp belong to a float8_e4m3fn cache and to no other")
        bufs = [k, v] + ([k_exp, v_exp] if e4m3 else [])
        if e4m3 and any(t.dtype != torch.uint8 or t.shape != k.shape[:3] for t in bufs[2:]):
            raise ValueError("PagedKvCache: k_exp and v_exp must be uint8 [n_pages, n_heads, page_size]")
        if any(not t.is_cuda or not t.is_contiguous() or t.device != k.device for t in bufs):
            raise ValueError("PagedKvCache: buffers must be contiguous CUDA tensors on one device")
        if any(t.data_ptr() % 16 for t in bufs):
            raise ValueError("PagedKvCache: buffers must be 16-byte aligned")
        self.ctx, self.k, self.v, self.k_exp, self.v_exp = ctx, k, v, k_exp, v_exp
        self.n_pages, self.n_heads, self.page_size, self.head_dim = k.shape
        self.dtype, self.device, self._index = k.dtype, k.device, k.get_device()
        self._c = _lib.KvCache(k.data_ptr(), v.data_ptr(), k_exp.data_ptr() if e4m3 else None, v_exp.data_ptr() if e4m3 else None,
                               *k.shape[:1], self.page_size, self.n_heads, self.head_dim,
                               _lib.DT_E4M3 if e4m3 else _DT[k.dtype])
        self._ref = C.byref(self._c)

    @classmethod
    def allocate(cls, ctx: _lib.Context, n_pages: int, page_size: int, n_heads: int, head_dim: int = 128,
                 dtype: torch.dtype = torch.float16, device="cuda") -> "PagedKvCache":
        """A cache with buffers of its own (zeros)."""
        shape = (n_pages, n_heads, page_size, head_dim)
        e4m3 = dtype == torch.float8_e4m3fn
        k, v = (torch.zeros(shape, dtype=torch.uint8 if e4m3 else dtype, device=device) for _ in range(2))
        if not e4m3:
            return cls(ctx, k, v)
        return cls(ctx, k.view(dtype), v.view(dtype), *(torch.full(shape[:3], 127, dtype=torch.uint8, device=device) for _ in range(2)))

    # ---- checks (in the order of what is cheap to ask: small calls are bound by the host) -------------------
    def _plan(self, who, lens, table, cu=None):
        i32, index = torch.int32, self._index
        for t, dim in ((lens, 1), (table, 2)) if cu is None else ((lens, 1), (table, 2), (cu, 1)):
            if t.dtype is not i32 or t.dim() != dim or t.get_device() != index or not t.is_contiguous():
                raise ValueError(f"PagedKvCache.{who}: cu_q, kv_lens and block_table must be contiguous int32 tensors [B + 1], [B] and "
                                 f"[B, n] on {self.device}")
        if table.shape[0] != lens.shape[0] or (cu is not None and cu.shape[0] != lens.shape[0] + 1):
            raise ValueError(f"PagedKvCache.{who}: one length and one row of the table per sequence, cu_q one entry more")

    def _rows(self, who, name, t, heads):
        """One [n, heads, head_dim] operand: its rows lie anywhere, their elements side by side.  -> token and head stride"""
        dtype, shape = t.dtype, t.shape
        if dtype not in _DT or len(shape) != 3 or shape[2] != self.head_dim or (heads is not None and shape[1] != heads) \
                or t.get_device() != self._index:
            raise ValueError(f"PagedKvCache.{who}: {name} must be a float16 or bfloat16 tensor [n, {heads or 'heads'}, {self.head_dim}] "
                             f"on {self.device}")
        if dtype is not self.dtype and self.dtype in _DT:
            raise ValueError(f"PagedKvCache.{who}: {name} must be {self.dtype}, as the cache is")
        ts, hs, es = t.stride()
        if (es != 1 or ts & 7 or hs & 7 or t.data_ptr() & 15) and t.numel():
            raise ValueError(f"PagedKvCache.{who}: {name} needs rows of contiguous elements, 16-byte aligned (strides in multiples of 8)")
        return ts, hs

    def _call(self, fn, *args):
        """fn(context, cache, *args, stream) on the cache's device."""
        if torch.cuda.current_device() != self._index:
            with torch.cuda.device(self._index):
                return self._call(fn, *args)
        rc = fn(self.ctx.handle, self._ref, *args, _lib.raw_stream(self._index))
        if rc:
            self.ctx.check(rc)

    # ---- operators ---------------------------------------------------------------------------
    def append(self, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor, kv_lens: torch.Tensor, block_table: torch.Tensor) -> None:
        """Writes the new rows' keys and values k, v [n, n_heads, head_dim] into their pages (quantised as they are written in
        an e4m3 cache).  Slices of a fused projection may be passed as they are."""
        self._plan("append", kv_lens, block_table, cu_q)
        kts, khs = self._rows("append", "k", k, self.n_heads)
        vts, vhs = self._rows("append", "v", v, self.n_heads)
        n = k.shape[0]
        if v.shape[0] != n or v.dtype is not k.dtype:
            raise ValueError("PagedKvCache.append: k and v must agree in shape and type")
        self._call(self.ctx.lib.asrfe_kv_append, k.data_ptr(), v.data_ptr(), _DT[k.dtype], kts, khs, vts, vhs, n, cu_q.data_ptr(),
                   kv_lens.data_ptr(), block_table.data_ptr(), block_table.shape[1], kv_lens.shape[0])

    def read(self, kv_lens: torch.Tensor, block_table: torch.Tensor, t_max: int, dtype: torch.dtype | None = None):
        """-> k, v [B, t_max, n_heads, head_dim]: positions 0 .. t_max - 1 of every sequence, zero at and past kv_lens[b] and
        where there is no page.  ``dtype``: of the copies (the cache's own for 16-bit caches; float16 unless given for e4m3)."""
        self._plan("read", kv_lens, block_table)
        dtype = dtype or (self.dtype if self.dtype in _DT else torch.float16)
        if dtype not in _DT or (self.dtype in _DT and dtype != self.dtype):
            raise ValueError("PagedKvCache.read: dtype must be the cache's own, float16 or bfloat16 for an e4m3 cache")
        batch = kv_lens.shape[0]
        k, v = torch.empty((2, batch, t_max, self.n_heads, self.head_dim), dtype=dtype, device=self.device).unbind(0)
        if batch and t_max:
            self._call(self.ctx.lib.asrfe_kv_read, kv_lens.data_ptr(), block_table.data_ptr(), block_table.shape[1], batch, t_max,
                       k.data_ptr(), v.data_ptr(), _DT[dtype])
        return k, v

    def attend(self, q: torch.Tensor, cu_q: torch.Tensor, kv_lens: torch.Tensor, block_table: torch.Tensor, window: int = 0,
               sinks: int = 0, causal: bool = True, scale: float | None = None, max_kv: int | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """q [n, heads, head_dim] (heads a multiple of the cache's) -> out of the same shape: the softmax-weighted values of
        the positions each row sees.  A row sees its sequence's positions up to its own (all of them with ``causal=False``);
        ``window`` > 0 keeps the last ``window`` up to its own, and the first ``sinks`` stay visible beside them.  A row
        that sees nothing is zero; rows behind cu_q[B] are not written (those of a new tensor hold no meaning).  ``scale``
        defaults to 1 / sqrt(head_dim); ``max_kv`` bounds kv_lens (the table's width unless given: a tighter bound shapes
        the launch better).  Statistics and sums are fp32, the weights enter their product in q's type; infinities and NaN
        reach the rows that see them and no other.  A call's work is cut by its mean: single tokens over very long caches are
        better off in a call of their own than beside a long prompt."""
        self._plan("attend", kv_lens, block_table, cu_q)
        qts, qhs = self._rows("attend", "q", q, None)
        n, heads, dim = q.shape
        if heads < 1 or heads % self.n_heads:
            raise ValueError(f"PagedKvCache.attend: the heads of q must be a multiple of the cache's {self.n_heads}")
        if window < 0 or sinks < 0:
            raise ValueError("PagedKvCache.attend: window and sinks must not be negative")
        if out is None:
            out = torch.empty((n, heads, dim), dtype=q.dtype, device=self.device)
            ots, ohs = heads * dim, dim
        else:
            ots, ohs = self._rows("attend", "out", out, heads)
            if out.shape[0] != n or out.dtype is not q.dtype:
                raise ValueError("PagedKvCache.attend: out must have q's shape and type")
            if n and not _rows_apart(n, heads, dim, ots, ohs):
                raise ValueError("PagedKvCache.attend: the rows of out must not overlap")
        if not n:
            return out
        batch, width = block_table.shape
        most = width * self.page_size
        max_kv = most if max_kv is None else min(int(max_kv), most)
        window, sinks = min(window, 1 << 30), min(sinks, 1 << 30)  # (a position is less: what does not fit 32 bits must not wrap)
        nbytes = self.ctx.lib.asrfe_paged_attention_workspace_bytes(self.ctx.handle, self._ref, n, heads, batch, max_kv)
        if nbytes < 0:
            raise ValueError("PagedKvCache.attend: bad sizes")
        # from the allocator of the current stream, so calls on several streams and captured graphs never share one
        ws = torch.empty((nbytes,), dtype=torch.uint8, device=self.device) if nbytes else None
        self._call(self.ctx.lib.asrfe_paged_attention, q.data_ptr(), _DT[q.dtype], qts, qhs, n, heads, cu_q.data_ptr(), kv_lens.data_ptr(),
                   block_table.data_ptr(), width, batch, max_kv, window, sinks, 1 if causal else 0,
                   1.0 / math.sqrt(dim) if scale is None else scale, out.data_ptr(), ots, ohs, ws.data_ptr() if nbytes else None, nbytes)
        return out
