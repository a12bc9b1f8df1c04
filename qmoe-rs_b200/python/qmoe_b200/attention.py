"""The attention half of a decoder layer in 8 bits, over the C ABI.

  Int8Tensor      a weight matrix in 8 bits; forward quantises the tokens
  plan_pages      block table and slot map of a step, from request lengths
  KVCache         paged keys and values in 8 bits: append, attend
  AttentionBlock  x + out(attention(qkv(LN(x)))), the half in front of
                  QMoELayer.forward_block (qmoe-rs src/model.rs:372-413);
                  BlockChain runs both halves of every layer

Activations are CUDA torch tensors, float32 or bfloat16.  Calls are
asynchronous on the current torch stream, and workspaces come from torch's
allocator in each call, so any of them may be captured into a CUDA graph.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Callable, Optional, Tuple

import torch

from . import capi
from .layer import Context, _ptr, default_context

_I64 = ctypes.c_int64
_CODE = {torch.float32: capi.QMOE_DTYPE_F32, torch.bfloat16: capi.QMOE_DTYPE_BF16}
_fns: dict = {}


def _fn(name: str):
    """The entry point, looked up once: these calls are as short as a few microseconds."""
    f = _fns.get(name)
    if f is None:
        f = _fns[name] = getattr(capi.lib(), name)
    return f


# the current stream's handle without a Stream object around it (1.3 us less)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda device: torch.cuda.current_stream(device).cuda_stream)


def _use_stream(ctx: Context) -> None:
    capi.check(_fn("qmoe_ctx_set_stream")(ctx.handle, _raw_stream(ctx.device)))


def _on(ctx: Context, name: str, t) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    if t.get_device() != ctx.device:
        raise ValueError(f"{name} is on cuda:{t.get_device()}, the context on cuda:{ctx.device}")


def _code(t) -> int:
    c = _CODE.get(t.dtype)
    if c is None:
        raise TypeError(f"activations must be float32 or bfloat16, got {t.dtype}")
    return c


def _context_of(x, ctx: Optional[Context]) -> Context:
    if ctx is not None:
        return ctx
    return default_context(x.device.index if isinstance(x, torch.Tensor) and x.is_cuda else 0)


def _i32(ctx: Context, t, name: str, shape) -> int:
    _on(ctx, name, t)
    if t.dtype != torch.int32 or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous int32 {list(shape)}, got {t.dtype} {list(t.shape)}")
    return t.data_ptr()


def quantize_int8(x, ctx: Optional[Context] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(codes int8 [rows, cols], scales f32 [rows]) of x [rows, cols]: with r
    the row's largest magnitude, code = round(127 x / r) and scale = r / 127."""
    ctx = _context_of(x, ctx)
    _on(ctx, "x", x)
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError(f"x must be [rows, cols], got {list(x.shape)}")
    dt = _code(x)
    rows, cols = x.shape
    stride, unit = x.stride()
    if unit != 1 or stride < cols:                # rows that repeat or overlap (expand, unfold) as well
        x = x.contiguous()
        stride = cols
    codes = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scales = torch.empty(x.shape[0], dtype=torch.float32, device=x.device)
    _use_stream(ctx)
    capi.call("qmoe_quantize_int8", ctx.handle, x.data_ptr(), dt, rows, cols, stride, codes.data_ptr(), scales.data_ptr())
    return codes, scales


class Int8Tensor:
    """Device-resident 8-bit weight matrix with a scale per output channel,
    the 8-bit counterpart of PackedQMoETensor (qmoe-rs src/tensor.rs:16-121)."""

    def __init__(self, handle, ctx: Context, scales):
        self._h = handle
        self.ctx = ctx
        self.scales = scales
        rows, cols, n = _I64(), _I64(), _I64()
        capi.call("qmoe_int8_shape", handle, ctypes.byref(rows), ctypes.byref(cols))
        capi.call("qmoe_int8_workspace", handle, 1, ctypes.byref(n))
        self.shape = (int(rows.value), int(cols.value))
        self._row_bytes = int(n.value)

    @classmethod
    def from_bytes(cls, codes, shape: Tuple[int, int], scales, ctx: Optional[Context] = None) -> "Int8Tensor":
        """codes int8 [out, in] and scales f32 [out], both host or both device memory."""
        ctx = _context_of(codes, ctx)
        out_f, in_f = (int(v) for v in shape)
        for name, a, kind, n in (("codes", codes, "int8", out_f * in_f), ("scales", scales, "float32", out_f)):
            have = a.numel() if isinstance(a, torch.Tensor) else a.size
            if str(a.dtype).replace("torch.", "") != kind or have != n:
                raise ValueError(f"{name} must hold {n} {kind} values, got {have} of {a.dtype}")
        cp, kind, keep1 = _ptr(codes)
        sp, kind2, keep2 = _ptr(scales)
        if kind != kind2:
            raise ValueError("codes and scales must both be host or both device memory")
        if kind == capi.QMOE_PTR_DEVICE:
            _on(ctx, "codes", codes)
            _on(ctx, "scales", scales)
        _use_stream(ctx)
        h = ctypes.c_void_p()
        capi.call("qmoe_int8_create", ctx.handle, cp, sp, out_f, in_f, kind, ctypes.byref(h))
        return cls(h, ctx, scales)

    @classmethod
    def from_float(cls, weight, ctx: Optional[Context] = None) -> "Int8Tensor":
        """A CUDA weight [out, in] in float32 or bfloat16, quantised by output channel."""
        codes, scales = quantize_int8(weight, ctx)
        return cls.from_bytes(codes, tuple(weight.shape), scales, ctx)

    def forward(self, x, residual=None, out=None):
        """y [..., out] = x [..., in] times the weight (+ residual), x quantised by token.

        `out` may be `residual` itself."""
        out_f, in_f = self.shape
        ctx = self.ctx
        _on(ctx, "x", x)
        dt = _code(x)
        shape = x.shape
        if len(shape) < 1 or shape[-1] != in_f:
            raise ValueError(f"x {list(shape)} does not end in in_features = {in_f}")
        rows = x if len(shape) == 2 else x.reshape(-1, in_f)
        stride, unit = rows.stride()
        if unit != 1 or stride < in_f:
            rows = rows.contiguous()
            stride = in_f
        batch = rows.shape[0]
        shape = (*shape[:-1], out_f)
        if out is None:
            out = torch.empty(shape, dtype=x.dtype, device=x.device)
        else:
            self._like(out, "out", shape, x.dtype)
        if residual is not None:
            self._like(residual, "residual", shape, x.dtype)
        need = batch * self._row_bytes
        ws = torch.empty(need, dtype=torch.uint8, device=x.device)
        _use_stream(ctx)
        capi.check(_fn("qmoe_int8_forward")(
            self._h, rows.data_ptr(), dt, batch, stride, residual.data_ptr() if residual is not None else None,
            out.data_ptr(), ws.data_ptr(), need))
        return out

    def _like(self, t, name: str, shape, dtype) -> None:
        _on(self.ctx, name, t)
        if t.shape != shape or t.dtype != dtype or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous {dtype} {list(shape)}")

    def close(self):
        if getattr(self, "_h", None):
            capi.lib().qmoe_int8_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


@dataclass
class PagePlan:
    """A step's place in the cache (qmoe_kv_plan)."""

    block_table: torch.Tensor   # [requests, max_blocks] int32, updated in place
    q_start: torch.Tensor       # [requests + 1] first row of each request
    kv_lens: torch.Tensor       # [requests] tokens held after the step, 0 for a denied request
    slots: torch.Tensor         # [rows] block * block_size + offset; -1 for none, and where the table's entry is no block
    positions: torch.Tensor     # [rows] place in the request, -1 for none
    taken: torch.Tensor         # [1] blocks taken from the front of the free list
    max_kv: int = 0             # longest kv_lens if known on the host


def plan_pages(cached_lens, new_lens, block_table, free_blocks, block_size: int, num_tokens: int,
               num_blocks: int, max_kv: int = 0, ctx: Optional[Context] = None) -> PagePlan:
    """Block table and slot map of a step: request r holds cached_lens[r] tokens
    in the blocks of its row of block_table [requests, max_blocks] and gets
    new_lens[r] more, taking what blocks it lacks from free_blocks in order.
    num_tokens: rows of the step's token buffer; num_blocks: of the cache.  All
    tensors int32 on the GPU; the host reads nothing.  A request that does not
    fit is denied: kv_lens 0, slots and positions -1."""
    ctx = _context_of(cached_lens, ctx)
    for name, t in (("block_table", block_table), ("free_blocks", free_blocks)):
        _on(ctx, name, t)
    if block_table.dim() != 2 or free_blocks.dim() != 1:
        raise ValueError("block_table must be [requests, max_blocks] and free_blocks [n]")
    R, width = block_table.shape
    n_free = free_blocks.shape[0]
    T = int(num_tokens)
    if T < 0:
        raise ValueError(f"num_tokens {T} < 0")
    cp = _i32(ctx, cached_lens, "cached_lens", (R,))
    np_ = _i32(ctx, new_lens, "new_lens", (R,))
    fp = _i32(ctx, free_blocks, "free_blocks", (n_free,))
    tp = _i32(ctx, block_table, "block_table", (R, width))
    buf = torch.empty(2 * (R + 1 + T), dtype=torch.int32, device=block_table.device)
    q_start, kv, taken, slots, positions = buf.split_with_sizes((R + 1, R, 1, T, T))
    at = buf.data_ptr()
    _use_stream(ctx)
    capi.check(_fn("qmoe_kv_plan")(
        ctx.handle, cp, np_, R, int(block_size), fp, n_free, int(num_blocks), tp, width, T, at,
        at + 4 * R + 4, at + 8 * R + 8, at + 8 * R + 8 + 4 * T, at + 8 * R + 4))
    return PagePlan(block_table, q_start, kv, slots, positions, taken, int(max_kv))


class KVCache:
    """Keys and values in 8 bits, in blocks of block_size tokens with one range
    per block and head (qmoe_kv_cache):

      k        int8 [num_blocks, kv_heads, k_dim / 64, block_size, 64]
      v        int8 [num_blocks, kv_heads, block_size / 16, v_dim, 16]
      k_range, v_range  f32 [num_blocks, kv_heads]; code c stands for c * range / 127
    """

    def __init__(self, num_blocks: int, block_size: int, kv_heads: int, k_dim: int, v_dim: Optional[int] = None,
                 ctx: Optional[Context] = None):
        ctx = ctx or default_context()
        v_dim = k_dim if v_dim is None else v_dim
        if k_dim % 64 or block_size % 16:
            raise ValueError(f"k_dim {k_dim} must be a multiple of 64 and block_size {block_size} of 16")
        dev = torch.device("cuda", ctx.device)
        z = lambda *s, dtype: torch.zeros(s, dtype=dtype, device=dev)  # noqa: E731
        self._set(z(num_blocks, kv_heads, k_dim // 64, block_size, 64, dtype=torch.int8),
                  z(num_blocks, kv_heads, block_size // 16, v_dim, 16, dtype=torch.int8),
                  z(num_blocks, kv_heads, dtype=torch.float32), z(num_blocks, kv_heads, dtype=torch.float32), ctx)

    @classmethod
    def from_tensors(cls, k, v, k_range, v_range, ctx: Optional[Context] = None) -> "KVCache":
        """A cache in the caller's tensors (layouts above)."""
        self = cls.__new__(cls)
        self._set(k, v, k_range, v_range, _context_of(k, ctx))
        return self

    def _set(self, k, v, k_range, v_range, ctx: Context) -> None:
        for name, t in (("k", k), ("v", v), ("k_range", k_range), ("v_range", v_range)):
            _on(ctx, name, t)
        if k.dim() != 5 or v.dim() != 5:
            raise ValueError("k and v must have 5 dimensions")
        nb, heads, chunks, bs, w = k.shape
        want = (nb, heads, bs // 16, v.shape[3], 16)
        if w != 64 or tuple(v.shape) != want or tuple(k_range.shape) != (nb, heads) or k_range.shape != v_range.shape:
            raise ValueError(f"shapes k {list(k.shape)}, v {list(v.shape)}, ranges {list(k_range.shape)}, "
                             f"{list(v_range.shape)} do not make a cache")
        if k.dtype != torch.int8 or v.dtype != torch.int8 or k_range.dtype != torch.float32 or v_range.dtype != torch.float32:
            raise TypeError("codes must be int8 and ranges float32")
        if not all(t.is_contiguous() for t in (k, v, k_range, v_range)):
            raise ValueError("a cache's tensors must be contiguous")
        self.ctx, self.k, self.v, self.k_range, self.v_range = ctx, k, v, k_range, v_range
        self.num_blocks, self.block_size, self.kv_heads = nb, bs, heads
        self.k_dim, self.v_dim = 64 * chunks, v.shape[3]
        self._c = capi.KvCacheC(k.data_ptr(), v.data_ptr(), k_range.data_ptr(), v_range.data_ptr(), nb, bs, heads,
                                self.k_dim, self.v_dim)
        self._p = ctypes.pointer(self._c)
        self._ws: dict = {}
        self._workspace(0, 0, 0, heads, 0, 0)     # checks the shape

    def _workspace(self, *key) -> int:
        """Workspace bytes of (dtype, tokens, requests, heads, max_blocks, max_kv)."""
        n = self._ws.get(key)
        if n is None:
            v = _I64()
            capi.check(_fn("qmoe_kv_attend_workspace")(self._p, *key, ctypes.byref(v)))
            if len(self._ws) >= 256:              # a server's batches come in few sizes
                self._ws.clear()
            n = self._ws[key] = v.value
        return n

    def _rows(self, x, name: str, heads: int, dim: int, dtype) -> Tuple[int, int]:
        """(pointer, token stride) of [tokens, heads, dim] whose heads are packed."""
        _on(self.ctx, name, x)
        if x.dim() != 3 or x.shape[1:] != (heads, dim):
            raise ValueError(f"{name} must be [tokens, {heads}, {dim}], got {list(x.shape)}")
        if x.dtype != dtype:
            raise TypeError(f"{name} must be {dtype}, got {x.dtype}")
        ts, hs, ds = x.stride()
        if ds != 1 or (heads > 1 and hs != dim):
            raise ValueError(f"the heads of {name} must be packed")
        if ts < heads * dim:
            if x.shape[0] > 1:
                raise ValueError(f"the tokens of {name} overlap")
            ts = heads * dim
        return x.data_ptr(), ts

    def append(self, k, v, slots) -> None:
        """Rows k [tokens, kv_heads, k_dim] and v [tokens, kv_heads, v_dim] (views
        whose heads are packed, e.g. of one projection's rows) to slots [tokens]
        (plan_pages); rows with slot -1 are skipped."""
        ctx = self.ctx
        kp, ks = self._rows(k, "k", self.kv_heads, self.k_dim, k.dtype)
        vp, vs = self._rows(v, "v", self.kv_heads, self.v_dim, k.dtype)
        T = k.shape[0]
        if v.shape[0] != T:
            raise ValueError(f"k has {T} tokens, v {v.shape[0]}")
        sp = _i32(ctx, slots, "slots", (T,))
        dt = _code(k)
        _use_stream(ctx)
        capi.check(_fn("qmoe_kv_append")(ctx.handle, self._p, kp, vp, dt, T, ks, vs, sp))

    def attend(self, q, q_start, kv_lens, block_table, scale: Optional[float] = None, max_kv: int = 0, out=None):
        """Causal attention of q [tokens, heads, k_dim] over the cache; rows
        q_start[r] .. q_start[r + 1] are the last tokens of request r, whose
        kv_lens[r] tokens are in the blocks of block_table[r].  -> [tokens, heads,
        v_dim].  Rows that see nothing are zeros; rows in front of the first request
        and past the last are left as `out` has them (zeros without one).  max_kv: the longest kv_lens
        if the host knows it (for speed alone)."""
        ctx = self.ctx
        _on(ctx, "q", q)
        if q.dim() != 3:
            raise ValueError(f"q must be [tokens, heads, {self.k_dim}], got {list(q.shape)}")
        T, heads, _ = q.shape
        qp, qs = self._rows(q, "q", heads, self.k_dim, q.dtype)
        dt = _code(q)
        _on(ctx, "block_table", block_table)
        if block_table.dim() != 2:
            raise ValueError("block_table must be [requests, max_blocks]")
        R, width = block_table.shape
        sp = _i32(ctx, q_start, "q_start", (R + 1,))
        lp = _i32(ctx, kv_lens, "kv_lens", (R,))
        tp = _i32(ctx, block_table, "block_table", (R, width))
        if out is None:
            out = torch.zeros(T, heads, self.v_dim, dtype=q.dtype, device=q.device)
        op, os_ = self._rows(out, "out", heads, self.v_dim, q.dtype)
        if out.shape[0] != T:
            raise ValueError(f"out has {out.shape[0]} tokens, q {T}")
        max_kv = int(max_kv)
        need = self._workspace(dt, T, R, heads, width, max_kv)
        ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
        _use_stream(ctx)
        capi.check(_fn("qmoe_kv_attend")(
            ctx.handle, self._p, qp, dt, T, qs, heads, sp, lp, R, tp, width, max_kv,
            self.k_dim ** -0.5 if scale is None else scale, op, os_, ws.data_ptr() if ws is not None else None, need))
        return out


def layer_norm(x, weight, bias, eps: float = 1e-6, ctx: Optional[Context] = None):
    """The block's LayerNorm (qmoe-rs src/model.rs:366-367) of x [tokens, hidden_dim]."""
    ctx = _context_of(x, ctx)
    for name, t in (("x", x), ("weight", weight), ("bias", bias)):
        _on(ctx, name, t)
    dt = _code(x)
    if x.dim() != 2 or weight.shape != (x.shape[1],) or bias.shape != weight.shape:
        raise ValueError(f"x {list(x.shape)}, weight {list(weight.shape)}, bias {list(bias.shape)}")
    if weight.dtype != torch.float32 or bias.dtype != torch.float32:
        raise TypeError("weight and bias must be float32")
    x, weight, bias = x.contiguous(), weight.contiguous(), bias.contiguous()
    out = torch.empty_like(x)
    _use_stream(ctx)
    capi.call("qmoe_layer_norm", ctx.handle, x.data_ptr(), dt, x.shape[0], x.shape[1], weight.data_ptr(),
              bias.data_ptr(), float(eps), out.data_ptr())
    return out


class AttentionBlock:
    """The attention half of a decoder layer (qmoe-rs src/model.rs:372-378,
    :394-400), with 8-bit projections and cache:

        y = LN(x);  q, k, v = qkv(y);  append k, v;  x + out(attention(q))

    qkv: Int8Tensor [heads * k_dim + kv_heads * (k_dim + v_dim), hidden], the
    rows of q, k and v one after the other; out: Int8Tensor [hidden, heads *
    v_dim]; norm: (weight, bias, eps) of the input LayerNorm.  `rotate(q, k,
    positions) -> (q, k)`, where given, applies the model's position encoding
    (torch work on the current stream) before the keys are cached."""

    def __init__(self, cache: KVCache, qkv: Int8Tensor, out: Int8Tensor, heads: int, norm,
                 scale: Optional[float] = None, rotate: Optional[Callable] = None):
        c = cache
        rows = heads * c.k_dim + c.kv_heads * (c.k_dim + c.v_dim)
        if heads % c.kv_heads:
            raise ValueError(f"heads {heads} must be a multiple of kv_heads {c.kv_heads}")
        if qkv.shape[0] != rows or out.shape != (qkv.shape[1], heads * c.v_dim):
            raise ValueError(f"qkv {list(qkv.shape)} must be [{rows}, hidden] and out {list(out.shape)} "
                             f"[hidden, {heads * c.v_dim}]")
        self.cache, self.qkv, self.out, self.heads = cache, qkv, out, heads
        self.norm, self.scale, self.rotate = norm, scale, rotate

    def forward(self, x, plan: PagePlan):
        """x [tokens, hidden] -> x + attention half; plan: plan_pages of the step."""
        c, H = self.cache, self.heads
        weight, bias, eps = self.norm
        y = self.qkv.forward(layer_norm(x, weight, bias, eps, c.ctx))
        q, k, v = y.split([H * c.k_dim, c.kv_heads * c.k_dim, c.kv_heads * c.v_dim], dim=1)
        q, k, v = q.unflatten(1, (H, c.k_dim)), k.unflatten(1, (c.kv_heads, c.k_dim)), v.unflatten(1, (c.kv_heads, c.v_dim))
        if self.rotate is not None:
            q, k = self.rotate(q, k, plan.positions)
        c.append(k, v, plan.slots)
        o = c.attend(q, plan.q_start, plan.kv_lens, plan.block_table, self.scale, plan.max_kv)
        return self.out.forward(o.flatten(1), residual=x.contiguous())
