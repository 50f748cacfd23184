"""The operators between the linears of a decoder layer.

The reference leaves them to its host framework; a decoder layer on this
library's linears (:class:`AWQQKVLinear`, :class:`AWQGateUpSiluMul`, ...) is
made whole by

* :func:`rms_norm` / :func:`rms_norm_fp8`: the residual's addition and the
  RMS norm in one pass, with the output in F or in 8 bits with row scales;
* :func:`rope_append`: the rotary embedding of q and k and the append of k
  and v to a paged cache, in one launch;
* :func:`attention_decode`: attention of one new token per sequence over the
  cache, split over its length;
* :func:`attention_prefill`: attention of prompts, or chunks of prompts, over
  the cache that already holds them; both causal, with an optional sliding
  window whose first tokens (sinks) stay visible.

The cache is a pair of tensors ``k_cache``, ``v_cache`` [pages, n_kv,
page_size, head_dim] (any strides that are multiples of 8 elements with a unit
innermost one, the same for both, so one may be a view into a larger pool or
hold its tokens outermost in a page; but prompts are attended at full speed
only where the page stride is a multiple of the head stride: heads outermost,
or pages padded by part of a head, take 4 to 20 times as long), with ``block_table`` int32 [batch,
table_width] (token j of sequence b is slot j % page_size of page
``block_table[b, j // page_size]``) and ``seq_lens`` int32 [batch], the tokens
of each sequence with the call's own. Several new tokens per sequence come
with ``q_start`` int32 [batch + 1]: rows ``q_start[b]:q_start[b + 1]`` are the
last tokens of sequence b. These three live on the GPU and are not read by the
host: pages and positions outside the cache are skipped by the kernels and
reported by :func:`device_error` (bit 2). The [tokens, heads, head_dim] operands
start on 16 bytes and have token strides that are multiples of 8 elements.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _lib
from .errors import CubeAwqError, DTypeError, ShapeError, check
from .kernel import _require_cuda, _torch_ext, cawq_dtype, stream_handle

# Each operator first calls its compiled host path (csrc/cawq_torch.cpp), which
# does the checks, the allocation and the C call in C++; it gives None for
# arguments that do not fit (and an int where the C call failed), and the
# functions here then say what is wrong. At decode sizes the host's work is of
# the order of the kernels' own time.

_SHAPE = _lib.CAWQ_ERR_INVALID_SHAPE
_HALVES = (torch.float16, torch.bfloat16)


def _same_device(*tensors: Optional[torch.Tensor]) -> None:
    _require_cuda(*tensors)
    if len({t.device for t in tensors if t is not None}) > 1:
        raise CubeAwqError("all tensors of a call must be on one device",
                           _lib.CAWQ_ERR_INVALID_ARGUMENT)


def _rows(name: str, t: torch.Tensor, shape, dtype: torch.dtype) -> None:
    """A [rows, d] operand: its shape and type, unit column stride, and rows that
    do not overlap (a broadcast one's stride of 0 means "dense" to the C calls)."""
    if t.dtype != dtype:
        raise DTypeError(f"{name} must be {dtype}, got {t.dtype}", _lib.CAWQ_ERR_DTYPE)
    if tuple(t.shape) != tuple(shape) or (t.numel() > 0 and t.shape[1] > 1 and t.stride(1) != 1):
        raise ShapeError(f"{name} must be {list(shape)} with unit column stride", _SHAPE)
    if t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise ShapeError(f"{name}: row stride {t.stride(0)} is below its {t.shape[1]} columns "
                         "(a broadcast operand has to be made contiguous)", _SHAPE)


def _norm(x, weight, eps, residual, out, out_dtype, residual_out, scales):
    _same_device(x, weight, residual, out, residual_out, scales)
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ShapeError("x must be [..., d] with d > 0", _SHAPE)
    code = cawq_dtype(x.dtype)
    d = x.shape[-1]
    if tuple(weight.shape) != (d,) or not weight.is_contiguous():
        raise ShapeError(f"weight must be a contiguous [{d}] tensor", _SHAPE)
    if weight.dtype != x.dtype:
        raise DTypeError("weight must have x's dtype", _lib.CAWQ_ERR_DTYPE)
    lead = x.shape[:-1]

    def flat(name, t, dtype):
        if t.shape != x.shape:
            raise ShapeError(f"{name} must have x's shape", _SHAPE)
        t2 = t.view(-1, d) if t.is_contiguous() else t
        if t2.dim() != 2:
            raise ShapeError(f"{name} must be contiguous, or 2-D with unit column stride", _SHAPE)
        _rows(name, t2, t2.shape, dtype)
        return t2

    x2 = flat("x", x if x.dim() == 2 else x.contiguous(), x.dtype)
    rows = x2.shape[0]
    r2 = None if residual is None else flat("residual", residual, x.dtype)
    if out is None:
        out = torch.empty(x.shape, dtype=out_dtype, device=x.device)
    o2 = flat("out", out, out_dtype)
    h2 = None
    if residual is None:
        if residual_out is not None:
            raise CubeAwqError("residual_out needs a residual", _lib.CAWQ_ERR_INVALID_ARGUMENT)
    else:
        if residual_out is None:
            residual_out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        h2 = flat("residual_out", residual_out, x.dtype)
    ld = lambda t: t.stride(0) if t is not None and rows > 1 else d  # noqa: E731
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    lib = _lib.lib()
    with torch.cuda.device(x.device):
        if out_dtype == torch.float8_e4m3fn:
            if scales is None:
                scales = torch.empty(lead, dtype=torch.float32, device=x.device)
            elif scales.shape != lead or scales.dtype != torch.float32 or not scales.is_contiguous():
                raise ShapeError(f"scales must be a contiguous float32 {list(lead)} tensor", _SHAPE)
            check(lib.cawq_rms_norm_fp8(ptr(x2), ptr(weight), ptr(r2), ptr(o2), ptr(scales),
                                        ptr(h2), rows, d, ld(x2), ld(r2), ld(o2), ld(h2), eps,
                                        code, stream_handle(x)))
            return out, scales, residual_out
        check(lib.cawq_rms_norm(ptr(x2), ptr(weight), ptr(r2), ptr(o2), ptr(h2), rows, d, ld(x2),
                                ld(r2), ld(o2), ld(h2), eps, code, stream_handle(x)))
    return out, residual_out


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
             residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
             residual_out: Optional[torch.Tensor] = None
             ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """RMS norm with the residual's addition (cawq_rms_norm) -> (y, h):
    h = x + residual, y = h / sqrt(mean(h^2) + eps) * weight over the last
    dimension, computed in fp32 and rounded once each. Without a residual h is
    None (it would be x). x, residual [..., d] f32, f16 or bf16, contiguous or
    2-D with a unit column stride and a row stride of at least d (a broadcast
    operand is refused). ``out`` may be x, ``residual_out`` may be ``residual``
    (the residual stream updated in place)."""
    ext = _torch_ext()
    if ext is not None:
        r = ext.rms_norm(x, weight, eps, residual, out, residual_out)
        if r.__class__ is tuple:
            return r
        if r is not None:
            check(r)
    return _norm(x, weight, eps, residual, out, x.dtype, residual_out, None)


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
                 residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                 scales: Optional[torch.Tensor] = None,
                 residual_out: Optional[torch.Tensor] = None
                 ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """:func:`rms_norm` with y in 8 bits (cawq_rms_norm_fp8) -> (y8, scales, h):
    scales[...] = max |y| / 448 of a row (fp32), y8 = float8_e4m3fn(y / scale),
    the operands of an 8-bit product with row scales (of a module that AutoAWQ
    left unquantised, such as lm_head; this package has no such product)."""
    ext = _torch_ext()
    if ext is not None:
        r = ext.rms_norm_fp8(x, weight, eps, residual, out, scales, residual_out)
        if r.__class__ is tuple:
            return r
        if r is not None:
            check(r)
    return _norm(x, weight, eps, residual, out, torch.float8_e4m3fn, residual_out, scales)


def rope_table(positions: int, head_dim: int, base: float = 10000.0, device="cuda") -> torch.Tensor:
    """The fp32 [positions, head_dim] table of :func:`rope_append`: the cosines
    of position p's angles p * base^(-2 i / head_dim) in the first half of row
    p, their sines in the second. Made in fp64; a model with scaled frequencies
    fills a table of its own in the same layout."""
    inv = float(base) ** (-torch.arange(0, head_dim, 2, dtype=torch.float64, device=device)
                          / head_dim)
    a = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * inv
    return torch.cat([a.cos(), a.sin()], dim=1).float()


def _paged(k_cache, v_cache, block_table, seq_lens, q_start, dtype) -> _lib.PagedKVC:
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
        raise ShapeError("k_cache and v_cache must be [pages, n_kv, page_size, head_dim]", _SHAPE)
    if k_cache.dtype != dtype or v_cache.dtype != dtype:
        raise DTypeError(f"k_cache and v_cache must be {dtype}", _lib.CAWQ_ERR_DTYPE)
    if k_cache.numel() > 0 and (k_cache.stride(3) != 1 or v_cache.stride() != k_cache.stride()):
        raise ShapeError("k_cache and v_cache must have the same strides, the innermost 1", _SHAPE)
    for name, t in (("block_table", block_table), ("seq_lens", seq_lens), ("q_start", q_start)):
        if t is not None and t.dtype != torch.int32:
            raise DTypeError(f"{name} must be int32", _lib.CAWQ_ERR_DTYPE)
    batch = seq_lens.numel()
    if seq_lens.dim() != 1 or not seq_lens.is_contiguous():
        raise ShapeError("seq_lens must be a contiguous [batch] tensor", _SHAPE)
    if block_table.dim() != 2 or block_table.shape[0] != batch or \
            (block_table.shape[1] > 1 and block_table.stride(1) != 1):
        raise ShapeError("block_table must be [batch, table_width] with unit column stride", _SHAPE)
    if q_start is not None and (tuple(q_start.shape) != (batch + 1,) or not q_start.is_contiguous()):
        raise ShapeError("q_start must be a contiguous [batch + 1] tensor", _SHAPE)
    kv = _lib.PagedKVC()
    kv.k, kv.v = k_cache.data_ptr(), v_cache.data_ptr()
    kv.pages, kv.n_kv, kv.page_size, kv.head_dim = k_cache.shape
    kv.stride_page, kv.stride_head, kv.stride_token = k_cache.stride()[:3]
    kv.block_table, kv.seq_lens = block_table.data_ptr(), seq_lens.data_ptr()
    kv.batch, kv.table_width = block_table.shape
    kv.ld_table = block_table.stride(0) if batch > 1 else kv.table_width
    kv.q_start = q_start.data_ptr() if q_start is not None else None
    return kv


def _heads(name: str, t: torch.Tensor, heads: Optional[int], d: int, dtype: torch.dtype,
           tokens: Optional[int] = None) -> int:
    """Token stride of a [tokens, heads, head_dim] operand with dense heads and
    tokens that do not overlap (0 means "dense" to the C calls)."""
    if t.dtype != dtype:
        raise DTypeError(f"{name} must be {dtype}, got {t.dtype}", _lib.CAWQ_ERR_DTYPE)
    if t.dim() != 3 or t.shape[2] != d or (heads is not None and t.shape[1] != heads) or \
            (tokens is not None and t.shape[0] != tokens):
        want = [tokens if tokens is not None else "tokens", heads if heads is not None else "heads", d]
        raise ShapeError(f"{name} must be {want}, got {list(t.shape)}", _SHAPE)
    if t.numel() > 0 and (t.stride(2) != 1 or (t.shape[1] > 1 and t.stride(1) != d)):
        raise ShapeError(f"{name} must hold its heads dense (strides [ld, {d}, 1])", _SHAPE)
    if t.shape[0] > 1 and t.stride(0) < t.shape[1] * d:
        raise ShapeError(f"{name}: token stride {t.stride(0)} is below its {t.shape[1]} x {d} elements "
                         "(a broadcast operand has to be made contiguous)", _SHAPE)
    return t.stride(0) if t.shape[0] > 1 else t.shape[1] * d


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, rope: torch.Tensor,
                k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                seq_lens: torch.Tensor, q_start: Optional[torch.Tensor] = None,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotary embedding of the new tokens' q and k, and the append of k and v
    to the cache (cawq_rope_append); returns the turned q.

    q [tokens, n_q, head_dim], k and v [tokens, n_kv, head_dim] f16 or bf16,
    heads dense, any token stride of at least the heads' width (views of a fused
    projection's output will do, a broadcast operand is refused); rope fp32 [positions, head_dim] (:func:`rope_table`). Element i of a
    head turns with element i + head_dim / 2. ``out`` may be q itself. Without
    ``q_start`` there is one new token per sequence. A token of an empty slot
    (negative position), or of no sequence (before ``q_start[0]`` or from
    ``q_start[batch]`` on), gets a zero q and is not stored."""
    ext = _torch_ext()
    if ext is not None:
        r = ext.rope_append(q, k, v, rope, k_cache, v_cache, block_table, seq_lens, q_start, out)
        if r.__class__ is torch.Tensor:
            return r
        if r is not None:
            check(r)
    _same_device(q, k, v, rope, k_cache, v_cache, block_table, seq_lens, q_start, out)
    if q.dtype not in _HALVES:
        raise DTypeError("the rotary append takes f16 or bf16", _lib.CAWQ_ERR_DTYPE)
    kv = _paged(k_cache, v_cache, block_table, seq_lens, q_start, q.dtype)
    d, tokens = kv.head_dim, q.shape[0]
    ld_q = _heads("q", q, None, d, q.dtype)
    ld_k = _heads("k", k, kv.n_kv, d, q.dtype, tokens)
    ld_v = _heads("v", v, kv.n_kv, d, q.dtype, tokens)
    if rope.dtype != torch.float32 or rope.dim() != 2 or rope.shape[1] != d or \
            not rope.is_contiguous():
        raise ShapeError(f"rope must be a contiguous float32 [positions, {d}] table", _SHAPE)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    ld_o = _heads("out", out, q.shape[1], d, q.dtype, tokens)
    with torch.cuda.device(q.device):
        check(_lib.lib().cawq_rope_append(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), rope.data_ptr(), rope.shape[0],
            out.data_ptr(), ctypes.byref(kv), tokens, q.shape[1], ld_q, ld_k, ld_v, ld_o,
            cawq_dtype(q.dtype), stream_handle(q)))
    return out


def _attention(q, k_cache, v_cache, block_table, seq_lens, q_start, scale, window, sinks, out):
    ext = _torch_ext()
    if ext is not None:
        r = ext.attention(q, k_cache, v_cache, block_table, seq_lens, q_start, scale, window, sinks,
                          out)
        if r.__class__ is torch.Tensor:
            return r
        if r is not None:
            check(r)
    _same_device(q, k_cache, v_cache, block_table, seq_lens, q_start, out)
    if q.dtype not in _HALVES:
        raise DTypeError("attention takes f16 or bf16", _lib.CAWQ_ERR_DTYPE)
    window, sinks = int(window or 0), int(sinks)
    if window < 0 or sinks < 0:
        raise CubeAwqError("window and sinks must be >= 0", _lib.CAWQ_ERR_INVALID_ARGUMENT)
    kv = _paged(k_cache, v_cache, block_table, seq_lens, q_start, q.dtype)
    d = kv.head_dim
    ld_q = _heads("q", q, None, d, q.dtype)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    tokens, n_q = q.shape[:2]
    ld_o = _heads("out", out, n_q, d, q.dtype, tokens)
    if q_start is None and tokens != kv.batch:
        raise ShapeError("attention_decode takes one new token per sequence", _SHAPE)
    lib = _lib.lib()
    with torch.cuda.device(q.device):
        need = lib.cawq_attention_workspace(ctypes.byref(kv), tokens, n_q)
        # from torch's allocator on the current stream, so it is this call's alone
        ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
        args = (n_q, ld_q, ld_o, float(scale if scale is not None else d ** -0.5), window, sinks,
                cawq_dtype(q.dtype), ws.data_ptr() if need else None, need, stream_handle(q))
        if q_start is None:
            check(lib.cawq_attention_decode(q.data_ptr(), out.data_ptr(), ctypes.byref(kv), *args))
        else:
            check(lib.cawq_attention_prefill(q.data_ptr(), out.data_ptr(), ctypes.byref(kv),
                                             tokens, *args))
    return out


def attention_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                     block_table: torch.Tensor, seq_lens: torch.Tensor,
                     scale: Optional[float] = None, window: Optional[int] = None, sinks: int = 0,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one new token per sequence over the paged cache that holds
    it already (cawq_attention_decode): q [batch, n_q, head_dim] -> the same
    shape. Query head h reads key / value head h // (n_q / n_kv). ``scale``
    defaults to head_dim^-0.5. With a ``window`` the token at position p sees
    positions > p - window and the first ``sinks`` ones; without (None or 0) it
    sees all. A sequence of length 0 gets zeros. f16 / bf16."""
    return _attention(q, k_cache, v_cache, block_table, seq_lens, None, scale, window, sinks, out)


def attention_prefill(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                      block_table: torch.Tensor, seq_lens: torch.Tensor, q_start: torch.Tensor,
                      scale: Optional[float] = None, window: Optional[int] = None, sinks: int = 0,
                      out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of the new tokens of ragged sequences over the paged
    cache that holds them already (cawq_attention_prefill): q [tokens, n_q,
    head_dim] -> the same shape. Rows q_start[b] .. q_start[b + 1] - 1 are the
    last tokens of sequence b; rows of no sequence are left as they are.
    ``scale``, ``window`` and ``sinks`` as in :func:`attention_decode`. Pages
    that no new token sees and slots past a sequence's length may hold
    anything; its other values must be finite."""
    if q_start is None:
        raise ShapeError("attention_prefill needs q_start", _SHAPE)
    return _attention(q, k_cache, v_cache, block_table, seq_lens, q_start, scale, window, sinks,
                      out)
