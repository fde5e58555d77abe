"""Causal attention inside a band, with an optional learned relative position bias
(``csrc/attention_band.cu``), as autograd ops.

Tensors are ``[B, S, heads, d]`` views as in :mod:`nano_megatron_b200.ops.attention`; ``k`` and ``v``
may have fewer (grouped) heads.  Query row ``i`` stands at position ``query_start + i`` and key ``j`` at
position ``j``, so that the queries may be a shard of the sequence.  A query sees key ``j`` when

    j <= position  and  (position - j < window  or  j < sinks)

and a row that sees no key at all (a shard that lies behind the keys by a window or more) gives zeros
and passes no gradient.  With a bias the scores are

    scale * q_i . k_j + table[head, bucket(position - j)]

and the table gets its gradient too: through its ``main_grad`` buffer when it has one (the parameters of
a data-parallel wrapper), else through autograd.

bf16 CUDA tensors with a head_dim of 64, 96 or 128 go to the kernels; everything else (CPU, fp32, other
head sizes) to the plain expression at the end of this file, in fp32 or wider.  The kernels multiply whole
tiles of 128 keys, with zero weights where a key is masked: as in the plain expression, keys and values have
to be finite in masked places too.
"""
from __future__ import annotations

import functools
import math
import struct
from typing import Optional

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import native
from .functional import _deliver_grad

MAX_BUCKETS = 128        # sizes of the kernels' table of first distances
MAX_DISTANCE = 2048
_MAX_POSITION = 2 ** 30
_INT_MAX = 2 ** 31 - 1

# BandArgs of csrc/attention_band.cu in two parts.  What changes from call to call: fourteen pointers, three flags.  What the
# shapes fix: three strides of eight tensors, ten whole numbers, the scale, the table of first distances.
_POINTERS = struct.Struct("14P4i")
_FIXED = struct.Struct("24q10ifi" + f"{2 * MAX_BUCKETS}s")


@functools.lru_cache(maxsize=None)
def relative_bucket_limits(num_buckets: int, max_distance: int) -> tuple[int, ...]:
    """First distance of every bucket but bucket 0.

    The lower half of the buckets holds one distance each; the others grow by a constant factor, such that the
    logarithm of the distance is divided evenly up to ``max_distance``, and the last one is open.  Bucket
    ``e + t`` (``e`` exact ones, ``g`` others) starts at the first ``n`` with ``(n / e)^g >= (max_distance / e)^t``,
    which is decided in whole numbers: a rounded logarithm puts distances on borders into the wrong bucket.
    """
    exact = num_buckets // 2
    grow = num_buckets - exact
    limits, n = list(range(1, exact + 1)), exact
    for t in range(1, grow):
        while n ** grow * exact ** t < max_distance ** t * exact ** grow:
            n += 1
        limits.append(n)
    return tuple(limits)


def relative_position_buckets(distance: Tensor, num_buckets: int, max_distance: int = 128) -> Tensor:
    """Bucket of every (non-negative) distance between a query and a key behind it."""
    _check_int("num_buckets", num_buckets, 2)
    _check_int("max_distance", max_distance, 1)
    _check_buckets(num_buckets, max_distance)
    limits = torch.tensor(relative_bucket_limits(num_buckets, max_distance), device=distance.device)
    return torch.bucketize(distance, limits, right=True)


def band_attention_supported(t: Tensor) -> bool:
    """True where the kernels run: bf16 on a GPU with a head_dim that they have."""
    return t.is_cuda and t.dtype == torch.bfloat16 and t.shape[-1] in (64, 96, 128)


# ---------------------------------------------------------------- launches --
class _Plan:
    """What follows from the shapes, strides and numbers of a call alone; worked out once for each of them."""

    __slots__ = ("q_ok", "k_ok", "v_ok", "fwd", "bwd", "bwd_packed", "width", "scratch", "stats")


def _loadable(shape, stride) -> bool:
    """Tile loads need contiguous rows and strides that are multiples of 16 bytes."""
    return stride[3] == 1 and all(n == 1 or (s > 0 and s % 8 == 0) for n, s in zip(shape[:3], stride[:3]))


def _dense(shape) -> tuple[int, ...]:
    return (shape[1] * shape[2] * shape[3], shape[2] * shape[3], shape[3], 1)


def _fixed(q, k, strides, scale, window, sinks, start, limits) -> bytes:
    flat = []
    for (shape, stride) in strides:
        # the stride of a dimension of one may be anything: give the tile loads one that is valid
        flat += [0, 0, 0] if shape is None else [s if n > 1 else shape[3] for n, s in zip(shape[:3], stride[:3])]
    return _FIXED.pack(*flat, q[0], q[2], k[2], q[1], k[1], q[3], start, min(window, _MAX_POSITION), min(sinks, k[1]),
                       len(limits) // 2 + 1 if limits else 0, scale, 0, limits)


@functools.lru_cache(maxsize=4096)
def _plan(q, q_stride, k, k_stride, v, v_stride, floating, buckets, max_distance, scale, window, sinks, start) -> _Plan:
    _check_shapes(q, k, v, floating, scale, start)
    limits = b""
    if buckets is not None:
        _check_buckets(buckets, max_distance)
        limits = struct.pack(f"{buckets - 1}H", *relative_bucket_limits(buckets, max_distance))
    p = _Plan()
    p.q_ok, p.k_ok, p.v_ok = _loadable(q, q_stride), _loadable(k, k_stride), _loadable(v, v_stride)
    p.stats, p.scratch = (2, q[0], q[2], q[1]), None
    inputs = [(s, st if ok else _dense(s)) for s, st, ok in ((q, q_stride, p.q_ok), (k, k_stride, p.k_ok), (v, v_stride, p.v_ok))]
    out, none = (q, _dense(q)), (None, None)
    numbers = (scale, window, sinks, start, limits)
    p.fwd = _fixed(q, k, inputs + [out] + [none] * 4, *numbers)
    p.bwd = _fixed(q, k, inputs + [out, out, out, (k, _dense(k)), (k, _dense(k))], *numbers)
    # the slices of one packed projection: their gradients go to the slices of one buffer and are joined without a copy
    p.width = q[2] + 2 * k[2]
    row = p.width * q[3]
    packed = (q[1] * row, row, q[3], 1)
    p.bwd_packed = None
    if q[1] == k[1] and q_stride == k_stride == v_stride == packed:
        p.bwd_packed = _fixed(q, k, inputs + [out, out, (q, packed), (k, packed), (k, packed)], *numbers)
    return p


def _scratch(p: _Plan, lib) -> int:
    if p.scratch is None:
        p.scratch = lib.nmb_band_bwd_scratch(_POINTERS.pack(*[0] * 18) + p.bwd)
    return p.scratch


def _readable(t: Tensor, ok: bool) -> Tensor:
    """``t``, or a copy where the kernels cannot address it: dense, or (an unaligned start) with the same strides."""
    if not ok:
        return t.clone(memory_format=torch.contiguous_format)
    if t.data_ptr() % 16 != 0:
        return torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=t.device).copy_(t)
    return t


def _band_fwd(p: _Plan, q, k, v, table):
    lib = native.lib()
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    stats = torch.empty(p.stats, dtype=torch.float32, device=q.device)
    m = stats.data_ptr()
    args = _POINTERS.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), 0, 0, 0, 0, m, m + 2 * stats.numel(), 0,
                          0 if table is None else table.data_ptr(), 0, native.status_word(q.device).data_ptr(),
                          table is not None and table.dtype == torch.float32, 0, 0, 0) + p.fwd
    native.check_rc(lib.nmb_band_fwd(args, torch.cuda.current_stream(q.device.index).cuda_stream), "nmb_band_fwd")
    return out, stats


def _band_bwd(p: _Plan, q, k, v, table, out, stats, dout, dtable=None, accumulate=False):
    lib = native.lib()
    dout = _readable(dout, dout.is_contiguous())
    q_at, k_at, v_at = q.data_ptr(), k.data_ptr(), v.data_ptr()
    h, g, d = q.shape[2], k.shape[2], q.shape[3]
    if p.bwd_packed is not None and k_at == q_at + 2 * h * d and v_at == k_at + 2 * g * d:
        fixed = p.bwd_packed
        packed = torch.empty((q.shape[0], q.shape[1], p.width, d), dtype=q.dtype, device=q.device)
        dq, dk, dv = packed.split((h, g, g), dim=2)
    else:
        fixed = p.bwd
        dq, dk, dv = (torch.empty(t.shape, dtype=q.dtype, device=q.device) for t in (q, k, v))
    scratch = torch.empty(_scratch(p, lib), dtype=torch.float32, device=q.device)
    m = stats.data_ptr()
    args = _POINTERS.pack(q_at, k_at, v_at, out.data_ptr(), dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), m,
                          m + 2 * stats.numel(), scratch.data_ptr(), 0 if table is None else table.data_ptr(),
                          0 if dtable is None else dtable.data_ptr(), native.status_word(q.device).data_ptr(),
                          table is not None and table.dtype == torch.float32,
                          dtable is not None and dtable.dtype == torch.float32, accumulate, 0) + fixed
    native.check_rc(lib.nmb_band_bwd(args, torch.cuda.current_stream(q.device.index).cuda_stream), "nmb_band_bwd")
    if dtable is not None:
        native.launches += 1
    return dq, dk, dv


def _on_its_device(t: Tensor, fn, *args):
    if t.device.index == torch.cuda.current_device():
        return fn(*args)
    with torch.cuda.device(t.device):
        return fn(*args)


class _BandAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, p):
        ctx.table_param, ctx.plan = table, p
        q, k, v = _readable(q, p.q_ok), _readable(k, p.k_ok), _readable(v, p.v_ok)
        if table is not None:
            table = table.contiguous()
        out, stats = _on_its_device(q, _band_fwd, p, q, k, v, table)
        ctx.save_for_backward(q, k, v, table, out, stats)
        return out

    @staticmethod
    def backward(ctx, dout):
        # only a backward pass that builds a graph itself needs the guard against a second differentiation
        return (_guarded_gradients if torch.is_grad_enabled() else _gradients)(ctx, dout)


def _gradients(ctx, dout):
    q, k, v, table, out, stats = ctx.saved_tensors
    if table is None or not ctx.needs_input_grad[3]:
        return (*_on_its_device(q, _band_bwd, ctx.plan, q, k, v, table, out, stats, dout), None, None)
    grads = []

    def compute(buffer, accumulate):
        # the kernels write dense tables of two types; any other buffer gets the gradient from one of those
        direct = buffer is not None and buffer.is_contiguous() and buffer.dtype in (torch.bfloat16, torch.float32)
        target = buffer if direct else torch.empty_like(table)
        grads.extend(_on_its_device(q, _band_bwd, ctx.plan, q, k, v, table, out, stats, dout, target, accumulate and direct))
        if buffer is not None and not direct:
            buffer.add_(target) if accumulate else buffer.copy_(target)
        return target

    dtable = _deliver_grad(ctx.table_param, compute)
    return (*grads, dtable, None)


_guarded_gradients = once_differentiable(_gradients)


# ------------------------------------------------------------------ checks --
def _check_int(name: str, value, low: int) -> int:
    if isinstance(value, bool) or not isinstance(value, int):
        raise TypeError(f"{name} must be an int, got {type(value).__name__}")
    if not low <= value <= _INT_MAX:
        raise ValueError(f"{name} must be at least {low}, got {value}")
    return value


def _check_buckets(num_buckets: int, max_distance: int) -> None:
    if not 2 <= num_buckets <= MAX_BUCKETS:
        raise ValueError(f"the table must have 2 to {MAX_BUCKETS} buckets, got {num_buckets}")
    if not num_buckets // 2 < max_distance <= MAX_DISTANCE:
        raise ValueError(f"max_distance must be above num_buckets // 2 ({num_buckets // 2}) and at most {MAX_DISTANCE}, "
                         f"got {max_distance}")


def _check_shapes(q, k, v, floating, scale, start) -> None:
    if len(q) != 4 or len(k) != 4 or len(v) != 4:
        raise ValueError(f"q, k, v must be 4D [B,S,H,D]; got q={tuple(q)}, k={tuple(k)}, v={tuple(v)}")
    if k != v:
        raise ValueError(f"k and v must share shape; got k={tuple(k)}, v={tuple(v)}")
    if q[0] != k[0] or q[3] != k[3]:
        raise ValueError(f"q/k batch and head_dim must match; got q={tuple(q)}, k={tuple(k)}")
    if k[2] == 0 or q[2] % k[2] != 0:
        raise ValueError(f"query heads must be a multiple of key heads; got q={tuple(q)}, k={tuple(k)}")
    if not floating:
        raise ValueError("q, k, v must be floating-point tensors")
    if not (math.isfinite(scale) and scale > 0.0):
        raise ValueError(f"scale must be finite and positive, got {scale}")
    if start + q[1] > _MAX_POSITION or k[1] > _MAX_POSITION:
        raise ValueError(f"positions must stay below {_MAX_POSITION}; got query_start {start}, q={tuple(q)}, k={tuple(k)}")


def _attend(q, k, v, table, max_distance, scale, window, sinks, start) -> Tensor:
    if not q.dtype == k.dtype == v.dtype:
        raise ValueError(f"q, k, v must share a floating type; got {q.dtype}, {k.dtype}, {v.dtype}")
    if not q.device == k.device == v.device:
        raise ValueError(f"q, k, v must be on one device; got {q.device}, {k.device}, {v.device}")
    window = _INT_MAX if window is None else _check_int("window", window, 1)
    sinks = _check_int("sinks", sinks, 0)
    start = _check_int("query_start", start, 0)
    scale = float(scale)
    buckets = None
    if table is not None:
        if table.dim() != 2 or q.dim() != 4 or table.shape[0] != q.shape[2]:
            raise ValueError(f"table must be [query heads, buckets]; got {tuple(table.shape)} with q={tuple(q.shape)}")
        if table.device != q.device:
            raise ValueError(f"table must be on {q.device}, got {table.device}")
        buckets = table.shape[1]
        _check_int("max_distance", max_distance, 1)
    p = _plan(q.shape, q.stride(), k.shape, k.stride(), v.shape, v.stride(), q.is_floating_point(), buckets, max_distance, scale,
              window, sinks, start)
    if band_attention_supported(q) and q.numel() and k.numel():
        if table is not None and table.dtype not in (torch.bfloat16, torch.float32):
            raise ValueError(f"table must be bfloat16 or float32, got {table.dtype}")
        return _BandAttention.apply(q, k, v, table, p)
    return _expression(q, k, v, table, max_distance, scale, window, sinks, start)


# ------------------------------------------------------------ entry points --
def window_attention(q: Tensor, k: Tensor, v: Tensor, scale: float, *, window: int, sinks: int = 0,
                     query_start: int = 0) -> Tensor:
    """Causal attention in which a query sees the last ``window`` positions, its own included, and the first ``sinks`` keys
    of the sequence.  ``[B, Sq, Hq, d]``, ``[B, Skv, Hkv, d]`` -> ``[B, Sq, Hq, d]``."""
    if window is None:
        raise TypeError("window must be an int")
    return _attend(q, k, v, None, 0, scale, window, sinks, query_start)


def relative_bias_attention(q: Tensor, k: Tensor, v: Tensor, table: Tensor, scale: float, *, max_distance: int = 128,
                            window: Optional[int] = None, sinks: int = 0, query_start: int = 0) -> Tensor:
    """Causal attention with the bias ``table[head, bucket(distance)]`` on the scores (``table`` is ``[Hq, buckets]``, bf16 or
    fp32; :func:`relative_bucket_limits` gives the buckets), inside a window as in :func:`window_attention` where one is
    given.  Entries of ``-inf`` mask their bucket."""
    if table is None:
        raise TypeError("table must be a tensor")
    return _attend(q, k, v, table, max_distance, scale, window, sinks, query_start)


def _expression(q, k, v, table, max_distance, scale, window, sinks, start) -> Tensor:
    wide = torch.promote_types(q.dtype, torch.float32)
    group = q.shape[2] // k.shape[2]
    qh, kh, vh = (t.transpose(1, 2).to(wide) for t in (q, k, v))
    if group > 1:
        kh, vh = kh.repeat_interleave(group, dim=1), vh.repeat_interleave(group, dim=1)
    key = torch.arange(k.shape[1], device=q.device)
    distance = torch.arange(start, start + q.shape[1], device=q.device)[:, None] - key
    hidden = (distance < 0) | ((distance >= window) & (key >= sinks))
    scores = torch.matmul(qh, kh.transpose(-2, -1)) * scale
    if table is not None:
        scores = scores + table.to(wide)[:, relative_position_buckets(distance.clamp(min=0), table.shape[1], max_distance)]
    scores = scores.masked_fill(hidden, float("-inf"))
    if k.shape[1] == 0:
        return torch.matmul(scores, vh).transpose(1, 2).to(q.dtype)
    top = scores.detach().amax(dim=-1, keepdim=True).clamp(min=torch.finfo(wide).min)
    weights = torch.exp(scores - top)
    total = weights.sum(dim=-1, keepdim=True)
    probs = weights / torch.where(total == 0, torch.ones_like(total), total)
    return torch.matmul(probs, vh).transpose(1, 2).to(q.dtype)
