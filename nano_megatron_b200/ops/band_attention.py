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

MAX_BUCKETS = 128        # sizes of the kernels' table of first distances
MAX_DISTANCE = 2048
_MAX_POSITION = 2 ** 30
_INT_MAX = 2 ** 31 - 1

# BandArgs of csrc/attention_band.cu: eight tensors (pointer and three strides), six pointers, thirteen whole
# numbers, the scale, the table of first distances.
_ARGS = struct.Struct("P3q" * 8 + "6P" + "13if" + f"{2 * MAX_BUCKETS}s")
_ABSENT = (0, 0, 0, 0)


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
    _check_buckets(num_buckets, max_distance)
    limits = torch.tensor(relative_bucket_limits(num_buckets, max_distance), device=distance.device)
    return torch.bucketize(distance, limits, right=True)


@functools.lru_cache(maxsize=None)
def _packed_limits(num_buckets: int, max_distance: int) -> bytes:
    limits = relative_bucket_limits(num_buckets, max_distance)
    return struct.pack(f"{len(limits)}H", *limits)


def band_attention_supported(t: Tensor) -> bool:
    """True where the kernels run: bf16 on a GPU with a head_dim that they have."""
    return t.is_cuda and t.dtype == torch.bfloat16 and t.shape[-1] in (64, 96, 128)


# ---------------------------------------------------------------- launches --
def _readable(t: Tensor) -> Tensor:
    """``t``, or a contiguous copy where the kernels cannot address it: tile loads need 16-byte rows and strides."""
    if t.stride(3) == 1 and t.data_ptr() % 16 == 0:
        if all(n == 1 or (s > 0 and s % 8 == 0) for n, s in zip(t.shape[:3], t.stride()[:3])):
            return t
    return t.contiguous() if t.stride(3) != 1 or not t.is_contiguous() else t.clone()


def _desc(t: Tensor) -> tuple[int, int, int, int]:
    # the stride of a dimension of one may be anything: give the tile loads one that is valid
    d = t.shape[3]
    sb, ss, sh = (s if n > 1 else d for n, s in zip(t.shape[:3], t.stride()[:3]))
    return t.data_ptr(), sb, ss, sh


def _ptr(t: Optional[Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _pack(q, k, v, table, limits, scale, window, sinks, start, *, o, dout=None, dq=None, dk=None, dv=None, m=None, l=None,
          scratch=None, dtable=None, accumulate=False) -> bytes:
    b, sq, hq, d = q.shape
    skv, hkv = k.shape[1], k.shape[2]
    tensors = []
    for t in (q, k, v, o, dout, dq, dk, dv):
        tensors += _ABSENT if t is None else _desc(t)
    buckets = 0 if table is None else table.shape[1]
    return _ARGS.pack(*tensors, _ptr(m), _ptr(l), _ptr(scratch), _ptr(table), _ptr(dtable),
                      native.status_word(q.device).data_ptr(), int(table is not None and table.dtype == torch.float32),
                      int(dtable is not None and dtable.dtype == torch.float32), int(accumulate), b, hq, hkv, sq, skv, d,
                      start, min(window, _MAX_POSITION), min(sinks, skv), buckets, scale, limits)


def _band_fwd(q, k, v, table, limits, scale, window, sinks, start):
    b, sq, hq, d = q.shape
    out = torch.empty((b, sq, hq, d), dtype=q.dtype, device=q.device)
    stats = torch.empty((2, b, hq, sq), dtype=torch.float32, device=q.device)
    args = _pack(q, k, v, table, limits, scale, window, sinks, start, o=out, m=stats[0], l=stats[1])
    native.check_rc(native.lib().nmb_band_fwd(args, native.stream_ptr(q.device)), "nmb_band_fwd")
    return out, stats


def _grad_buffers(q, k, v):
    """Buffers of the three gradients: the slices of one packed buffer where ``q``, ``k`` and ``v`` are the slices of one
    packed projection (their gradients are joined without a copy then), else three tensors."""
    b, s, hq, d = q.shape
    hkv = k.shape[2]
    width = (hq + 2 * hkv) * d
    strides = (s * width, width, d, 1)
    if q.stride() == k.stride() == v.stride() == strides and k.data_ptr() == q.data_ptr() + 2 * hq * d and \
            v.data_ptr() == k.data_ptr() + 2 * hkv * d:
        packed = torch.empty((b, s, hq + 2 * hkv, d), dtype=q.dtype, device=q.device)
        return packed[:, :, :hq], packed[:, :, hq:hq + hkv], packed[:, :, hq + hkv:]
    return tuple(torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))


def _band_bwd(q, k, v, table, limits, scale, window, sinks, start, out, stats, dout, dtable=None, accumulate=False):
    dq, dk, dv = _grad_buffers(q, k, v)
    lib = native.lib()
    common = dict(o=out, dout=_readable(dout), dq=dq, dk=dk, dv=dv, m=stats[0], l=stats[1], dtable=dtable, accumulate=accumulate)
    head = (q, k, v, table, limits, scale, window, sinks, start)
    scratch = torch.empty(lib.nmb_band_bwd_scratch(_pack(*head, **common)), dtype=torch.float32, device=q.device)
    native.check_rc(lib.nmb_band_bwd(_pack(*head, scratch=scratch, **common), native.stream_ptr(q.device)), "nmb_band_bwd")
    return dq, dk, dv


class _BandAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, limits, scale, window, sinks, start):
        ctx.table_param = table
        ctx.meta = (limits, scale, window, sinks, start)
        q, k, v = _readable(q), _readable(k), _readable(v)
        if table is not None:
            table = table.contiguous()
        with torch.cuda.device(q.device):
            out, stats = _band_fwd(q, k, v, table, *ctx.meta)
        ctx.save_for_backward(q, k, v, table, out, stats)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        from .functional import _deliver_grad
        q, k, v, table, out, stats = ctx.saved_tensors
        grads = []

        def run(dtable=None, accumulate=False):
            with torch.cuda.device(q.device):
                grads.extend(_band_bwd(q, k, v, table, *ctx.meta, out, stats, dout, dtable, accumulate))

        dtable = None
        if table is not None and ctx.needs_input_grad[3]:
            def compute(buffer, accumulate):
                target = torch.empty_like(table) if buffer is None else buffer
                if not target.is_contiguous() or target.dtype not in (torch.bfloat16, torch.float32):
                    target = torch.empty_like(table)
                run(target, accumulate and target is buffer)
                if buffer is not None and target is not buffer:
                    buffer.add_(target) if accumulate else buffer.copy_(target)
                return target
            dtable = _deliver_grad(ctx.table_param, compute)
        else:
            run()
        dq, dk, dv = grads
        return dq, dk, dv, dtable, None, None, None, None, None


# ------------------------------------------------------------------ checks --
def _check_int(name: str, value, low: int) -> int:
    if isinstance(value, bool) or not isinstance(value, int):
        raise TypeError(f"{name} must be an int, got {type(value).__name__}")
    if not low <= value <= _INT_MAX:
        raise ValueError(f"{name} must be at least {low}, got {value}")
    return value


def _check_buckets(num_buckets: int, max_distance: int) -> None:
    _check_int("max_distance", max_distance, 1)
    if not 2 <= num_buckets <= MAX_BUCKETS:
        raise ValueError(f"the table must have 2 to {MAX_BUCKETS} buckets, got {num_buckets}")
    if not num_buckets // 2 < max_distance <= MAX_DISTANCE:
        raise ValueError(f"max_distance must be above num_buckets // 2 ({num_buckets // 2}) and at most {MAX_DISTANCE}, "
                         f"got {max_distance}")


def _check(q: Tensor, k: Tensor, v: Tensor, scale: float, window: Optional[int], sinks: int, query_start: int):
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError(f"q, k, v must be 4D [B,S,H,D]; got q={tuple(q.shape)}, k={tuple(k.shape)}, v={tuple(v.shape)}")
    if k.shape != v.shape:
        raise ValueError(f"k and v must share shape; got k={tuple(k.shape)}, v={tuple(v.shape)}")
    if q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError(f"q/k batch and head_dim must match; got q={tuple(q.shape)}, k={tuple(k.shape)}")
    if k.shape[2] == 0 or q.shape[2] % k.shape[2] != 0:
        raise ValueError(f"query heads must be a multiple of key heads; got q={tuple(q.shape)}, k={tuple(k.shape)}")
    if not q.dtype == k.dtype == v.dtype or not q.is_floating_point():
        raise ValueError(f"q, k, v must share a floating type; got {q.dtype}, {k.dtype}, {v.dtype}")
    if not q.device == k.device == v.device:
        raise ValueError(f"q, k, v must be on one device; got {q.device}, {k.device}, {v.device}")
    scale = float(scale)
    if not (math.isfinite(scale) and scale > 0.0):
        raise ValueError(f"scale must be finite and positive, got {scale}")
    window = _INT_MAX if window is None else _check_int("window", window, 1)
    sinks = _check_int("sinks", sinks, 0)
    start = _check_int("query_start", query_start, 0)
    if start + q.shape[1] > _MAX_POSITION or k.shape[1] > _MAX_POSITION:
        raise ValueError(f"positions must stay below {_MAX_POSITION}; got query_start {start}, q={tuple(q.shape)}, "
                         f"k={tuple(k.shape)}")
    return scale, window, sinks, start


# ------------------------------------------------------------ entry points --
def window_attention(q: Tensor, k: Tensor, v: Tensor, scale: float, *, window: int, sinks: int = 0,
                     query_start: int = 0) -> Tensor:
    """Causal attention in which a query sees the last ``window`` positions, its own included, and the first ``sinks`` keys
    of the sequence.  ``[B, Sq, Hq, d]``, ``[B, Skv, Hkv, d]`` -> ``[B, Sq, Hq, d]``."""
    if window is None:
        raise TypeError("window must be an int")
    scale, window, sinks, start = _check(q, k, v, scale, window, sinks, query_start)
    if band_attention_supported(q) and q.numel() and k.numel():
        return _BandAttention.apply(q, k, v, None, b"", scale, window, sinks, start)
    return _expression(q, k, v, None, 0, scale, window, sinks, start)


def relative_bias_attention(q: Tensor, k: Tensor, v: Tensor, table: Tensor, scale: float, *, max_distance: int = 128,
                            window: Optional[int] = None, sinks: int = 0, query_start: int = 0) -> Tensor:
    """Causal attention with the bias ``table[head, bucket(distance)]`` on the scores (``table`` is ``[Hq, buckets]``, bf16 or
    fp32; :func:`relative_bucket_limits` gives the buckets), inside a window as in :func:`window_attention` where one is
    given.  Entries of ``-inf`` mask their bucket."""
    scale, window, sinks, start = _check(q, k, v, scale, window, sinks, query_start)
    if table.dim() != 2 or table.shape[0] != q.shape[2]:
        raise ValueError(f"table must be [query heads, buckets] with {q.shape[2]} heads; got {tuple(table.shape)}")
    if table.device != q.device:
        raise ValueError(f"table must be on {q.device}, got {table.device}")
    _check_buckets(table.shape[1], max_distance)
    if band_attention_supported(q) and q.numel() and k.numel():
        if table.dtype not in (torch.bfloat16, torch.float32):
            raise ValueError(f"table must be bfloat16 or float32, got {table.dtype}")
        return _BandAttention.apply(q, k, v, table, _packed_limits(table.shape[1], max_distance), scale, window, sinks, start)
    return _expression(q, k, v, table, max_distance, scale, window, sinks, start)


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
