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
to be finite in masked places too.  Values that are not finite show: a row that sees a score of NaN or +inf
(an overflow of fp32 among them, or an entry of the table) is NaN, and so are the gradients that it takes part
in; a score of -inf is a weight of 0, as an entry of -inf in the table is, and a row that has nothing else
gives zeros.

With a bias table, or where rows see few keys, a call that will be differentiated carries the weights to twice
bf16's digits, for the gradients' sake: its output may differ from that of the same call without gradients by
the roundings of the weights.  Results do not depend on timing: the same call gives the same bits.

The kernels cannot be traced (``torch.compile``, fake tensors) nor transformed (``torch.func``): such calls are
refused.
"""
from __future__ import annotations

import functools
import math
from typing import Optional

import torch
from torch import Tensor

from . import native
from .functional import _deliver_grad

MAX_BUCKETS = 128        # sizes of the kernels' tables
MAX_DISTANCE = 2048
_MAX_POSITION = 2 ** 30
_INT_MAX = 2 ** 31 - 1
_SCALE_LIMIT = 2.0 ** 126  # held in fp32 by the kernels, times log2(e)


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


# --------------------------------------------------------------- operators --
_ready = []  # the operator, once a device has been set up


@functools.lru_cache(maxsize=None)
def _operator(device_index: int):
    """The operator of ``csrc/torch_binding.cpp``, ready for a device (whose status word the kernels report to)."""
    ops = native.torch_lib()
    with torch.cuda.device(device_index):
        native.lib()
        ops.band_device(device_index, native.status_word(torch.device("cuda", device_index)).data_ptr())
    _ready[:] = [ops.band_attention.default]
    return _ready[0]


@functools.lru_cache(maxsize=None)
def _register_buckets(num_buckets: int, max_distance: int) -> None:
    native.torch_lib().band_limits(num_buckets, max_distance, list(relative_bucket_limits(num_buckets, max_distance)))


class _ToMainGrad(torch.autograd.Function):
    """A table whose gradient is kept in ``main_grad``: passes the table on, and what comes back to that buffer."""

    @staticmethod
    def forward(ctx, table):
        ctx.param = table
        return table.view_as(table)

    @staticmethod
    def backward(ctx, grad):
        def compute(buffer, accumulate):
            if buffer is None:
                return grad
            buffer.add_(grad) if accumulate else buffer.copy_(grad)
            return buffer
        return _deliver_grad(ctx.param, compute)


def _trained(table):
    if table is not None and getattr(table, "main_grad", None) is not None and table.requires_grad and torch.is_grad_enabled():
        return _ToMainGrad.apply(table)
    return table


# ------------------------------------------------------------------ checks --
def _check_int(name: str, value, low: int) -> int:
    if isinstance(value, bool) or not isinstance(value, int):
        raise TypeError(f"{name} must be an int, got {type(value).__name__}")
    if not low <= value <= _INT_MAX:
        raise ValueError(f"{name} must be at least {low} and below 2 ** 31, got {value}")
    return value


def _check_buckets(num_buckets: int, max_distance: int) -> None:
    if not 2 <= num_buckets <= MAX_BUCKETS:
        raise ValueError(f"the table must have 2 to {MAX_BUCKETS} buckets, got {num_buckets}")
    if not num_buckets // 2 < max_distance <= MAX_DISTANCE:
        raise ValueError(f"max_distance must be above num_buckets // 2 ({num_buckets // 2}) and at most {MAX_DISTANCE}, "
                         f"got {max_distance}")


def check_band(window: Optional[int], sinks: int, num_buckets: Optional[int], max_distance: Optional[int]) -> None:
    """Refuses what the operators refuse of these (``None`` for a window or a table that is not there)."""
    if window is not None:
        _check_int("window", window, 1)
    _check_int("sinks", sinks, 0)
    if num_buckets is not None:
        _check_int("the number of buckets", num_buckets, 2)
        _check_int("max_distance", max_distance, 1)
        _check_buckets(num_buckets, max_distance)


@functools.lru_cache(maxsize=4096)
def _check_shapes(q, k, v, floating, buckets, max_distance, scale, start) -> None:
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
    if not 1.0 / _SCALE_LIMIT <= scale <= _SCALE_LIMIT:  # a NaN neither
        raise ValueError(f"scale must be positive and within 2 ** -126 and 2 ** 126, got {scale}")
    if start + q[1] > _MAX_POSITION or k[1] > _MAX_POSITION:
        raise ValueError(f"positions must stay below {_MAX_POSITION}; got query_start {start}, q={tuple(q)}, k={tuple(k)}")
    if buckets is not None:
        _check_buckets(buckets, max_distance)


def _refuse_tracing(*tensors) -> None:
    """What ``csrc/torch_binding.cpp`` refuses, before a device is set up under a mode that hands out tensors without memory."""
    keys = torch._C._TorchDispatchModeKey
    if (any(torch._C._get_dispatch_mode(key) is not None for key in (keys.FAKE, keys.PROXY, keys.FUNCTIONAL))
            or any(t is not None and torch._C._dispatch_keys(t).has(torch._C.DispatchKey.Python) for t in tensors)):
        raise NotImplementedError("banded attention: the kernels cannot be traced; wrap the call in torch.compiler.disable")


def _attend(q, k, v, table, max_distance, scale, window, sinks, start) -> Tensor:
    if _ready and q.is_cuda and type(scale) is float and type(window) is type(sinks) is type(start) is type(max_distance) is int:
        # one look from C++ in place of those below, which took as long as the rest of a call together
        out = _ready[0](q, k, v, _trained(table), scale, window, sinks, start, max_distance)
        if out is not None:
            return out
    if not q.dtype == k.dtype == v.dtype:
        raise ValueError(f"q, k, v must share a floating type; got {q.dtype}, {k.dtype}, {v.dtype}")
    if not q.device == k.device == v.device:
        raise ValueError(f"q, k, v must be on one device; got {q.device}, {k.device}, {v.device}")
    window = _check_int("window", window, 1)
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
    _check_shapes(q.shape, k.shape, v.shape, q.is_floating_point(), buckets, max_distance, scale, start)
    if band_attention_supported(q) and q.numel() and k.numel():
        _refuse_tracing(q, k, v, table)
        if table is not None:
            if table.dtype not in (torch.bfloat16, torch.float32):
                raise ValueError(f"table must be bfloat16 or float32, got {table.dtype}")
            _register_buckets(buckets, max_distance)
        out = _operator(q.device.index)(q, k, v, _trained(table), scale, window, sinks, start, max_distance)
        if out is not None:
            return out
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
    return _attend(q, k, v, table, max_distance, scale, _INT_MAX if window is None else window, sinks, query_start)


def visible_softmax(scores: Tensor) -> Tensor:
    """Softmax over the last dimension in which a score of ``-inf`` weighs nothing; a row of nothing else gives zeros."""
    if scores.shape[-1] == 0:
        return scores
    top = scores.detach().amax(dim=-1, keepdim=True).clamp(min=torch.finfo(scores.dtype).min)
    weights = torch.exp(scores - top)
    total = weights.sum(dim=-1, keepdim=True)
    return weights / torch.where(total == 0, torch.ones_like(total), total)


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
    return torch.matmul(visible_softmax(scores), vh).transpose(1, 2).to(q.dtype)
