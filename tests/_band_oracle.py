"""Banded causal attention with a relative position bias, written from its definition in 64 bits, with the bounds that
the kernels' roundings to bf16 allow (``torch.finfo(bfloat16).eps / 2`` relative to the rounded value each)."""
from __future__ import annotations

import math

import torch

U = torch.finfo(torch.bfloat16).eps / 2      # one rounding to bf16
E = 2.0 ** -13                               # everything held in fp32: sums of up to 2^10 terms, exponentials, scores
RMS = U / math.sqrt(3.0)                     # root mean square of a rounding's relative error


def bucket(n: int, buckets: int, max_distance: int) -> int:
    """Bucket of distance ``n``: exact below half of the buckets, then evenly in the logarithm, in whole numbers."""
    exact = buckets // 2
    if n < exact:
        return n
    grow = buckets - exact
    t = 0
    while exact + t + 1 < buckets and n ** grow * exact ** (t + 1) >= max_distance ** (t + 1) * exact ** grow:
        t += 1
    return exact + t


def visible(sq, skv, window, sinks, start, device="cpu"):
    p = torch.arange(start, start + sq, device=device)[:, None]
    j = torch.arange(skv, device=device)[None, :]
    see = j <= p
    if window is not None:
        see = see & ((p - j < window) | (j < sinks))
    return see


def oracle(q, k, v, dout, scale, *, window=None, sinks=0, start=0, table=None, max_distance=128):
    """``(values, bounds, rms)``: dicts with out, dq, dk, dv (and dtable) in 64 bits, the largest error of each element
    that the roundings of the weights, of the score gradients, of the output and of the results allow, and the relative
    Frobenius error that independent roundings of that size amount to."""
    q, k, v, dout = (t.detach().double() for t in (q, k, v, dout))
    b, sq, hq, d = q.shape
    skv, hkv = k.shape[1], k.shape[2]
    group = hq // hkv
    qh, g = q.transpose(1, 2), dout.transpose(1, 2)
    kh = k.transpose(1, 2).repeat_interleave(group, 1)
    vh = v.transpose(1, 2).repeat_interleave(group, 1)
    x = qh @ kh.transpose(2, 3) * scale
    if table is not None:
        apart = (torch.arange(start, start + sq)[:, None] - torch.arange(skv)[None, :]).clamp(min=0)
        of = torch.tensor([bucket(n, table.shape[1], max_distance) for n in range(start + sq)], dtype=torch.long)
        at = of[apart].to(q.device)
        x = x + table.detach().double()[:, at]
    see = visible(sq, skv, window, sinks, start, q.device)
    x = x.masked_fill(~see, -math.inf)
    top = x.amax(-1, keepdim=True)
    w = torch.where(torch.isneginf(x), torch.zeros_like(x), torch.exp(x - torch.where(torch.isneginf(top), 0.0, top)))
    total = w.sum(-1, keepdim=True)
    p = w / torch.where(total == 0, 1.0, total)
    out = p @ vh
    out_bound = U * out.abs() + (U + E) * (p @ vh.abs())
    dp = g @ vh.transpose(2, 3)
    delta = (g * out).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    # D comes from the output and what its rounding cut off, both in bf16: an error of the weights' rounding and of U * U;
    # dP - D from sums of absolute size |dO| |V| and |dO| |O|
    soft = (g.abs() * (U * U * out.abs() + (U + E) * (p @ vh.abs()))).sum(-1, keepdim=True) + E * (g.abs() @ vh.abs().transpose(2, 3) + (g * out).abs().sum(-1, keepdim=True))
    ds_err = p * soft + E * ds.abs()

    def grouped(t):  # sum of a group's query heads
        return t.reshape(b, hkv, group, skv, d).sum(2).transpose(1, 2)

    def rows(t):
        return t.transpose(1, 2)

    dq = ds @ kh * scale
    dk = grouped(ds.transpose(2, 3) @ qh * scale)
    dv = grouped(p.transpose(2, 3) @ g)
    dq_bound = U * dq.abs() + (((U + E) * ds.abs() + ds_err) @ kh.abs() * scale)
    dk_bound = U * dk.abs() + grouped(((U + E) * ds.abs() + ds_err).transpose(2, 3) @ qh.abs() * scale)
    dv_bound = U * dv.abs() + (U + E) * grouped(p.transpose(2, 3) @ g.abs())
    values = {"out": rows(out), "dq": rows(dq), "dk": dk, "dv": dv}
    bounds = {"out": rows(out_bound), "dq": rows(dq_bound), "dk": dk_bound, "dv": dv_bound}
    # independent roundings: the weights and the result (out, dv); these, the score gradients and D (dq, dk)
    rms = {"out": math.sqrt(2) * RMS, "dv": math.sqrt(2) * RMS, "dq": 2 * RMS, "dk": 2 * RMS}
    if table is not None:
        n = table.shape[1]
        hot = torch.nn.functional.one_hot(at, n).double()
        hot = hot * see.unsqueeze(-1)
        dtable = torch.einsum("bhij,ijn->hn", ds, hot)
        last = U if table.dtype == torch.bfloat16 else 0.0
        values["dtable"] = dtable
        bounds["dtable"] = last * dtable.abs() + torch.einsum("bhij,ijn->hn", ds_err, hot)
        rms["dtable"] = 2 * RMS
    return values, bounds, rms


def check(got, values, bounds, rms, what=""):
    for name, t in got.items():
        if t is None:
            continue
        want, bound = values[name], bounds[name]
        assert t.shape == want.shape, (what, name, t.shape, want.shape)
        t = t.detach().double()
        assert torch.isfinite(t).all(), f"{what} {name}: not finite"
        off = (t - want).abs()
        # values that are zero but for cancellation: fp32 sums of the terms, which the bounds hold in E
        worst = (off - bound - 1e-30).max().item()
        assert worst <= 0, f"{what} {name}: an element is {off.flatten()[(off - bound).argmax()].item():.3e} off, " \
                           f"{bound.flatten()[(off - bound).argmax()].item():.3e} is allowed"
        norm = want.norm().item()
        # the statistics of independent roundings need enough of them, and a result that is more than cancellation
        if want.numel() >= 4096 and norm > 16 * bound.norm().item():
            rel = off.norm().item() / norm
            assert rel <= 1.25 * rms[name], f"{what} {name}: relative Frobenius error {rel:.2e} > {1.25 * rms[name]:.2e}"
