"""Scores that are not finite in the banded attention kernels: a run that has diverged must show it.

A NaN or +inf among the scores that a row sees makes the row NaN; a score of -inf is a weight of 0, as an entry of -inf in the
table is, and a row that has nothing else gives zeros."""
from __future__ import annotations

import math

import pytest
import torch

from tests.test_gpu_band_attention import _call, _tensors

pytestmark = pytest.mark.gpu

HUGE = 3.0e38  # bf16 holds it, the product of two does not fit fp32


def _run(q, k, v, table, dout, grads=True, **kw):
    if not grads:
        with torch.no_grad():
            return [_call(q, k, v, table, 0.125, 128, **kw)]
    out = _call(q, k, v, table, 0.125, 128, **kw)
    leaves = [q, k, v] + ([] if table is None else [table])
    return [out, *torch.autograd.grad(out, leaves, dout)]


def _nan_rows(t, rows):
    """All of these rows NaN, in every element, and no other."""
    bad = t.isnan()
    return bool(bad[:, rows].all()) and not bool(bad[:, ~rows].any())


# 700 rows: tiles that are masked in part and tiles that are not, also of query rows of another tile; 16 heads make pairs of tiles
SHAPES = [(1, 700, 2, 2, 64, 0), (1, 700, 2, 1, 96, 0), (1, 700, 2, 2, 128, 0), (1, 700, 2, 1, 64, 32), (1, 700, 2, 2, 128, 32),
          (2, 700, 16, 8, 64, 0), (2, 700, 15, 5, 128, 0)]


@pytest.mark.parametrize("b,s,hq,hkv,d,buckets", SHAPES)
@pytest.mark.parametrize("grads", [False, True])
@pytest.mark.parametrize("key", [5, 6, 7, 391])
def test_nan_in_a_key(b, s, hq, hkv, d, buckets, grads, key):
    q, k, v, table, dout = _tensors(b, s, s, hq, hkv, d, buckets)
    clean = _run(q, k, v, table, dout, grads, window=600)
    with torch.no_grad():
        k[:, key] = math.nan
    got = _run(q, k, v, table, dout, grads, window=600)
    at = torch.arange(s, device="cuda")
    rows = (at >= key) & (at - key < 600)
    assert _nan_rows(got[0], rows)
    assert torch.equal(got[0][:, ~rows], clean[0][:, ~rows])
    if grads:
        # whole tiles are multiplied: a key that is not finite also shows in dQ of rows of the tile that do not see it
        assert got[1].isnan()[:, rows].all() and torch.equal(got[1][:, :key // 128 * 128], clean[1][:, :key // 128 * 128])
        seen = (at > key - 600) & (at < key + 600)  # by a row that sees `key`
        for g in got[2:4]:
            assert g.isnan()[:, seen].all()
        if buckets:
            assert got[4].isnan().all()


@pytest.mark.parametrize("b,s,hq,hkv,d,buckets", SHAPES)
def test_nan_in_a_query(b, s, hq, hkv, d, buckets):
    row = 414
    q, k, v, table, dout = _tensors(b, s, s, hq, hkv, d, buckets)
    clean = _run(q, k, v, table, dout, window=250)
    with torch.no_grad():
        q[:, row, :, 3] = math.nan
    got = _run(q, k, v, table, dout, window=250)
    at = torch.arange(s, device="cuda")
    for n in range(2):
        assert _nan_rows(got[n], at == row) and torch.equal(got[n][:, at != row], clean[n][:, at != row])
    seen = (at <= row) & (at > row - 250)
    for n in (2, 3):
        assert got[n].isnan()[:, seen].all()
        apart = (at >= 512) | (at < 128)  # key tiles that the row does not see
        assert torch.equal(got[n][:, apart], clean[n][:, apart])


@pytest.mark.parametrize("b,s,hq,hkv,d,buckets", SHAPES)
@pytest.mark.parametrize("key", [5, 6, 391])
def test_a_score_beyond_fp32(b, s, hq, hkv, d, buckets, key):
    row = 500
    q, k, v, table, dout = _tensors(b, s, s, hq, hkv, d, buckets)
    with torch.no_grad():
        q[..., 0] = 0
        k[..., 0] = 0
        clean = _run(q, k, v, table, dout, False, window=600)[0]
        q[:, row, :, 0] = HUGE
        k[:, key, :, 0] = HUGE
    got = _run(q, k, v, table, dout, window=600)
    at = torch.arange(s, device="cuda")
    assert _nan_rows(got[0], at == row) and _nan_rows(got[1], at == row)
    for n in (2, 3):
        assert got[n].isnan()[:, at <= row].all()
    with torch.no_grad():
        k[:, key, :, 0] = -HUGE
        off = _run(q, k, v, table, dout, False, window=600)[0]
        k[:, key] = 0
        v[:, key] = 0
    # -inf: as if the key were not there
    assert off.isfinite().all() and torch.equal(off[:, at != row], clean[:, at != row])
    want = _expression_without(q, k, v, table, row, key)
    assert (off[:, row].double() - want).abs().max() <= 2 * torch.finfo(torch.bfloat16).eps / 2 * v.abs().max()


def _expression_without(q, k, v, table, row, key):
    from tests._band_oracle import bucket

    group = q.shape[2] // k.shape[2]
    kh, vh = (t[:, :row + 1].double().transpose(1, 2).repeat_interleave(group, 1) for t in (k.detach(), v.detach()))
    x = torch.einsum("bhd,bhjd->bhj", q.detach()[:, row].double(), kh) * 0.125
    if table is not None:
        x = x + table.detach().double()[:, torch.tensor([bucket(row - j, table.shape[1], 128) for j in range(row + 1)], device=x.device)]
    x[..., key] = -math.inf
    return torch.einsum("bhj,bhjd->bhd", torch.softmax(x, -1), vh)


@pytest.mark.parametrize("b,s,hq,hkv,d,buckets", SHAPES)
def test_a_row_of_scores_below_fp32(b, s, hq, hkv, d, buckets):
    q, k, v, table, dout = _tensors(b, s, s, hq, hkv, d, buckets)
    rows = torch.zeros(s, dtype=torch.bool, device="cuda")
    rows[[0, 140, 500, 699]] = True
    with torch.no_grad():
        q[..., 0] = 0
        clean = _run(q, k, v, table, dout, False, window=2000)[0]
        q[:, rows, :, 0] = HUGE
        k[..., 0] = -HUGE
    out, dq = _run(q, k, v, table, dout, window=2000)[:2]
    assert (out[:, rows] == 0).all() and out.isfinite().all()
    # such a row passes nothing on but what rounding leaves of zero
    with torch.no_grad():
        out = _run(q, k, v, table, dout, False, window=2000)[0]
    assert (out[:, rows] == 0).all() and out.isfinite().all()
    assert (out[:, ~rows] - clean[:, ~rows]).abs().max() <= 4 * torch.finfo(torch.bfloat16).eps * v.abs().max()


@pytest.mark.parametrize("grads", [False, True])
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("at_bucket", [0, 9, 31])
def test_table_entries(grads, value, d, at_bucket):
    from nano_megatron_b200.ops.band_attention import relative_bucket_limits

    q, k, v, table, dout = _tensors(1, 700, 700, 2, 2, d, 32)
    clean = _run(q, k, v, table, dout, grads)
    with torch.no_grad():
        table[1, at_bucket] = value
    got = _run(q, k, v, table, dout, grads)
    first = (0, *relative_bucket_limits(32, 128))[at_bucket]
    rows = torch.arange(700, device="cuda") >= first
    for n in range(2 if grads else 1):
        assert torch.equal(got[n][:, :, 0], clean[n][:, :, 0])
        assert _nan_rows(got[n][:, :, 1], rows)
        assert torch.equal(got[n][:, ~rows], clean[n][:, ~rows])
    if grads:
        assert torch.equal(got[4][0], clean[4][0]) and got[4][1].isnan().all()


@pytest.mark.parametrize("buckets", [0, 32])
@pytest.mark.parametrize("key", [6, 1500, 4000])
def test_few_rows_over_many_keys(buckets, key):
    q, k, v, table, dout = _tensors(1, 3, 4096, 4, 2, 128, buckets)
    with torch.no_grad():
        k[:, key, 0] = math.nan
    got = _run(q, k, v, table, dout, window=5000, query_start=4093)
    for n in range(2):
        assert got[n][:, :, :2].isnan().all() and got[n][:, :, 2:].isfinite().all()
    for n in (2, 3):
        assert got[n][:, :4094, 0].isnan().all() and got[n][:, :, 1].isfinite().all()
