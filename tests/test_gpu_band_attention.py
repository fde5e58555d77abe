"""The banded attention kernels against the definition in 64 bits."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from tests._band_oracle import bucket, check, oracle, visible

pytestmark = pytest.mark.gpu


class _Stride(ctypes.Structure):
    _fields_ = [(n, ctypes.c_longlong) for n in "bsh"]


_TENSORS = ("q", "k", "v", "o", "dout", "dq", "dk", "dv")
_POINTERS = ("q", "k", "v", "o", "o_rest", "dout", "dq", "dk", "dv", "m", "l", "scratch", "table", "dtable", "status")


class _Args(ctypes.Structure):
    """BandArgs of csrc/band_args.h."""
    _fields_ = ([(n, ctypes.c_void_p) for n in _POINTERS]
                + [(n + "_st", _Stride) for n in _TENSORS]
                + [(n, ctypes.c_int) for n in ("table_fp32", "dtable_fp32", "B", "Hq", "Hkv", "Sq", "Skv", "d", "q_pos0", "window",
                                               "sinks", "buckets")]
                + [("scale", ctypes.c_float), ("rest_rows", ctypes.c_int), ("limit", ctypes.c_ushort * 128)])


def _launches():
    from nano_megatron_b200.ops import native

    return native.lib().nmb_band_launches()


def _tensors(b, sq, skv, hq, hkv, d, buckets=0, layout="bshd", seed=0, table_dtype=torch.bfloat16, gain=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(torch.bfloat16)

    if layout == "packed":
        assert sq == skv
        q, k, v = normal(b, sq, (hq + 2 * hkv) * d).split([hq * d, hkv * d, hkv * d], dim=-1)
        q, k, v = q.unflatten(-1, (hq, d)), k.unflatten(-1, (hkv, d)), v.unflatten(-1, (hkv, d))
    elif layout == "bhsd":
        q, k, v = (normal(b, h, s, d).transpose(1, 2) for h, s in ((hq, sq), (hkv, skv), (hkv, skv)))
    elif layout == "odd":  # rows that tile loads cannot address: the last dimension with a stride, an unaligned start
        q = normal(b, sq, hq, 2 * d)[..., ::2]
        k = normal(b * skv * hkv * d + 1)[1:].view(b, skv, hkv, d)
        v = normal(b, skv, hkv, d + 4)[..., :d]
    else:
        q, k, v = normal(b, sq, hq, d), normal(b, skv, hkv, d), normal(b, skv, hkv, d)
    if gain != 1.0:
        q = (q.float() * gain).to(torch.bfloat16)
    table = None
    if buckets:
        table = torch.randn(hq, buckets, generator=g, device="cuda").to(table_dtype).requires_grad_(True)
    return [t.detach().requires_grad_(True) for t in (q, k, v)] + [table, normal(b, sq, hq, d)]


def _call(q, k, v, table, scale, max_distance, **kw):
    from nano_megatron_b200.ops.band_attention import relative_bias_attention, window_attention

    if table is None:
        return window_attention(q, k, v, scale, **kw)
    return relative_bias_attention(q, k, v, table, scale, max_distance=max_distance, **kw)


def _compare(q, k, v, table, dout, *, window=None, sinks=0, start=0, max_distance=128, scale=None, what=""):
    from nano_megatron_b200.ops import native

    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    before = _launches()
    out = _call(q, k, v, table, scale, max_distance, window=window, sinks=sinks, query_start=start)
    leaves = [q, k, v] + ([] if table is None else [table])
    grads = torch.autograd.grad(out, leaves, dout)
    torch.cuda.synchronize()
    native.check_status()
    assert _launches() >= before + 3  # the kernels ran: forward, dQ, dK and dV
    values, bounds, rms = oracle(q, k, v, dout, scale, window=window, sinks=sinks, start=start, table=table, max_distance=max_distance)
    check(dict(zip(("out", "dq", "dk", "dv", "dtable"), (out, *grads))), values, bounds, rms, what)


# b, sq, skv, hq, hkv, d, window, sinks, start
WINDOWS = [
    (1, 1, 1, 1, 1, 64, 1, 0, 0), (2, 2, 2, 2, 1, 128, 2, 0, 0), (1, 5, 5, 2, 2, 96, 3, 1, 0),
    (1, 64, 64, 2, 2, 64, 16, 0, 0), (1, 127, 127, 2, 1, 96, 40, 3, 0), (2, 128, 128, 1, 1, 128, 128, 0, 0),
    (1, 129, 129, 4, 2, 64, 2, 0, 0), (1, 255, 255, 3, 1, 128, 64, 65, 0), (2, 256, 256, 2, 2, 64, 127, 1, 0),
    (1, 257, 257, 2, 2, 96, 128, 0, 0), (1, 300, 300, 8, 1, 64, 129, 4, 0), (2, 513, 513, 4, 4, 64, 1, 0, 0),
    (1, 640, 640, 2, 1, 128, 256, 130, 0), (1, 777, 777, 3, 3, 96, 300, 0, 0), (1, 1000, 1000, 2, 2, 64, 100, 1000, 0),
    (1, 1100, 1100, 1, 1, 128, 2000, 0, 0),
    # shards: one row, rows that start inside a tile, few rows over many keys, more keys than rows can see
    (2, 1, 700, 4, 2, 64, 200, 3, 699), (1, 33, 500, 2, 1, 128, 90, 0, 467), (1, 300, 900, 4, 4, 96, 1000, 0, 600),
    (1, 200, 900, 2, 2, 64, 64, 5, 100), (1, 130, 2000, 2, 1, 64, 1500, 0, 1870),
    # shards behind the keys: rows whose window holds no key, with sinks and without
    (1, 200, 100, 2, 2, 64, 30, 0, 50), (1, 200, 100, 2, 1, 128, 30, 2, 50), (2, 10, 5, 1, 1, 96, 3, 0, 200), (1, 400, 128, 2, 2, 64, 100, 0, 0),
]


@pytest.mark.parametrize("b,sq,skv,hq,hkv,d,window,sinks,start", WINDOWS)
def test_window(b, sq, skv, hq, hkv, d, window, sinks, start):
    _compare(*_tensors(b, sq, skv, hq, hkv, d), window=window, sinks=sinks, start=start)


# b, sq, skv, hq, hkv, d, window, sinks, start, buckets, max_distance
BIASES = [
    (1, 1, 1, 1, 1, 64, None, 0, 0, 2, 2), (2, 3, 3, 2, 1, 128, None, 0, 0, 32, 128), (1, 33, 33, 4, 4, 64, None, 0, 0, 32, 128),
    (1, 128, 128, 2, 2, 96, None, 0, 0, 32, 128), (2, 200, 200, 4, 2, 64, None, 0, 0, 20, 40), (1, 257, 257, 2, 2, 128, None, 0, 0, 5, 300),
    (3, 390, 390, 3, 1, 96, None, 0, 0, 128, 256), (1, 700, 700, 2, 2, 64, None, 0, 0, 64, 600), (1, 1300, 1300, 2, 1, 128, None, 0, 0, 32, 128),
    (1, 600, 600, 2, 2, 64, None, 0, 0, 3, 2), (1, 600, 600, 1, 1, 128, None, 0, 0, 128, 2048),
    (1, 513, 513, 4, 1, 64, 100, 3, 0, 16, 64), (2, 300, 300, 2, 2, 128, 33, 0, 0, 32, 128), (1, 450, 450, 8, 2, 96, 200, 140, 0, 32, 100),
    (1, 1, 600, 2, 2, 64, None, 0, 599, 32, 128), (2, 70, 500, 4, 2, 128, None, 0, 430, 32, 128), (1, 150, 700, 2, 1, 96, 120, 4, 333, 32, 128),
    (1, 200, 90, 2, 2, 64, 40, 0, 60, 16, 30), (1, 200, 90, 2, 2, 64, None, 0, 60, 16, 30),
]


@pytest.mark.parametrize("b,sq,skv,hq,hkv,d,window,sinks,start,buckets,distance", BIASES)
def test_bias(b, sq, skv, hq, hkv, d, window, sinks, start, buckets, distance):
    _compare(*_tensors(b, sq, skv, hq, hkv, d, buckets), window=window, sinks=sinks, start=start, max_distance=distance)


@pytest.mark.parametrize("layout", ["packed", "bhsd", "odd"])
@pytest.mark.parametrize("d", [64, 96, 128])
def test_layouts(layout, d):
    _compare(*_tensors(2, 200, 200, 4, 2, d, layout=layout), window=70, sinks=2)
    _compare(*_tensors(2, 200, 200, 4, 2, d, 32, layout=layout))


def test_fp32_table():
    _compare(*_tensors(2, 300, 300, 4, 2, 64, 32, table_dtype=torch.float32))


def test_peaked_scores():
    # maxima that move by more than the threshold between tiles, in both directions
    _compare(*_tensors(1, 600, 600, 2, 2, 64, gain=12.0), window=400, sinks=4)
    _compare(*_tensors(1, 600, 600, 2, 2, 128, 32, gain=12.0))


@pytest.mark.parametrize("mask", [-math.inf, torch.finfo(torch.bfloat16).min, torch.finfo(torch.bfloat16).max])
@pytest.mark.parametrize("window", [None, 40])
def test_masked_buckets(mask, window):
    q, k, v, table, dout = _tensors(1, 400, 400, 4, 2, 64, 16)
    with torch.no_grad():
        table[0, 0] = mask      # a head that does not see its own position: its first row sees nothing, or itself after all
        table[1, 15] = mask     # nothing from some distance on
        table[2, 3:9] = mask
        table[3] = mask if mask == -math.inf else table[3]  # a head that sees nothing at all
    _compare(q, k, v, table, dout, window=window, max_distance=100)


def test_rows_of_one_lowest_value_are_averaged():
    q, k, v, table, dout = _tensors(1, 300, 300, 2, 2, 64, 16)
    with torch.no_grad():
        table.fill_(torch.finfo(torch.bfloat16).min)
        q.zero_()               # the scores add nothing: an even average of the visible keys
    _compare(q, k, v, table, dout, window=50, max_distance=100)


def test_broadcast_inputs_and_gradients():
    from nano_megatron_b200.ops.band_attention import window_attention

    q, k, v, _, _ = _tensors(1, 150, 150, 4, 1, 64)
    kb, vb = (t.expand(2, 150, 2, 64) for t in (k, v))
    qb = q.expand(2, 150, 4, 64)
    out = window_attention(qb, kb, vb, 0.125, window=40)
    ones = torch.ones((), device="cuda", dtype=torch.bfloat16).expand(out.shape)
    grads = torch.autograd.grad(out, (qb, kb, vb), ones, retain_graph=True)
    values, bounds, rms = oracle(qb, kb, vb, ones, 0.125, window=40)
    check(dict(zip(("out", "dq", "dk", "dv"), (out, *grads))), values, bounds, rms)
    out.sum().backward()
    assert q.grad.shape == q.shape and k.grad.shape == k.shape


def test_same_results_twice_and_only_what_is_asked_for():
    from nano_megatron_b200.ops.band_attention import relative_bias_attention

    q, k, v, table, dout = _tensors(2, 500, 500, 4, 2, 64, 32)
    runs = []
    for _ in range(3):
        out = relative_bias_attention(q, k, v, table, 0.125, window=300, sinks=4)
        runs.append((out, *torch.autograd.grad(out, (q, k, v, table), dout)))
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))
    frozen = table.detach()
    out = relative_bias_attention(q, k, v, frozen, 0.125, window=300, sinks=4)
    for a, b in zip(runs[0][1:], torch.autograd.grad(out, (q, k, v), dout)):
        assert torch.equal(a, b)


def test_main_grad_of_the_table():
    from nano_megatron_b200.ops.band_attention import relative_bias_attention

    q, k, v, table, dout = _tensors(1, 200, 200, 2, 2, 64, 16, table_dtype=torch.float32)
    want = torch.autograd.grad(relative_bias_attention(q, k, v, table, 0.125, max_distance=60), table, dout)[0]
    param = torch.nn.Parameter(table.detach().clone())
    for buffer in (torch.ones(2, 16, device="cuda"), torch.ones(16, 2, device="cuda").t()):
        param.main_grad, ready = buffer, []
        param._nmb_grad_ready = lambda: ready.append(1)
        relative_bias_attention(q, k, v, param, 0.125, max_distance=60).backward(dout)
        torch.testing.assert_close(buffer, want + 1, rtol=1e-6, atol=1e-6)
        assert param.grad is None
        param._nmb_overwrite_next = True
        relative_bias_attention(q, k, v, param, 0.125, max_distance=60).backward(dout)
        torch.testing.assert_close(buffer, want, rtol=0, atol=0)
        assert ready == [1, 1] and param.grad is None


def test_other_stream_and_two_calls_at_once():
    from nano_megatron_b200.ops.band_attention import relative_bias_attention

    sets = [_tensors(1, 400, 400, 4, 4, 64, 32, seed=s) for s in range(2)]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    results = []
    for _ in range(3):
        for st, (q, k, v, table, dout) in zip(streams, sets):
            with torch.cuda.stream(st):
                out = relative_bias_attention(q, k, v, table, 0.125)
                results.append((out, *torch.autograd.grad(out, (q, k, v, table), dout)))
    torch.cuda.synchronize()
    for n, (q, k, v, table, dout) in enumerate(sets):
        values, bounds, rms = oracle(q, k, v, dout, 0.125, table=table)
        for got in results[n::2]:
            check(dict(zip(("out", "dq", "dk", "dv", "dtable"), got)), values, bounds, rms)


def test_two_captured_graphs():
    from nano_megatron_b200.ops import native
    from nano_megatron_b200.ops.band_attention import relative_bias_attention, window_attention

    native.lib()
    q, k, v, table, dout = _tensors(2, 300, 300, 4, 2, 64, 32)
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # warm-up outside of a capture
        torch.autograd.grad(relative_bias_attention(q, k, v, table, 0.125), (q, k, v, table), dout)
    torch.cuda.current_stream().wait_stream(side)
    for n in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = window_attention(q, k, v, 0.125, window=77, sinks=3) if n == 0 else relative_bias_attention(q, k, v, table, 0.125)
            outs.append((out, *torch.autograd.grad(out, (q, k, v) if n == 0 else (q, k, v, table), dout)))
        graphs.append(g)
    for seed in (1, 2):
        fresh = _tensors(2, 300, 300, 4, 2, 64, 32, seed=seed)
        with torch.no_grad():
            for t, f in zip((q, k, v, table, dout), fresh):
                t.copy_(f)
        for g in graphs + graphs[::-1]:
            g.replay()
        torch.cuda.synchronize()
        native.check_status()
        for n in range(2):
            values, bounds, rms = oracle(q, k, v, dout, 0.125, **(dict(window=77, sinks=3) if n == 0 else dict(table=table)))
            check(dict(zip(("out", "dq", "dk", "dv", "dtable"), outs[n])), values, bounds, rms)


@pytest.mark.parametrize("sq,skv,d,start", [(1, 1, 64, 0), (37, 37, 96, 0), (130, 200, 128, 70), (300, 300, 64, 0)])
@pytest.mark.parametrize("buckets", [0, 32])
def test_nothing_is_written_outside(sq, skv, d, start, buckets):
    """Outputs inside larger buffers: what lies around them stays as it was."""
    from nano_megatron_b200.ops import band_attention as ba
    from nano_megatron_b200.ops import native

    b, hq, hkv, pad = 2, 4, 2, 9
    q, k, v, table, dout = (None if t is None else t.detach() for t in _tensors(b, sq, skv, hq, hkv, d, buckets))
    mark = 7.0
    lib = native.lib()
    assert lib.nmb_band_args_size() == ctypes.sizeof(_Args)

    def inside(s, h):
        big = torch.full((b, s + 2 * pad, h, d), mark, device="cuda", dtype=torch.bfloat16)
        return big, big[:, pad:pad + s]

    def flat(n):
        big = torch.full((n + 64,), mark, device="cuda")
        return big, big[32:32 + n]

    bufs = {n: inside(s, h) for n, s, h in (("o", sq, hq), ("dq", sq, hq), ("dk", skv, hkv), ("dv", skv, hkv))}
    stats = {n: flat(b * hq * sq) for n in ("m", "l")}
    if buckets:
        stats["dtable"] = flat(hq * buckets)
    rest = torch.full((b * sq * hq * d + 128,), mark, device="cuda", dtype=torch.bfloat16)
    args = _Args(o_rest=rest[64:].data_ptr(), B=b, Hq=hq, Hkv=hkv, Sq=sq, Skv=skv, d=d, q_pos0=start, window=50, sinks=3, buckets=buckets, scale=0.125, rest_rows=sq, dtable_fp32=1,
                 status=native.status_word(q.device).data_ptr(), table=None if table is None else table.data_ptr())
    if buckets:
        args.limit[:buckets - 1] = ba.relative_bucket_limits(buckets, 128)
    views = {n: t[1] for n, t in {**bufs, **stats}.items()} | {"q": q, "k": k, "v": v, "dout": dout}
    for n, t in views.items():
        setattr(args, n, t.data_ptr())
        if n in _TENSORS:
            setattr(args, n + "_st", _Stride(*t.stride()[:3]))
    stats["scratch"] = flat(lib.nmb_band_bwd_scratch(ctypes.byref(args)))
    args.scratch = stats["scratch"][1].data_ptr()
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    native.check_rc(lib.nmb_band_fwd(ctypes.byref(args), stream), "nmb_band_fwd")
    native.check_rc(lib.nmb_band_bwd(ctypes.byref(args), stream), "nmb_band_bwd")
    torch.cuda.synchronize()
    native.check_status()
    assert (rest[:64] == mark).all() and (rest[-64:] == mark).all() and not (rest[64:-64] == mark).all()
    for n, (big, view) in bufs.items():
        assert (big[:, :pad] == mark).all() and (big[:, pad + view.shape[1]:] == mark).all(), n
        assert not (view == mark).all(), n
    for n, (big, view) in stats.items():
        assert (big[:32] == mark).all() and (big[-32:] == mark).all(), n
    values, bounds, rms = oracle(q, k, v, dout, 0.125, window=50, sinks=3, start=start, table=table)
    check({n: views[n] for n in ("dq", "dk", "dv")} | {"out": views["o"]}, values, bounds, rms)


def test_float32_on_the_gpu_takes_the_expression():
    q, k, v, table, dout = (t.detach().float().requires_grad_(True) for t in _tensors(1, 70, 70, 2, 1, 64, 8))
    out = _call(q, k, v, table, 0.125, 20, window=30)
    values, _, _ = oracle(q, k, v, dout, 0.125, window=30, table=table, max_distance=20)
    torch.testing.assert_close(out.double(), values["out"], rtol=1e-4, atol=1e-5)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_tensors_of_another_device():
    q, k, v, table, dout = (t.detach().to("cuda:1").requires_grad_(True) for t in _tensors(1, 200, 200, 2, 2, 64, 32))
    with torch.cuda.device(0):
        _compare(q, k, v, table, dout)


def test_layout_of_the_gradients():
    from nano_megatron_b200.ops.band_attention import window_attention

    for layout in ("bshd", "bhsd"):  # the inputs' own layouts
        q, k, v, _, dout = _tensors(2, 100, 100, 4, 2, 64, layout=layout)
        for t, g in zip((q, k, v), torch.autograd.grad(window_attention(q, k, v, 0.125, window=30), (q, k, v), dout)):
            assert g.stride() == t.stride()
    qkv = torch.randn(2, 100, 8 * 64, device="cuda").to(torch.bfloat16)  # one buffer for the slices of a packed projection
    q, k, v = (t.unflatten(-1, (-1, 64)).detach().requires_grad_(True) for t in qkv.split([4 * 64, 2 * 64, 2 * 64], dim=-1))
    dq, dk, dv = torch.autograd.grad(window_attention(q, k, v, 0.125, window=30), (q, k, v), torch.ones(2, 100, 4, 64, device="cuda", dtype=torch.bfloat16))
    assert dq.stride() == q.stride() and dk.data_ptr() == dq.data_ptr() + 2 * 4 * 64 and dv.data_ptr() == dk.data_ptr() + 2 * 2 * 64


def test_not_differentiable_twice():
    from nano_megatron_b200.ops.band_attention import relative_bias_attention

    q, k, v, table, dout = _tensors(1, 40, 40, 2, 2, 64, 8)
    out = relative_bias_attention(q, k, v, table, 0.125, max_distance=20)
    grads = torch.autograd.grad(out, (q, k, v, table), dout, create_graph=True)
    plain = torch.autograd.grad(relative_bias_attention(q, k, v, table, 0.125, max_distance=20), (q, k, v, table), dout)
    assert all(torch.equal(a, b) for a, b in zip(grads, plain))
    with pytest.raises(RuntimeError, match="differentiated again"):
        grads[0].float().square().sum().backward()


@pytest.mark.parametrize("sq,hq,hkv,d,window,buckets,max_distance", [
    (3, 8, 1, 64, None, 18, 43), (22, 8, 1, 64, 21, 3, 27), (344, 4, 1, 128, None, 30, 43), (512, 2, 2, 96, None, 32, 128),
    (700, 2, 1, 64, 130, 4, 60)])
def test_gradient_of_the_bias_over_few_keys(sq, hq, hkv, d, window, buckets, max_distance):
    """Where a row sees few keys the table's gradient is as exact as fp32 sums of D's error allow: D comes from weights of
    twice bf16's digits, the output and what its rounding cut off: 2^-17 and 2^-18 of sum_j P_j sum_d |dO V_j|; the rest is held in
    fp32: 2^-17 of the terms for scores, exponentials and sums."""
    q, k, v, table, dout = _tensors(2, sq, sq, hq, hkv, d, buckets, table_dtype=torch.float32)
    out = _call(q, k, v, table, d ** -0.5, max_distance, window=window)
    got = torch.autograd.grad(out, (q, k, v, table), dout)[3]
    values, _, _ = oracle(q, k, v, dout, d ** -0.5, window=window, table=table, max_distance=max_distance)
    g, kh, vh = dout.double().transpose(1, 2), k.detach().double().transpose(1, 2), v.detach().double().transpose(1, 2)
    kh, vh = (t.repeat_interleave(hq // hkv, 1) for t in (kh, vh))
    at = (torch.arange(sq)[:, None] - torch.arange(sq)[None, :]).clamp(min=0)
    at = torch.tensor([bucket(n, buckets, max_distance) for n in range(sq)])[at].cuda()
    see = visible(sq, sq, window, 0, 0, "cuda")
    x = (q.detach().double().transpose(1, 2) @ kh.transpose(2, 3)) * d ** -0.5 + table.detach().double()[:, at]
    p = torch.softmax(x.masked_fill(~see, -math.inf), -1)
    size = g.abs() @ vh.abs().transpose(2, 3)              # of dP's sums
    per_row = (p * size).sum(-1, keepdim=True)             # of D's
    terms = p * (2.0 ** -16 * per_row + 2.0 ** -17 * (size + per_row))
    bound = torch.zeros_like(values["dtable"]).index_add_(1, at.flatten(), terms.sum(0).flatten(1))
    assert ((got.double() - values["dtable"]).abs() <= bound + 1e-30).all(), \
        f"{((got.double() - values['dtable']).abs() / (bound + 1e-30)).max().item():.2f} times what is allowed"


@pytest.mark.parametrize("sq,skv,hq,hkv,d,window,sinks,buckets", [
    (28, 50, 4, 4, 64, 2, 0, 0), (300, 300, 4, 2, 96, 40, 24, 0), (64, 64, 2, 1, 128, 1000, 0, 0), (257, 257, 2, 2, 64, 100, 3, 12)])
def test_output_over_few_keys_in_training(sq, skv, hq, hkv, d, window, sinks, buckets):
    """The weights have twice bf16's digits then, for the sake of the gradients: 2^-17 of sum_j P_j |V_j|, as much for what is
    held in fp32, and the result's own rounding are all that the output may be off."""
    q, k, v, table, _ = _tensors(2, sq, skv, hq, hkv, d, buckets)
    out = _call(q, k, v, table, d ** -0.5, 60, window=window, sinks=sinks, query_start=skv - sq)
    assert out.requires_grad
    values, bounds, _ = oracle(q, k, v, torch.zeros_like(q), d ** -0.5, window=window, sinks=sinks, start=skv - sq, table=table,
                               max_distance=60)
    half = torch.finfo(torch.bfloat16).eps / 2
    size = (bounds["out"] - half * values["out"].abs()) / (half + 2.0 ** -13)  # sum_j P_j |V_j|: the oracle's bound without its parts
    bound = half * values["out"].abs() + (1 + half) * 2.0 ** -16 * size
    assert ((out.double() - values["out"]).abs() <= bound).all()


@pytest.mark.parametrize("sq,h,window,sinks", [(65536, 16, 64, 65536), (65536, 128, 64, 128), (16384, 64, 1024, 16384), (8192, 2, 1024, 16)])
def test_scratch_stays_small(sq, h, window, sinks):
    """Key tiles are cut where SMs would be idle, not where there are enough of them: pieces of 128 x (dK, dV) in fp32."""
    from nano_megatron_b200.ops import native

    args = _Args(B=1, Hq=h, Hkv=h, Sq=sq, Skv=sq, d=128, window=window, sinks=sinks, scale=1.0)
    floats = native.lib().nmb_band_bwd_scratch(ctypes.byref(args))
    stats = h * (sq // 128) * 512
    assert stats <= floats <= stats + 16 * 148 * 128 * 256
    if h * sq // 128 >= 16 * 148:
        assert floats == stats or sinks < sq, "more key tiles than 16 for each SM are not cut"


def test_refusals_where_the_kernels_run():
    from nano_megatron_b200.ops.band_attention import relative_bias_attention, window_attention

    q, k, v, table, _ = _tensors(1, 70, 70, 4, 2, 64, 8)
    window_attention(q, k, v, 0.125, window=9)  # the operator is there: what follows is looked at from C++ first
    for kw, error in ((dict(window=0), ValueError), (dict(window=2.0), TypeError), (dict(window=True), TypeError),
                      (dict(window=3, sinks=-1), ValueError), (dict(window=3, query_start=-1), ValueError),
                      (dict(window=3, query_start=2 ** 30), ValueError), (dict(window=2 ** 40), ValueError)):
        with pytest.raises(error):
            window_attention(q, k, v, 0.125, **kw)
    for scale in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(ValueError):
            window_attention(q, k, v, scale, window=3)
    for bad in ((q[0], k, v), (q, k, v[:, :3]), (q[..., :32], k, v), (q[:, :, :3], k, v), (q.float(), k, v), (q, k.cpu(), v.cpu()),
                (q.expand(2, -1, -1, -1), k, v), (q, k[:, :, :0], v[:, :, :0])):
        with pytest.raises(ValueError):
            window_attention(*bad, 0.125, window=2)
    for bad in (table[:2], table[0], table[:, :1], table.cpu(), table.half(), torch.zeros(4, 129, device="cuda")):
        with pytest.raises(ValueError):
            relative_bias_attention(q, k, v, bad, 0.125)
    for distance, error in ((4, ValueError), (2049, ValueError), (8.0, TypeError)):
        with pytest.raises(error):
            relative_bias_attention(q, k, v, table, 0.125, max_distance=distance)
    for empty in (q[:0], q[:, :0]):
        assert window_attention(empty, k[:empty.shape[0]], v[:empty.shape[0]], 0.125, window=3).shape == empty.shape
    assert (window_attention(q, k[:, :0], v[:, :0], 0.125, window=3) == 0).all()


@pytest.mark.parametrize("b,sq,skv,hq,hkv,d,window,sinks,start,buckets", [
    (1, 1, 8192, 4, 2, 64, 10 ** 6, 0, 8191, 0), (2, 3, 5000, 2, 1, 128, 3000, 130, 4990, 0), (1, 130, 2500, 2, 2, 96, None, 0, 2370, 32),
    (1, 300, 4100, 3, 1, 64, 1500, 700, 3800, 16), (1, 1100, 1100, 1, 1, 128, None, 0, 0, 8), (1, 200, 3000, 2, 1, 96, 1100, 5, 2950, 0),
    (1, 150, 2000, 2, 2, 64, 1200, 0, 3100, 0)])
def test_few_rows_over_many_keys(b, sq, skv, hq, hkv, d, window, sinks, start, buckets):
    """Cut into pieces of the keys, which are joined: also pieces that some rows, or all of them, see nothing of."""
    from nano_megatron_b200.ops import native

    args = _Args(B=b, Hq=hq, Hkv=hkv, Sq=sq, Skv=skv, d=d, q_pos0=start, window=min(window or 2 ** 30, 2 ** 30), sinks=min(sinks, skv), scale=1.0)
    assert native.lib().nmb_band_fwd_scratch(ctypes.byref(args)) > 0
    tensors = _tensors(b, sq, skv, hq, hkv, d, buckets)
    _compare(*tensors, window=window, sinks=sinks, start=start)
    q, k, v, table, _ = tensors
    with torch.no_grad():
        one, two = (_call(q, k, v, table, 0.1, 128, window=window, sinks=sinks, query_start=start) for _ in range(2))
    assert torch.equal(one, two)


@pytest.mark.parametrize("seed", [0, 1])
@pytest.mark.parametrize("sq,skv,hq,hkv,d,window,buckets,max_distance", [
    (100, 3000, 4, 4, 128, None, 8, 60), (300, 2000, 8, 8, 96, None, 4, 20), (1024, 3000, 4, 2, 64, 1000, 24, 64)])
def test_gradient_of_the_last_bucket(sq, skv, hq, hkv, d, window, buckets, max_distance, seed):
    """The last bucket has nearly all keys of a row and the terms of its gradient cancel.  What is in the bf16 result besides its
    own rounding is no larger than that: sqrt(2) of it in all, since the two are independent."""
    start = skv - sq
    q, k, v, table, dout = _tensors(1, sq, skv, hq, hkv, d, buckets, seed=seed)
    out = _call(q, k, v, table, d ** -0.5, max_distance, window=window, query_start=start)
    got = torch.autograd.grad(out, (q, k, v, table), dout)[3].double()
    want = oracle(q, k, v, dout, d ** -0.5, window=window, start=start, table=table, max_distance=max_distance)[0]["dtable"]
    rounding = (want.to(torch.bfloat16).double() - want).norm()
    assert (got - want).norm() <= math.sqrt(2) * rounding, f"{((got - want).norm() / rounding).item():.2f} times its rounding"
