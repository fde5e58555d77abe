"""Calls that the kernels must not be launched for: tensors without memory, traces, null addresses."""
from __future__ import annotations

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from nano_megatron_b200.ops import native
from nano_megatron_b200.ops.band_attention import relative_bias_attention, window_attention

needs_library = pytest.mark.skipif(not native.available(), reason="the kernel library is not built")


def _fake(grad=False):
    q = torch.empty(2, 40, 2, 64, device="cuda", dtype=torch.bfloat16)
    return q.requires_grad_() if grad else q


@pytest.mark.parametrize("grad", [False, True])
def test_fake_tensors_are_refused(grad):
    with FakeTensorMode():
        q = _fake(grad)
        with pytest.raises(NotImplementedError, match="traced"):
            window_attention(q, q, q, 0.125, window=9)
        with pytest.raises(NotImplementedError, match="traced"):
            relative_bias_attention(q, q, q, torch.empty(2, 8, device="cuda"), 0.125)
    with pytest.raises(NotImplementedError, match="traced"):  # outside of the mode that made it
        window_attention(q, q, q, 0.125, window=9)


@needs_library
def test_the_operator_refuses_fake_tensors_before_it_looks_at_them():
    op = native.torch_lib().band_attention
    with FakeTensorMode():
        q = _fake()
        with pytest.raises(NotImplementedError, match="traced"):
            op(q, q, q, None, 0.125, 9, 0, 0, 0)
    with pytest.raises(NotImplementedError, match="traced"):
        op(q, q, q, None, 0.125, 9, 0, 0, 0)


def test_tensors_without_a_device_take_the_expression():
    q = torch.empty(2, 40, 2, 64, device="meta", dtype=torch.bfloat16)
    assert window_attention(q, q, q, 0.125, window=9).shape == q.shape


@needs_library
def test_null_addresses_end_in_a_code():
    from tests.test_gpu_band_attention import _Args, _Stride, _TENSORS

    lib = native.lib()
    buffer = torch.zeros(4096)  # host memory: no call below gets as far as a launch
    address = (buffer.data_ptr() + 63) // 64 * 64
    stride = _Stride(128, 64, 64)

    def args(**kw):
        every = dict.fromkeys(("q", "k", "v", "o", "dout", "dq", "dk", "dv", "m", "l", "scratch"), address)
        a = _Args(**{**every, "B": 1, "Hq": 1, "Hkv": 1, "Sq": 2, "Skv": 2, "d": 64, "window": 2, "scale": 1.0, **kw})
        for n in _TENSORS:
            setattr(a, n + "_st", stride)
        return ctypes.byref(a)

    for n in ("q", "k", "v", "o"):
        assert lib.nmb_band_fwd(args(**{n: None}), None) != 0 and lib.nmb_band_bwd(args(**{n: None}), None) != 0
    assert lib.nmb_band_fwd(args(l=None), None) != 0 and lib.nmb_band_fwd(args(rest_rows=1), None) != 0
    assert lib.nmb_band_fwd(args(rest_rows=3, o_rest=address), None) != 0
    for n in ("dout", "dq", "dk", "dv", "m", "scratch"):
        assert lib.nmb_band_bwd(args(**{n: None}), None) != 0
    assert lib.nmb_band_bwd(args(dtable=address), None) != 0
    assert lib.nmb_band_bwd_scratch(args()) >= 512  # where there is no GPU, too


@pytest.mark.gpu
def test_traces_are_refused_after_an_ordinary_call():
    from torch.fx.experimental.proxy_tensor import make_fx

    q = torch.randn(2, 40, 2, 64, device="cuda").to(torch.bfloat16)
    table = torch.zeros(2, 8, device="cuda")
    want = window_attention(q, q, q, 0.125, window=9)
    relative_bias_attention(q, q, q, table, 0.125)
    with pytest.raises(NotImplementedError, match="traced"):
        make_fx(lambda t: window_attention(t, t, t, 0.125, window=9))(q)
    with FakeTensorMode(allow_non_fake_inputs=True):
        for grad in (False, True):
            fake = _fake(grad)
            with pytest.raises(NotImplementedError, match="traced"):
                relative_bias_attention(fake, fake, fake, table, 0.125)
        wide = torch.empty(2, 40, 2, 64, device="cuda")  # not for the kernels: the expression
        assert window_attention(wide, wide, wide, 0.125, window=9).shape == wide.shape
    apart = torch.compiler.disable(window_attention)
    assert torch.equal(torch.compile(lambda t: apart(t, t, t, 0.125, window=9) * 2, backend="eager")(q), want * 2)
