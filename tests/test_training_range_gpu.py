"""Attention gradients away from the ordinary: scalings of any sign and size, fp16 values near the type's ends, rows of very
different magnitude."""
import pytest
import torch

import nestedtensor_b200 as nt
import _training_reference as ref
from _helpers import stream_ptr
from nestedtensor_b200 import _cabi
from nestedtensor_b200.nn import training

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _rows(n, width, dtype, gen):
    return torch.randn(n, width, generator=gen).to(dtype).cuda()


def _inputs(lq, lk, heads, d, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    E = heads * d
    return (_rows(sum(lq), E, dtype, gen), _rows(sum(lk), E, dtype, gen), _rows(sum(lk), E, dtype, gen), _rows(sum(lq), E, dtype, gen))


def _nested(x, lengths):
    return nt.NestedTensor(x.view(-1), torch.tensor([[n, x.size(1)] for n in lengths]))


def _self(q, k, v, g, lengths, heads, scaling=None):
    qkv = torch.cat([q, k, v], 1).requires_grad_()
    y = training.self_attention(_nested(qkv, lengths), heads, scaling).values()
    grad, = torch.autograd.grad(y, [qkv], g)
    return dict(zip(("out", "dq", "dk", "dv"), (y, *grad.split(q.size(1), 1))))


def _cross(q, k, v, g, lq, lk, heads, scaling=None):
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    y = training.attention(_nested(q, lq), _nested(k, lk), _nested(v, lk), heads, scaling).values()
    return dict(zip(("out", "dq", "dk", "dv"), (y, *torch.autograd.grad(y, [q, k, v], g))))


def _check(got, want, bound, what):
    for name in want:
        ref.assert_within(got[name], want[name], bound[name], "%s %s" % (what, name))


# no score counts, the largest score counts least, and powers of two that fp32 products flush to zero
@pytest.mark.parametrize("scaling", [0.0, -0.2, -2.0 ** -130, 2.0 ** -130, 2.0 ** -100])
@pytest.mark.parametrize("d", [32, 64, 80, 128])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_attention_scaling_of_any_sign(cuda_device, dtype, d, scaling):
    nt.device_error_flags()
    for lengths in ([1, 17, 5, 30], [50, 0, 130, 9, 600]):
        q, k, v, g = _inputs(lengths, lengths, 2, d, dtype, d)
        want, bound = ref.attention(q, k, v, g, lengths, lengths, 2, scaling)
        _check(_self(q, k, v, g, lengths, 2, scaling), want, bound, "self")
        lk = lengths[::-1]
        q, k, v, g = _inputs(lengths, lk, 2, d, dtype, d + 1)
        want, bound = ref.attention(q, k, v, g, lengths, lk, 2, scaling)
        _check(_cross(q, k, v, g, lengths, lk, 2, scaling), want, bound, "cross")
    assert nt.device_error_flags() == 0


@pytest.mark.parametrize("scaling", [0.0, -0.2, 2.0 ** -130])
@pytest.mark.parametrize("d", [32, 64, 80, 128])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_inference_attention_scaling_of_any_sign(cuda_device, dtype, d, scaling):
    lib, heads, code = _cabi.load(), 2, {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype]
    E = heads * d
    for lengths in ([1, 17, 5, 30], [50, 0, 130, 9, 600]):
        T, B = sum(lengths), len(lengths)
        q, k, v, g = _inputs(lengths, lengths, heads, d, dtype, d)
        qkv, out, crossed = torch.cat([q, k, v], 1), torch.empty_like(q), torch.empty_like(q)
        off = (torch.tensor([0] + lengths).cumsum(0) * E).cuda()
        n = lib.ntb200_varlen_attention_workspace_bytes(B, T, heads, d, code)
        ws = torch.empty(n + 16, dtype=torch.uint8, device="cuda")
        _cabi.check("self", lib.ntb200_varlen_attention(qkv.data_ptr(), out.data_ptr(), off.data_ptr(), B, T, heads, d, max(lengths), scaling,
                                                        code, 0, ws.data_ptr(), n, stream_ptr()))
        _cabi.check("cross", lib.ntb200_varlen_cross_attention_ws(
            q.data_ptr(), E, k.data_ptr(), E, v.data_ptr(), E, crossed.data_ptr(), off.data_ptr(), off.data_ptr(), B, T, T, heads, d, max(lengths),
            scaling, code, 0, ws.data_ptr(), n, stream_ptr()))
        want, bound = ref.attention(q, k, v, g, lengths, lengths, heads, scaling)
        for name, got in (("self", out), ("cross", crossed)):
            ref.assert_within(got, want["out"], bound["out"], name)
