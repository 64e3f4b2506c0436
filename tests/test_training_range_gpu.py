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


def _half_steps(q, k, v, g, lq, lk, heads, scaling):
    """What the last place of a subnormal fp16 dS may add to dQ and dK: dS is held relative to a power of two that brings R = max|dO_i|
    max|V_j| (2-norms, of the sequence and head) to (2^15, 2^16], so half a step of 2^-24 is at most R 2^-40."""
    d = q.size(1) // heads
    extra = {"dq": torch.zeros(q.shape, dtype=torch.float64, device=q.device), "dk": torch.zeros(k.shape, dtype=torch.float64, device=q.device)}
    a = c = 0
    for n, m in zip(lq, lk):
        rows, cols = slice(a, a + n), slice(c, c + m)
        a, c = a + n, c + m
        if n == 0 or m == 0:
            continue
        Q, G = (t[rows].double().view(n, heads, d) for t in (q, g))
        K, V = (t[cols].double().view(m, heads, d) for t in (k, v))
        R = G.norm(dim=2).amax(0) * V.norm(dim=2).amax(0)
        e = (abs(scaling) * R * 2.0 ** -40)[None, :, None]
        extra["dq"][rows] = (e * K.abs().sum(0)).expand(n, heads, d).reshape(n, -1)
        extra["dk"][cols] = (e * Q.abs().sum(0)).expand(m, heads, d).reshape(m, -1)
    return extra


# each kernel's range of lengths: mma.sync, whole sequences, tiles
@pytest.mark.parametrize("lengths", [[40, 3, 64], [130, 20, 500], [700, 33]], ids=str)
@pytest.mark.parametrize("d", [32, 64, 72, 128])
def test_attention_fp16_large_values(cuda_device, d, lengths):
    """|V| near fp16's largest against small dO that lie along single rows of it: dO . V is in the millions relative to the largest
    |dO|, dQ and dK are ordinary."""
    H, gen = 2, torch.Generator().manual_seed(d)
    q, k, v, g = _inputs(lengths, lengths, H, d, torch.float16, d)
    v = (torch.sign(v.float()) * 30000).half()
    pick = torch.cat([torch.randint(0, n, (n,), generator=gen) + sum(lengths[:i]) for i, n in enumerate(lengths)]).cuda()
    g = (torch.sign(v[pick].float()) * 1e-3).half()
    scaling = d ** -0.5
    want, bound = ref.attention(q, k, v, g, lengths, lengths, H, scaling)
    for name, e in _half_steps(q, k, v, g, lengths, lengths, H, scaling).items():
        bound[name] = bound[name] + e
        assert float(want[name].abs().max()) < 30000
    _check(_self(q, k, v, g, lengths, H), want, bound, "large values")


@pytest.mark.parametrize("lengths", [[40, 3, 64], [130, 20, 500], [700, 33]], ids=str)
@pytest.mark.parametrize("d", [32, 64, 72, 128])
def test_attention_fp16_rows_of_different_magnitude(cuda_device, d, lengths):
    """Rows of dO from 2^8 down to 2^-8 of the ordinary in one sequence: dQ of a row is linear in the row's dO, and is held as well as
    that of a row among its like."""
    H = 2
    q, k, v, g = _inputs(lengths, lengths, H, d, torch.float16, d + 7)
    g = torch.where(g < 0, g - 1, g + 1)  # (at least 1: the powers of two below stay exact)
    scaling = d ** -0.5
    want, bound = ref.attention(q, k, v, g, lengths, lengths, H, scaling)
    s = torch.pow(2.0, torch.arange(g.size(0), device="cuda") * 5 % 17 - 8).double()[:, None]
    scaled = (g.double() * s).half()
    assert torch.equal(scaled.double(), g.double() * s)
    got = _self(q, k, v, scaled, lengths, H)
    extra = _half_steps(q, k, v, scaled, lengths, lengths, H, scaling)["dq"]
    ref.assert_within(got["dq"], want["dq"] * s, bound["dq"] * s + extra + ref.tiny(torch.float16), "dq")
    want, bound = ref.attention(q, k, v, scaled, lengths, lengths, H, scaling)
    _check({n: got[n] for n in ("dk", "dv")}, {n: want[n] for n in ("dk", "dv")}, bound, "all rows")


@pytest.mark.parametrize("lengths", [[40, 3, 64], [130, 20, 500], [700, 33]], ids=str)
@pytest.mark.parametrize("d", [32, 64, 128])
def test_attention_fp16_one_row_of_no_number(cuda_device, d, lengths):
    """A row of dO that holds Inf or NaN is lost, and with it its sequence's dK and dV; the small gradients of the other rows are not."""
    H = 2
    q, k, v, g = _inputs(lengths, lengths, H, d, torch.float16, d + 9)
    g = torch.where(g < 0, g - 1, g + 1) * 2.0 ** -12
    scaling = d ** -0.5
    want, bound = ref.attention(q, k, v, g * 2.0 ** 12, lengths, lengths, H, scaling)
    for bad in (float("inf"), float("nan")):
        g2 = g.clone()
        g2[::37] = bad
        rows = torch.ones(g.size(0), dtype=torch.bool, device="cuda")
        rows[::37] = False
        got = _self(q, k, v, g2, lengths, H)
        extra = _half_steps(q, k, v, g, lengths, lengths, H, scaling)["dq"]
        s = 2.0 ** -12
        ref.assert_within(got["dq"][rows], (want["dq"] * s)[rows], (bound["dq"] * s + extra + ref.tiny(torch.float16))[rows], "dq")


@pytest.mark.parametrize("d", [32, 64, 80, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16], ids=str)
def test_attention_row_statistics_hold_32_bits(cuda_device, dtype, d):
    """The base-2 logarithm of a row's softmax denominator where the scores are exact: one key at 0, the others all at -c / 128, for
    every c up to d.  Exponentials are off by 2^-22, their sum by 2^-24 a term."""
    lib, code = _cabi.load(), {torch.float32: 0, torch.float16: 1}[dtype]
    lengths = [33, 100, 130]
    T, B = sum(lengths), len(lengths)
    q = torch.eye(d, dtype=dtype, device="cuda")[torch.arange(T, device="cuda") % d].contiguous()
    k = (torch.arange(d, device="cuda") / -128).to(dtype).expand(T, d).contiguous()
    for i in range(B):
        k[sum(lengths[:i])] = 0
    v = torch.ones(T, d, dtype=dtype, device="cuda")
    out, lse = torch.empty_like(q), torch.empty(1, T, device="cuda")
    off = torch.tensor([0] + lengths).cumsum(0).cuda()
    n = lib.ntb200_varlen_attention_train_workspace_bytes(B, T, 1, d, code)
    ws = torch.empty(n + 16, dtype=torch.uint8, device="cuda")
    _cabi.check("train", lib.ntb200_varlen_attention_train(
        q.data_ptr(), d, k.data_ptr(), d, v.data_ptr(), d, out.data_ptr(), lse.data_ptr(), off.data_ptr(), 1, off.data_ptr(), 1, B, T, T, 1, d,
        max(lengths), 1.0, code, 0, ws.data_ptr(), n, stream_ptr()))
    a = 0
    for m in lengths:
        S = q[a:a + m].double() @ k[a:a + m].double().t()
        want = torch.logsumexp(S, 1) / 0.6931471805599453
        # exponents of at most 1.45 after two roundings, exponentials, m additions: as parts of the denominator, times log2(e); the
        # logarithm and the sum with the row's maximum
        bound = (3 * 1.45 + 4 + m) * ref.W * 1.45 + 4 * ref.W * want.abs()
        off_by = (lse[0, a:a + m].double() - want).abs()
        assert bool((off_by <= bound).all()), (m, float((off_by / bound).max()), int((off_by / bound).argmax()))
        a += m
