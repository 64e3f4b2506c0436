"""Gradients of the training operators (nn.training) against plain 64-bit forms, within bounds derived from the roundings
(_training_reference), their bit-for-bit repeatability, and their use together, on streams and in captured graphs."""
import math

import pytest
import torch

import nestedtensor_b200 as nt
import _training_reference as ref
from _helpers import stream_ptr
from nestedtensor_b200 import _cabi
from nestedtensor_b200.nn import training

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _ragged(lengths, features, dtype, gen, std=1.0):
    x = (torch.randn(sum(lengths), features, generator=gen) * std).to(dtype).cuda()
    sizes = torch.tensor([[n, features] for n in lengths], dtype=torch.int64).reshape(len(lengths), 2)
    return x, sizes


def _nested(x, sizes):
    return nt.NestedTensor(x.view(-1), sizes)


def _check(got, want, bound, what):
    for name in want:
        ref.assert_within(got[name], want[name], bound[name], "%s %s" % (what, name))


# ------------------------------------------------------------------ layer norm
def _run_norm(x, sizes, w, b, g, eps=1e-5):
    leaves = [t.detach().requires_grad_() for t in (x, w, b) if t is not None]
    y = training.layer_norm(_nested(leaves[0], sizes), (x.size(1),), *(leaves[1:] or (None, None)), eps).values()
    grads = torch.autograd.grad(y, leaves, g)
    return dict(zip(("out", "dx", "dweight", "dbias"), (y, *grads)))


# whole 16-byte vectors: rows on 8, 16, 32 threads, a warp with 2 to 4 vectors a thread, blocks of 64 to 256 threads, and beyond; odd
# widths on single elements; the widest that neither holds in registers
@pytest.mark.parametrize("features", [1, 7, 8, 64, 72, 128, 250, 256, 333, 512, 771, 768, 1000, 1001, 1024, 1536, 2048, 2055, 4096, 4100, 6144,
                                      8192, 8200, 16384])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_layer_norm_gradients(cuda_device, dtype, features):
    gen = torch.Generator().manual_seed(features)
    lengths = [3, 0, 17, 1, 40] if features < 4096 else [2, 3]
    x, sizes = _ragged(lengths, features, dtype, gen, 2.0)
    x = x + 0.5
    w, b = (1 + 0.2 * torch.randn(features, generator=gen)).to(dtype).cuda(), torch.randn(features, generator=gen).to(dtype).cuda()
    g = torch.randn(x.shape, generator=gen).to(dtype).cuda()
    want, bound = ref.layer_norm(x, w, b, g, 1e-5)
    _check(_run_norm(x, sizes, w, b, g), want, bound, "affine")
    want, bound = ref.layer_norm(x, None, None, g, 1e-5)
    del want["dweight"], want["dbias"]
    _check(_run_norm(x, sizes, None, None, g), want, bound, "plain")


@pytest.mark.parametrize("rows", [0, 1, 2, 9, 1185, 5000])
def test_layer_norm_row_counts(cuda_device, rows):
    """Fewer rows than a block holds, and more than all resident blocks hold at once; no rows: zero column sums."""
    gen = torch.Generator().manual_seed(rows)
    x, sizes = _ragged([rows // 2, rows - rows // 2], 256, torch.bfloat16, gen)
    w, b = torch.randn(256, generator=gen).bfloat16().cuda(), torch.randn(256, generator=gen).bfloat16().cuda()
    g = torch.randn(x.shape, generator=gen).bfloat16().cuda()
    want, bound = ref.layer_norm(x, w, b, g, 1e-5)
    _check(_run_norm(x, sizes, w, b, g), want, bound, "%d rows" % rows)


def test_layer_norm_only_wanted_gradients(cuda_device):
    gen = torch.Generator().manual_seed(1)
    x, sizes = _ragged([5, 9], 64, torch.float32, gen)
    w, b = torch.randn(64, generator=gen).cuda(), torch.randn(64, generator=gen).cuda()
    g = torch.randn(x.shape, generator=gen).cuda()
    full = _run_norm(x, sizes, w, b, g)
    for which in range(3):
        leaves = [t.detach().requires_grad_(i == which) for i, t in enumerate((x, w, b))]
        y = training.layer_norm(_nested(leaves[0], sizes), 64, leaves[1], leaves[2]).values()
        got, = torch.autograd.grad(y, [leaves[which]], g)
        assert torch.equal(got, full[("dx", "dweight", "dbias")[which]])


def test_layer_norm_unaligned_buffer_and_expanded_gradient(cuda_device):
    gen = torch.Generator().manual_seed(2)
    base = torch.randn(10 * 64 + 1, generator=gen).half().cuda()
    x = base[1:].view(10, 64)  # whole vectors, but no 16-byte boundary
    sizes = torch.tensor([[4, 64], [6, 64]])
    w, b = torch.randn(64, generator=gen).half().cuda(), torch.randn(64, generator=gen).half().cuda()
    g = torch.randn(1, 64, generator=gen).half().cuda().expand(10, 64)
    want, bound = ref.layer_norm(x, w, b, g, 1e-5)
    _check(_run_norm(x, sizes, w, b, g), want, bound, "unaligned")


# ------------------------------------------------------------------ embedding
def _run_embed(weight, index, lengths, g, **kw):
    weight = weight.detach().requires_grad_()
    sizes = torch.tensor(lengths, dtype=torch.int64).reshape(-1, 1)
    y = training.embedding(nt.NestedTensor(index, sizes), weight, **kw).values()
    dw, = torch.autograd.grad(y, [weight], g)
    return dict(out=y, dweight=dw)


@pytest.mark.parametrize("features", [1, 8, 40, 64, 129, 256, 333, 512, 768, 1000, 1024, 2056])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_embedding_gradient(cuda_device, dtype, features):
    gen = torch.Generator().manual_seed(features)
    lengths, vocab = [30, 0, 1, 170], 50
    T = sum(lengths)
    index = torch.where(torch.rand(T, generator=gen) < 0.5, torch.full((T,), 7), torch.randint(0, vocab, (T,), generator=gen)).cuda()
    weight = torch.randn(vocab, features, generator=gen).to(dtype).cuda()
    g = torch.randn(T, features, generator=gen).to(dtype).cuda()
    for scale, pad in ((1.0, None), (math.sqrt(features), 7), (0.3, -1)):
        want, bound = ref.embedding(weight, index, g, scale, None if pad is None else pad % vocab)
        got = _run_embed(weight, index, lengths, g, padding_idx=pad, scale=scale)
        _check(got, want, bound, "scale %g padding %s" % (scale, pad))
    assert torch.equal(got["dweight"], _run_embed(weight, index.int(), lengths, g, padding_idx=pad, scale=scale)["dweight"])


# one and several sorting blocks; tables of 1 to 4 passes; runs over many warps, none, all the same token
@pytest.mark.parametrize("tokens", [1, 31, 32, 33, 4096, 4097, 70000])
@pytest.mark.parametrize("vocab", [1, 2, 511, 512, 70000, 300000])
def test_embedding_token_counts_and_tables(cuda_device, tokens, vocab):
    gen = torch.Generator().manual_seed(tokens * 7 + vocab)
    index = torch.clamp((torch.rand(tokens, generator=gen) ** 6 * vocab).long(), max=vocab - 1).cuda()
    weight = torch.randn(vocab, 16, generator=gen).cuda()
    g = torch.randn(tokens, 16, generator=gen).cuda()
    want, bound = ref.embedding(weight, index, g, 2.0, None)
    got = _run_embed(weight, index, [tokens], g, scale=2.0)
    _check(got, want, bound, "embedding")
    assert torch.equal(got["dweight"], _run_embed(weight, index, [tokens], g, scale=2.0)["dweight"])


def test_embedding_out_of_range_index(cuda_device):
    nt.device_error_flags()
    gen = torch.Generator().manual_seed(3)
    weight = torch.randn(10, 64, generator=gen).cuda()
    index = torch.tensor([3, -1, 10, 3, 1 << 40, 9]).cuda()
    g = torch.randn(6, 64, generator=gen).cuda()
    for scale in (1.0, 2.0):
        want, bound = ref.embedding(weight, index, g, scale, None)
        _check(_run_embed(weight, index, [2, 4], g, scale=scale), want, bound, "out of range")
        assert nt.device_error_flags() == 1 << 16


def test_embedding_no_tokens(cuda_device):
    weight = torch.randn(10, 64).cuda()
    got = _run_embed(weight, torch.empty(0, dtype=torch.int64).cuda(), [0, 0], torch.empty(0, 64).cuda())
    assert got["out"].shape == (0, 64) and torch.equal(got["dweight"], torch.zeros_like(weight))


# ------------------------------------------------------------------ attention
def _attend_inputs(lq, lk, heads, d, dtype, seed, gstd=1.0):
    gen = torch.Generator().manual_seed(seed)
    E = heads * d
    q, qs = _ragged(lq, E, dtype, gen)
    k, ks = _ragged(lk, E, dtype, gen)
    v, _ = _ragged(lk, E, dtype, gen)
    g = (torch.randn(q.shape, generator=gen) * gstd).to(dtype).cuda()
    return q, k, v, g, qs, ks


def _run_attend(q, k, v, g, qs, ks, heads, scaling=None):
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    y = training.attention(_nested(q, qs), _nested(k, ks), _nested(v, ks), heads, scaling).values()
    return dict(zip(("out", "dq", "dk", "dv"), (y, *torch.autograd.grad(y, [q, k, v], g))))


def _run_self(q, k, v, g, qs, heads, scaling=None):
    qkv = torch.cat([q, k, v], 1).requires_grad_()
    sizes = qs.clone()
    sizes[:, 1] *= 3
    y = training.self_attention(_nested(qkv, sizes), heads, scaling).values()
    grad, = torch.autograd.grad(y, [qkv], g)
    return dict(zip(("out", "dq", "dk", "dv"), (y, *grad.split(q.size(1), 1))))


@pytest.mark.parametrize("d", [1, 5, 16, 32, 64, 80, 128, 200, 256])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_attention_gradients_head_sizes(cuda_device, dtype, d):
    lq, heads = [1, 33, 0, 70, 129], 2
    q, k, v, g, qs, _ = _attend_inputs(lq, lq, heads, d, dtype, d)
    want, bound = ref.attention(q, k, v, g, lq, lq, heads, d ** -0.5)
    _check(_run_self(q, k, v, g, qs, heads), want, bound, "self")
    lk = [40, 1, 5, 0, 260]
    q, k, v, g, qs, ks = _attend_inputs(lq, lk, heads, d, dtype, d + 1)
    want, bound = ref.attention(q, k, v, g, lq, lk, heads, d ** -0.5)
    _check(_run_attend(q, k, v, g, qs, ks, heads), want, bound, "cross")


# tile borders of every kernel: 16, 32, 64, 128 rows and one more or less, lengths of zero and one, several tiles
@pytest.mark.parametrize("lengths", [[1], [2, 15, 16, 17], [31, 32, 33, 0], [63, 64, 65], [127, 128, 129], [255, 256, 257], [640, 1], [0, 0, 3],
                                     [383, 511, 700]], ids=str)
@pytest.mark.parametrize("dtype,d", [(torch.float32, 64), (torch.float16, 64), (torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float16, 128),
                                     (torch.float16, 32)], ids=str)
def test_attention_gradients_lengths(cuda_device, dtype, d, lengths):
    q, k, v, g, qs, _ = _attend_inputs(lengths, lengths, 3, d, dtype, len(lengths))
    want, bound = ref.attention(q, k, v, g, lengths, lengths, 3, d ** -0.5)
    got = _run_self(q, k, v, g, qs, 3)
    _check(got, want, bound, "self")
    again = _run_self(q, k, v, g, qs, 3)
    assert all(torch.equal(got[n], again[n]) for n in got)
    lk = lengths[::-1]
    q, k, v, g, qs, ks = _attend_inputs(lengths, lk, 3, d, dtype, 1 + len(lengths))
    want, bound = ref.attention(q, k, v, g, lengths, lk, 3, d ** -0.5)
    _check(_run_attend(q, k, v, g, qs, ks, 3), want, bound, "cross")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_attention_one_side_empty(cuda_device, dtype):
    """Queries without keys, keys without queries: zeros, whatever was in the memory before."""
    for lq, lk in (([3, 0, 40], [0, 7, 0]), ([0, 0], [5, 200]), ([5, 200], [0, 0])):
        q, k, v, g, qs, ks = _attend_inputs(lq, lk, 2, 64, dtype, 5)
        junk = [torch.full((1 << 20,), float("nan"), device="cuda") for _ in range(4)]
        del junk
        got = _run_attend(q, k, v, g, qs, ks, 2)
        for name, t in got.items():
            assert torch.equal(t, torch.zeros_like(t)), name


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_attention_does_not_mix_sequences(cuda_device, dtype, d):
    """NaN and Inf in one sequence stay there, and the others' gradients have the bits they have alone."""
    lengths, H = [20, 33, 130, 77, 530, 9], 2
    q, k, v, g, qs, _ = _attend_inputs(lengths, lengths, H, d, dtype, 6)
    clean = _run_self(q, k, v, g, qs, H)
    for bad in range(1, len(lengths)):
        a = sum(lengths[:bad])
        sl = slice(a, a + lengths[bad])
        q2, k2, v2, g2 = q.clone(), k.clone(), v.clone(), g.clone()
        q2[sl] = float("nan")
        k2[sl] = float("inf")
        v2[sl] = float("inf")
        g2[sl] = float("-inf")
        got = _run_self(q2, k2, v2, g2, qs, H)
        for name in got:
            for other in range(len(lengths)):
                o = sum(lengths[:other])
                part = slice(o, o + lengths[other])
                if other != bad:
                    assert torch.equal(got[name][part], clean[name][part]), (name, bad, other)
    # a batch cut in two reproduces the whole
    cut = lengths[0] + lengths[1]
    for rows, sizes in ((slice(0, cut), qs[:2]), (slice(cut, None), qs[2:])):
        part = _run_self(q[rows], k[rows], v[rows], g[rows], sizes.contiguous(), H)
        for name in part:
            assert torch.equal(part[name], clean[name][rows]), name


@pytest.mark.parametrize("d", [24, 32, 64, 128])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_attention_over_one_key_has_no_score_gradient(cuda_device, dtype, d):
    """The softmax of one score is 1 whatever the score is: dQ = dK = 0, up to what fp32 sums leave of dP - dP."""
    heads, lq = 3, [1, 90, 1, 300]
    q, k, v, g, qs, ks = _attend_inputs(lq, [1, 1, 1, 1], heads, d, dtype, 77)
    got = _run_attend(q, k, v, g, qs, ks, heads)
    want, bound = ref.attention(q, k, v, g, lq, [1, 1, 1, 1], heads, d ** -0.5)
    assert float(want["dq"].abs().max()) < 1e-12 and float(want["dk"].abs().max()) < 1e-12
    _check(got, want, bound, "one key")


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_attention_carries_nan(cuda_device, dtype, d):
    """One NaN query reaches its own output row and dQ row and, through its probabilities, every dK and dV row of its sequence
    and no other's, at every position in the kernels' tiles."""
    lengths, H = [40, 150], 1
    q, k, v, g, qs, _ = _attend_inputs(lengths, lengths, H, d, dtype, 16)
    for row in list(range(40, 56)) + [100, 167, 168, 189]:
        q2 = q.clone()
        q2[row] = float("nan")
        got = _run_self(q2, k, v, g, qs, H)
        for name in ("out", "dq"):
            bad = torch.isnan(got[name]).all(1)
            assert bool(bad[row]) and int(torch.isnan(got[name]).any(1).sum()) == 1, (name, row)
        for name in ("dk", "dv"):
            assert bool(torch.isnan(got[name][40:]).all()) and not bool(torch.isnan(got[name][:40]).any()), (name, row)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_attention_carries_nan_keys(cuda_device, dtype, d):
    """One NaN key makes every probability of its sequence and head NaN, at every position in the kernels' tiles, and no other's."""
    lengths = [40, 150]
    q, k, v, g, qs, _ = _attend_inputs(lengths, lengths, 2, d, dtype, 17)
    for row in list(range(40, 72)) + [100, 167, 168, 189]:
        k2 = k.clone()
        k2[row, :d] = float("nan")
        got = _run_self(q, k2, v, g, qs, 2)
        for name, t in got.items():
            assert bool(torch.isnan(t[40:, :d]).all()), (name, row)
            assert not bool(torch.isnan(t[:40]).any()) and not bool(torch.isnan(t[:, d:]).any()), (name, row)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_attention_large_logits_and_gradients(cuda_device, dtype):
    """Probabilities that are one or nothing; gradients under and over the ordinary (fp16: a loss scale's)."""
    lengths = [64, 190]
    q, k, v, g, qs, _ = _attend_inputs(lengths, lengths, 2, 64, dtype, 7)
    for scaling, factor in ((1.0, 1.0), (0.125, 500.0), (0.125, 1e-3)):
        gs = (g.float() * factor).to(dtype)
        want, bound = ref.attention(q, k, v, gs, lengths, lengths, 2, scaling)
        _check(_run_self(q, k, v, gs, qs, 2, scaling), want, bound, "scaling %g, gradients times %g" % (scaling, factor))


def _cabi_backward(q, k, v, g, lq, lk, heads, path, ld_extra=0):
    """Forward with row statistics and backward through the C ABI on one path, token offsets, gradients in wider rows."""
    lib, E, d = _cabi.load(), q.size(1), q.size(1) // heads
    code = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[q.dtype]
    off = [torch.tensor([0] + list(torch.tensor(n).cumsum(0))).cuda() for n in (lq, lk)]
    out, lse = torch.empty_like(q), torch.empty(heads, q.size(0), device="cuda")
    B, Tq, Tk, scaling = len(lq), q.size(0), k.size(0), d ** -0.5
    n = lib.ntb200_varlen_attention_train_workspace_bytes(B, Tq, heads, d, code)
    ws = torch.empty(n + 16, dtype=torch.uint8, device="cuda")
    _cabi.check("train", lib.ntb200_varlen_attention_train(
        q.data_ptr(), E, k.data_ptr(), E, v.data_ptr(), E, out.data_ptr(), lse.data_ptr(), off[0].data_ptr(), 1, off[1].data_ptr(), 1, B, Tq, Tk,
        heads, d, max(lq), scaling, code, min(path, 3), ws.data_ptr(), n, stream_ptr()))
    n = lib.ntb200_varlen_attention_backward_workspace_bytes(B, Tq, Tk, heads, d, max(lq), max(lk), code, path)
    ws = torch.full((n + 64,), 0xAB, dtype=torch.uint8, device="cuda")
    wide = E + ld_extra
    grads = [torch.full((t.size(0) + 3, wide), 7.0, dtype=q.dtype, device="cuda") for t in (q, k, v)]
    _cabi.check("backward", lib.ntb200_varlen_attention_backward(
        g.data_ptr(), q.data_ptr(), E, k.data_ptr(), E, v.data_ptr(), E, out.data_ptr(), lse.data_ptr(), grads[0].data_ptr(), wide,
        grads[1].data_ptr(), wide, grads[2].data_ptr(), wide, off[0].data_ptr(), 1, off[1].data_ptr(), 1, B, Tq, Tk, heads, d, max(lq), max(lk),
        scaling, code, path, ws.data_ptr(), n, stream_ptr()))
    torch.cuda.synchronize()
    assert bool((ws[n:] == 0xAB).all()), "workspace overrun"
    for t in grads:  # rows behind the last sequence and columns beside the heads are left as they were
        assert bool((t[-3:] == 7.0).all()) and bool((t[:, E:] == 7.0).all())
    assert lib.ntb200_device_error_flags() == 0
    return dict(zip(("out", "dq", "dk", "dv"), (out, *(t[:-3, :E] for t in grads))))


@pytest.mark.parametrize("path,dtype,d", [(1, torch.float32, 64), (1, torch.bfloat16, 64), (1, torch.float16, 72), (2, torch.float16, 32),
                                          (2, torch.bfloat16, 64), (2, torch.float16, 64), (2, torch.bfloat16, 128), (2, torch.float16, 128),
                                          (3, torch.bfloat16, 64), (3, torch.float16, 64), (3, torch.bfloat16, 128), (3, torch.float16, 128), (4, torch.bfloat16, 64),
                                          (4, torch.float16, 64)],
                         ids=str)
def test_attention_backward_paths(cuda_device, path, dtype, d):
    nt.device_error_flags()
    lq, lk = [1, 0, 64, 130, 300, 17], [5, 3, 0, 257, 129, 16]
    q, k, v, g, _, _ = _attend_inputs(lq, lk, 2, d, dtype, path + d)
    want, bound = ref.attention(q, k, v, g, lq, lk, 2, d ** -0.5)
    _check(_cabi_backward(q, k, v, g, lq, lk, 2, path, 24), want, bound, "path %d" % path)


@pytest.mark.parametrize("path,dtype,d", [(0, torch.float32, 64), (0, torch.float16, 24), (0, torch.float16, 64), (0, torch.bfloat16, 128),
                                          (2, torch.float16, 32), (3, torch.float16, 64), (4, torch.float16, 64), (4, torch.bfloat16, 64)], ids=str)
def test_attention_rows_behind_the_last_sequence(cuda_device, path, dtype, d):
    """Tokens that belong to no sequence hold anything: they are neither written nor do they reach a result (fp16: nor the power
    of two that dO is brought to)."""
    lq, lk = [70, 3, 200, 9], [65, 40, 140, 30]
    q, k, v, g, _, _ = _attend_inputs(lq + [50], lk + [50], 2, d, dtype, 31)
    for t in (q, k, v, g):
        t[-50:-25] = float("nan")
        t[-25:] = torch.finfo(dtype).max
    nq, nk = sum(lq), sum(lk)
    want, bound = ref.attention(q[:nq], k[:nk], v[:nk], g[:nq], lq, lk, 2, d ** -0.5)
    got = _cabi_backward(q, k, v, g, lq, lk, 2, path)
    for name, n in (("dq", nq), ("dk", nk), ("dv", nk)):
        assert bool((got[name][n:] == 7.0).all())
    _check({n: t[:nq if n in ("out", "dq") else nk] for n, t in got.items()}, want, bound, "path %d" % path)


@pytest.mark.parametrize("op", ["norm", "attend"])
def test_gradients_against_differences(cuda_device, op):
    """Directional derivative by central differences of the operator's own fp32 forward pass."""
    gen = torch.Generator().manual_seed(8)
    lengths = [9, 30]
    sizes = torch.tensor([[n, 96] for n in lengths])
    x = torch.randn(39, 96, generator=gen).cuda()
    w, b = torch.randn(96, generator=gen).cuda(), torch.randn(96, generator=gen).cuda()

    def f(t):
        if op == "norm":
            return training.layer_norm(_nested(t, sizes), 96, w, b).values()
        return training.self_attention(_nested(t, sizes), 2).values()

    leaf = x.clone().requires_grad_()
    y = f(leaf)
    g = torch.randn(y.shape, generator=gen).cuda()
    grad, = torch.autograd.grad(y, [leaf], g)
    for k in range(4):
        v = torch.randn(x.shape, generator=gen).cuda()
        h = 2.0 ** -7
        diff = ((f(x + h * v).double() - f(x - h * v).double()) * g.double()).sum() / (2 * h)
        got = (grad.double() * v.double()).sum()
        # truncation h^2/6 of a third derivative of order |g||v|^3 / sqrt(n) and fp32 rounding 2^-24 |y||g| / h, both with room
        assert abs(diff - got) <= 2e-3 * g.double().norm() * v.double().norm() / math.sqrt(96), (k, float(diff), float(got))


# ------------------------------------------------------------------ together
def _block(table, w_norm, b_norm, w_in, b_in, w_out, index, sizes, heads):
    E = table.size(1)
    x = training.embedding(nt.NestedTensor(index, sizes), table, padding_idx=0, scale=math.sqrt(E))
    h = training.layer_norm(x, (E,), w_norm, b_norm)
    qkv = h.with_values(torch.nn.functional.linear(h.values(), w_in, b_in))
    a = training.self_attention(qkv, heads)
    return x.values() + torch.nn.functional.linear(a.values(), w_out)


def _block_inputs(dtype, E=128, seed=9):
    gen = torch.Generator().manual_seed(seed)
    lengths = [5, 0, 40, 131, 1]
    index = torch.randint(0, 60, (sum(lengths),), generator=gen).cuda()
    sizes = torch.tensor(lengths).reshape(-1, 1)
    shapes = [(60, E), (E,), (E,), (3 * E, E), (3 * E,), (E, E)]
    params = [((torch.randn(s, generator=gen) * 0.1) + (1.0 if i == 1 else 0.0)).to(dtype).cuda().requires_grad_() for i, s in enumerate(shapes)]
    return params, index, sizes, lengths


def _plain_block(params, index, lengths, heads):
    table, w_norm, b_norm, w_in, b_in, w_out = params
    E = table.size(1)
    # (the padding row takes no gradient)
    x = torch.where((index == 0)[:, None], table[index].detach(), table[index]) * math.sqrt(E)
    qkv = torch.nn.functional.linear(torch.nn.functional.layer_norm(x, (E,), w_norm, b_norm), w_in, b_in)
    outs = []
    for part in qkv.split(lengths):
        q, k, v = (t.view(-1, heads, E // heads).transpose(0, 1) for t in part.split(E, 1))
        p = torch.softmax(q @ k.transpose(1, 2) * (E // heads) ** -0.5, 2)
        outs.append((p @ v).transpose(0, 1).reshape(-1, E))
    return x + torch.nn.functional.linear(torch.cat(outs), w_out)


def test_block_fp32_gradients(cuda_device):
    params, index, sizes, lengths = _block_inputs(torch.float32)
    y = _block(*params, index, sizes, 2)
    g = torch.randn(y.shape, generator=torch.Generator().manual_seed(1)).cuda()
    got = torch.autograd.grad(y, params, g)
    p64 = [p.detach().double().requires_grad_() for p in params]
    y64 = _plain_block(p64, index, lengths, 2)
    want = torch.autograd.grad(y64, p64, g.double())
    assert (y.double() - y64).abs().max() <= 1e-5 * y64.abs().max()
    for a, b in zip(got, want):  # chains of fp32 sums of at most a few hundred terms: 2^-24 * 500 of the largest
        assert (a.double() - b).abs().max() <= 500 * ref.W * b.abs().max()


def test_block_trains(cuda_device):
    params, index, sizes, _ = _block_inputs(torch.bfloat16)
    opt = torch.optim.SGD(params, lr=1e-3)
    for _ in range(3):
        opt.zero_grad()
        _block(*params, index, sizes, 2).float().square().mean().backward()
        assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in params)
        opt.step()


def test_block_in_a_captured_graph(cuda_device):
    """Forward and backward captured, replayed on other inputs: the bits of the eager pass, twice over, beside a second graph."""
    params, index, sizes, _ = _block_inputs(torch.bfloat16)
    inputs = nt.NestedTensor(index, sizes)
    inputs._row_offsets()  # the offsets are on the device before the capture
    g = torch.randn(index.numel(), 128, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()

    def step(idx):
        E = 128
        nested = nt.NestedTensor(idx, sizes, inputs._meta)
        x = training.embedding(nested, params[0], padding_idx=0, scale=math.sqrt(E))
        h = training.layer_norm(x, (E,), params[1], params[2])
        a = training.self_attention(h.with_values(torch.nn.functional.linear(h.values(), params[3], params[4])), 2)
        y = x.values() + torch.nn.functional.linear(a.values(), params[5])
        return (y.detach(), *torch.autograd.grad(y, params, g))

    static = index.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(static)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(static)
        graphs.append((graph, outs))
    for shift in (0, 7, 23):
        static.copy_((index + shift) % 60)
        want = step(static.clone())
        for graph, outs in graphs + graphs[::-1]:
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(outs, want):
                assert torch.equal(a, b)


def test_block_on_another_stream(cuda_device):
    params, index, sizes, _ = _block_inputs(torch.float16)
    g = torch.randn(index.numel(), 128, generator=torch.Generator().manual_seed(3)).half().cuda()
    y = _block(*params, index, sizes, 2)
    want = (y, *torch.autograd.grad(y, params, g))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for s in streams:  # two calls in flight at once
        with torch.cuda.stream(s):
            y = _block(*params, index, sizes, 2)
            got.append((y, *torch.autograd.grad(y, params, g)))
    torch.cuda.synchronize()
    for one in got:
        assert all(torch.equal(a, b) for a, b in zip(one, want))


def test_capture_beside_an_eager_graph_of_the_same_leaf(cuda_device):
    """Refused with an error, and the process, the eager graph and a capture without it go on."""
    sizes = torch.tensor([[3, 64], [5, 64]])
    x = torch.randn(8, 64, device="cuda")
    w, b = (torch.randn(64, device="cuda", requires_grad=True) for _ in range(2))
    nested = nt.NestedTensor(x.view(-1), sizes)
    g = torch.randn(8, 64, device="cuda")

    def step():
        y = training.layer_norm(nested, 64, w, b).values()
        return torch.autograd.grad(y, [w, b], g)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = step()
    torch.cuda.current_stream().wait_stream(side)
    eager = training.layer_norm(nested, 64, w, b).values()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="eager graph of the same leaves"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step()
    assert all(torch.equal(a, c) for a, c in zip(torch.autograd.grad(eager, [w, b], g), want))
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_second_derivatives_are_refused(cuda_device):
    x = torch.randn(6, 32, device="cuda", requires_grad=True)
    sizes = torch.tensor([[2, 32], [4, 32]])
    y = training.layer_norm(_nested(x, sizes), 32).values()
    grad, = torch.autograd.grad(y.square().sum(), [x], create_graph=True)
    with pytest.raises(NotImplementedError, match="first derivatives only"):
        grad.sum().backward()


def test_inference_functions_refuse_tracked_values(cuda_device):
    x = torch.randn(6, 32, device="cuda", requires_grad=True)
    nested = nt.nested_tensor([torch.randn(2, 32), torch.randn(4, 32)], device="cuda").with_values(x * 1)
    with pytest.raises(RuntimeError, match="does not track gradients"):
        nested.to_padded_tensor(0)
    with torch.no_grad():
        assert nested.to_padded_tensor(0).shape == (2, 4, 32)
        want = nt.nn.layer_norm(nested, 32)
    assert torch.equal(training.layer_norm(nested, 32).values().view(-1), want._buffer)
