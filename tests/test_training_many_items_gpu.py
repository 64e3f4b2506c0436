"""Gradients of batches whose work is many times what the GPU holds at once, so that every block of the persistent kernels takes one
item after another: small cases elsewhere give most blocks one item."""
import pytest
import torch

import nestedtensor_b200 as nt
import _training_reference as ref
from test_training_gpu import _attend_inputs, _cabi_backward, _check, _ragged, _run_attend, _run_embed, _run_norm, _run_self

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]

# 40 sequences in an order that mixes the kernels' classes and tiles, some empty; the other side in another order
LENGTHS = [(0, 1, 65, 129, 300, 513, 17, 128)[i * 5 % 8] for i in range(40)]
OTHERS = [(300, 0, 64, 1, 129, 40, 513, 65)[i * 3 % 8] for i in range(40)]


def _twice(run):
    """One result, if the second run's bits are the first's."""
    got, again = run(), run()
    assert all(torch.equal(got[n], again[n]) for n in got)
    return got


# up to 1100 tiles or 640 sequences and heads a kernel, on 148 multiprocessors
@pytest.mark.parametrize("dtype,heads,d", [(torch.float16, 16, 64), (torch.bfloat16, 16, 64), (torch.float16, 12, 128), (torch.bfloat16, 12, 128),
                                           (torch.float16, 16, 32), (torch.float32, 8, 64), (torch.bfloat16, 8, 80)], ids=str)
def test_attention_many_items(cuda_device, dtype, heads, d):
    nt.device_error_flags()
    q, k, v, g, qs, _ = _attend_inputs(LENGTHS, LENGTHS, heads, d, dtype, d)
    want, bound = ref.attention(q, k, v, g, LENGTHS, LENGTHS, heads, d ** -0.5)
    _check(_twice(lambda: _run_self(q, k, v, g, qs, heads)), want, bound, "self")
    q, k, v, g, qs, ks = _attend_inputs(LENGTHS, OTHERS, heads, d, dtype, d + 1)
    want, bound = ref.attention(q, k, v, g, LENGTHS, OTHERS, heads, d ** -0.5)
    _check(_twice(lambda: _run_attend(q, k, v, g, qs, ks, heads)), want, bound, "cross")
    assert nt.device_error_flags() == 0


@pytest.mark.parametrize("path,dtype,heads,d", [(1, torch.bfloat16, 8, 64), (2, torch.float16, 16, 64), (2, torch.bfloat16, 12, 128),
                                                (3, torch.float16, 16, 64), (3, torch.bfloat16, 16, 64), (3, torch.float16, 12, 128),
                                                (3, torch.bfloat16, 12, 128), (4, torch.float16, 16, 64), (4, torch.bfloat16, 16, 64)], ids=str)
def test_attention_many_items_on_one_path(cuda_device, path, dtype, heads, d):
    """All sequences on one kernel, the empty ones and those of one token among them."""
    nt.device_error_flags()
    q, k, v, g, _, _ = _attend_inputs(LENGTHS, OTHERS, heads, d, dtype, path + d)
    want, bound = ref.attention(q, k, v, g, LENGTHS, OTHERS, heads, d ** -0.5)
    _check(_twice(lambda: _cabi_backward(q, k, v, g, LENGTHS, OTHERS, heads, path, 8)), want, bound, "path %d" % path)


@pytest.mark.parametrize("dtype,d", [(torch.float16, 64), (torch.bfloat16, 128), (torch.float32, 32)], ids=str)
def test_attention_many_sequences(cuda_device, dtype, d):
    """More sequences than the blocks that build the work lists have threads, most of them short or empty."""
    lq = [(i * 7 % 11) % 4 if i % 90 else 70 + i % 300 for i in range(2600)]
    lk = [(i * 5 % 13) % 3 if i % 70 else 66 + i % 200 for i in range(2600)]
    q, k, v, g, qs, _ = _attend_inputs(lq, lq, 2, d, dtype, d)
    want, bound = ref.attention(q, k, v, g, lq, lq, 2, d ** -0.5)
    _check(_run_self(q, k, v, g, qs, 2), want, bound, "self")
    q, k, v, g, qs, ks = _attend_inputs(lq, lk, 2, d, dtype, d + 1)
    want, bound = ref.attention(q, k, v, g, lq, lk, 2, d ** -0.5)
    _check(_run_attend(q, k, v, g, qs, ks, 2), want, bound, "cross")


@pytest.mark.parametrize("features", [8, 64, 72, 200, 250, 333, 512, 768, 771, 1000, 1024, 1536, 2048, 2055, 4096, 6144, 8192])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_layer_norm_many_rows(cuda_device, dtype, features):
    """Rows for several turns of every block, with a remainder."""
    gen = torch.Generator().manual_seed(features)
    rows = 80003 if features <= 72 else 20003 if features <= 512 else 6003 if features <= 2055 else 2003
    x, sizes = _ragged([rows // 3, rows - rows // 3], features, dtype, gen, 2.0)
    w, b = (1 + 0.2 * torch.randn(features, generator=gen)).to(dtype).cuda(), torch.randn(features, generator=gen).to(dtype).cuda()
    g = torch.randn(x.shape, generator=gen).to(dtype).cuda()
    want, bound = ref.layer_norm(x, w, b, g, 1e-5)
    _check(_twice(lambda: _run_norm(x, sizes, w, b, g)), want, bound, "affine")
    want, bound = ref.layer_norm(x, None, None, g, 1e-5)
    del want["dweight"], want["dbias"]
    _check(_run_norm(x, sizes, None, None, g), want, bound, "plain")


# runs of equal indices over several warps: more of them than warps (2000 of about 75 tokens), and than blocks (200 of 1500)
@pytest.mark.parametrize("tokens,vocab", [(150000, 2000), (300000, 200)])
@pytest.mark.parametrize("features", [1024, 1000])
def test_embedding_many_long_runs(cuda_device, tokens, vocab, features):
    gen = torch.Generator(device="cuda").manual_seed(tokens + features)
    dtype = torch.bfloat16 if features == 1024 else torch.float32
    index = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda")
    weight = torch.randn(vocab, features, generator=gen, device="cuda").to(dtype)
    g = torch.randn(tokens, features, generator=gen, device="cuda").to(dtype)
    want, bound = ref.embedding(weight, index, g, 2.0, 7)
    _check(_twice(lambda: _run_embed(weight, index, [tokens], g, padding_idx=7, scale=2.0)), want, bound, "long runs")


def test_operators_of_one_size_after_another(cuda_device):
    """Batches that grow and shrink on the same leaves: nothing of one call is left for the next."""
    heads, d, dtype = 4, 64, torch.float16
    for lengths in ([700, 3], [5], LENGTHS, [1] * 30, [600, 600], [0, 9]):
        q, k, v, g, qs, _ = _attend_inputs(lengths, lengths, heads, d, dtype, len(lengths))
        want, bound = ref.attention(q, k, v, g, lengths, lengths, heads, d ** -0.5)
        _check(_run_self(q, k, v, g, qs, heads), want, bound, str(len(lengths)))
