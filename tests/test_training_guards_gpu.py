"""The training operators where a call could go wrong unseen: structures of any trailing sizes, what autograd sees of the caller's
tensors, captured graphs."""
import pytest
import torch

import nestedtensor_b200 as nt
from nestedtensor_b200.nn import training

pytestmark = pytest.mark.gpu


def _nested(shapes, dtype):
    sizes = torch.tensor(shapes, dtype=torch.int64)
    return nt.NestedTensor(torch.zeros(int(sizes.prod(1).sum()), dtype=dtype, device="cuda"), sizes)


@pytest.mark.parametrize("widths", [(5, 7, 1, 3), (9, 0, 2, 40), (0, 0, 0, 0), (6, 5, 4, 3)], ids=str)
@pytest.mark.parametrize("dtype,heads,d", [(torch.float32, 2, 16), (torch.float16, 2, 64), (torch.bfloat16, 1, 128)], ids=str)
def test_attention_over_the_rows_of_irregular_constituents(cuda_device, dtype, heads, d, widths):
    """with_values() keeps the lengths alone: the bits of the same rows in a regular structure."""
    lengths, keys = (3, 4, 70, 200), (1, 90, 0, 33)
    gen = torch.Generator().manual_seed(d)
    E = heads * d

    def rows(n, width):
        return torch.randn(n, width, generator=gen).to(dtype).cuda().requires_grad_()

    odd = _nested([(n, w) for n, w in zip(lengths, widths)], dtype)
    odd_keys = _nested([(n, w) for n, w in zip(keys, widths[::-1])], dtype)
    even, even_keys = (_nested([(n, 8) for n in ls], dtype) for ls in (lengths, keys))
    qkv, q, k, v = rows(sum(lengths), 3 * E), rows(sum(lengths), E), rows(sum(keys), E), rows(sum(keys), E)
    g = torch.randn(sum(lengths), E, generator=gen).to(dtype).cuda()
    results = []
    for a, b in ((odd, odd_keys), (even, even_keys)):
        y = training.self_attention(a.with_values(qkv), heads).values()
        z = training.attention(a.with_values(q), b.with_values(k), b.with_values(v), heads).values()
        results.append((y, z, *torch.autograd.grad([y, z], [qkv, q, k, v], [g, g])))
    for x, want in zip(*results):
        assert torch.equal(x, want) and bool(torch.isfinite(x).all())
