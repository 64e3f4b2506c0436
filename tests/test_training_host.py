"""Refusals and the host side of the training operators: nothing here reaches a GPU."""
import pytest
import torch

import nestedtensor_b200 as nt
from nestedtensor_b200 import _cabi
from nestedtensor_b200.nn import training


def test_values_and_with_values():
    ts = [torch.randn(3, 4), torch.randn(0, 4), torch.randn(2, 4)]
    a = nt.nested_tensor(ts)
    assert torch.equal(a.values(), torch.cat(ts)) and a.values().data_ptr() == a._buffer.data_ptr()
    x = torch.randn(5, 7, requires_grad=True)
    b = a.with_values(x)
    assert b.nested_size() == (torch.Size([3, 7]), torch.Size([0, 7]), torch.Size([2, 7]))
    assert b.values() is x and b.requires_grad and not a.requires_grad
    b.unbind()[2].sum().backward()
    assert torch.equal(x.grad, torch.cat([torch.zeros(3, 7), torch.ones(2, 7)]))
    assert a.with_values(torch.arange(5)).nested_size() == (torch.Size([3]), torch.Size([0]), torch.Size([2]))
    t = torch.randn(7, 5).t()
    assert torch.equal(a.with_values(t).values(), t) and a.with_values(t).values().is_contiguous()
    half = b.to(torch.float16)
    assert half.requires_grad and half.dtype == torch.float16 and half.nested_size() == b.nested_size()
    with pytest.raises(RuntimeError, match="got 4 rows for 5"):
        a.with_values(torch.randn(4, 2))
    with pytest.raises(TypeError):
        a.with_values(3)
    with pytest.raises(RuntimeError, match="regular dimensions"):
        nt.nested_tensor([torch.randn(2, 3), torch.randn(2, 4)]).values()
    empty = nt.nested_tensor([])
    assert empty.values().numel() == 0 and len(empty.with_values(torch.randn(0, 3))) == 0


def test_no_cpu_implementation(native_libs):
    a = nt.nested_tensor([torch.randn(3, 6), torch.randn(5, 6)])
    for call in (lambda: training.layer_norm(a, 6), lambda: training.self_attention(a, 1), lambda: training.attention(a, a, a, 1)):
        with pytest.raises(RuntimeError, match="no CPU implementation"):
            call()
    with pytest.raises(RuntimeError, match="CUDA weight"):
        training.embedding(nt.nested_tensor([torch.tensor([1, 2])], dtype=torch.int64), torch.randn(4, 8))


def test_argument_errors(native_libs):
    a = nt.nested_tensor([torch.randn(3, 6), torch.randn(5, 6)])
    with pytest.raises(TypeError):
        training.layer_norm(torch.randn(3, 6), 6)
    with pytest.raises(NotImplementedError):
        training.embedding(a, torch.randn(3, 3))
    for kw in (dict(max_norm=1.0), dict(scale_grad_by_freq=True), dict(sparse=True)):
        with pytest.raises(NotImplementedError):
            training.embedding(nt.nested_tensor([torch.tensor([1])], dtype=torch.int64), torch.randn(3, 3), **kw)
    with pytest.raises(RuntimeError, match="3 dim"):
        training.self_attention(nt.nested_tensor([torch.randn(3)]), 1)
    with pytest.raises(RuntimeError, match="same nested size"):
        training.attention(a, a, nt.nested_tensor([torch.randn(3, 6), torch.randn(4, 6)]), 1)


def test_cabi_rejects_bad_arguments_without_launching(native_libs):
    lib = _cabi.load()
    # layer norm
    assert lib.ntb200_layer_norm_train(16, None, None, -1.0, 16, 16, 16, 4, 8, 0, None) == -1          # eps
    assert lib.ntb200_layer_norm_train(16, 16, None, 1e-5, 16, 16, 16, 4, 8, 0, None) == -1            # gamma without beta
    assert lib.ntb200_layer_norm_train(16, None, None, 1e-5, 16, 16, 16, 4, 8, 3, None) == -2          # dtype
    assert lib.ntb200_layer_norm_train(16, None, None, 1e-5, 16, None, 16, 4, 8, 0, None) == -1        # statistics missing
    assert lib.ntb200_layer_norm_train(None, None, None, 1e-5, None, None, None, 0, 8, 0, None) == 0   # no rows
    need = lib.ntb200_layer_norm_backward_workspace_bytes(100, 64)
    assert need == 100 * 2 * 64 * 4 and lib.ntb200_layer_norm_backward_workspace_bytes(0, 64) == 0
    assert lib.ntb200_layer_norm_backward(16, 16, 16, 16, 16, 16, 16, 16, 100, 64, 0, 16, need - 1, None) == -6
    assert lib.ntb200_layer_norm_backward(16, 16, 16, 16, 16, 16, 16, 16, 100, 64, 0, 18, need, None) == -3
    assert lib.ntb200_layer_norm_backward(16, 16, 16, 16, None, 16, 16, None, 100, 64, 0, 16, need, None) == -1  # no gamma
    assert lib.ntb200_layer_norm_backward(None, 16, 16, 16, None, 16, None, None, 100, 64, 0, None, 0, None) == -1
    assert lib.ntb200_layer_norm_backward(16, 16, 16, 16, None, 16, None, None, 100, 64, 9, None, 0, None) == -2
    assert lib.ntb200_layer_norm_backward(None, None, None, None, None, None, None, None, 0, 64, 0, None, 0, None) == 0
    # embedding
    assert lib.ntb200_embedding_scaled(16, 16, 2, 16, 4, 10, 8, 1.0, 0, None) == -1                    # index width
    assert lib.ntb200_embedding_scaled(16, 16, 8, 16, 4, 0, 8, 1.0, 0, None) == -1                     # empty table
    assert lib.ntb200_embedding_scaled(16, 16, 8, 16, 4, 10, 8, 1.0, 5, None) == -2
    need = lib.ntb200_embedding_backward_workspace_bytes(1000, 64)
    assert need > 0 and lib.ntb200_embedding_backward_workspace_bytes(0, 64) == 0
    assert lib.ntb200_embedding_backward(16, 16, 8, 16, 1000, 10, 64, -1, 1.0, 0, 16, need - 1, None) == -6
    assert lib.ntb200_embedding_backward(16, 16, 8, 16, 1000, 10, 64, -1, 1.0, 0, 24, need, None) == -3
    assert lib.ntb200_embedding_backward(16, 16, 8, None, 1000, 10, 64, -1, 1.0, 0, 16, need, None) == -1
    assert lib.ntb200_embedding_backward(16, 16, 3, 16, 1000, 10, 64, -1, 1.0, 0, 16, need, None) == -1
    assert lib.ntb200_embedding_backward(16, 16, 8, 16, 1 << 31, 10, 64, -1, 1.0, 0, 16, need, None) == -7
    assert lib.ntb200_embedding_backward(None, None, 8, None, 0, 0, 64, -1, 1.0, 0, None, 0, None) == 0

    # attention
    def train(q=16, ld=64, k=16, out=32, lse=16, offs=16, row=64, batch=1, tq=4, tk=4, heads=1, d=64, dtype=2, path=0, ws=None, n=0):
        return lib.ntb200_varlen_attention_train(q, ld, k, ld, k, ld, out, lse, offs, row, offs, row, batch, tq, tk, heads, d, 4, 0.125, dtype,
                                                 path, ws, n, None)

    assert train(ld=63) == -1 and train(lse=None) == -1 and train(row=0) == -1 and train(path=4) == -1 and train(dtype=3) == -2
    assert train(d=257, ld=300) == -7 and train(batch=0) == 0 and train(tq=0) == 0 and train(k=None) == -1
    assert train(path=3, ws=16, n=3) == -6 and train(path=3, d=32) == -7
    assert train(path=3, ws=16, n=1 << 20, out=16) == -7  # the tcgen05 kernel stores 32 bytes at a time
    assert lib.ntb200_varlen_attention(16, 16, 16, 1, 4, 1, 64, 4, 0.125, 2, 3, 16, 1 << 20, None) == -7

    def backward(g=16, ld=64, offs=16, row=64, batch=1, tq=4, tk=4, heads=1, d=64, dtype=2, path=0, ws=16, n=1 << 20, dq=16):
        return lib.ntb200_varlen_attention_backward(g, 16, ld, 16, ld, 16, ld, 16, 16, dq, ld, 16, ld, 16, ld, offs, row, offs, row, batch, tq,
                                                    tk, heads, d, 4, 4, 0.125, dtype, path, ws, n, None)

    need = lib.ntb200_varlen_attention_backward_workspace_bytes(1, 4, 4, 1, 64, 4, 4, 2, 0)
    assert need > 0
    assert backward(ld=63) == -1 and backward(g=None) == -1 and backward(dq=None) == -1 and backward(row=0) == -1 and backward(path=9) == -1
    assert backward(dtype=3) == -2 and backward(d=257, ld=300) == -7 and backward(ws=None) == -1 and backward(n=need - 1) == -6
    assert backward(ws=24) == -3 and backward(batch=0) == 0 and backward(tq=0, tk=0) == 0 and backward(tq=1 << 31, n=1 << 62) == -7
