"""Differentiable LayerNorm, embedding and attention on nested tensors, for training on ragged batches.

    x = nn.training.embedding(tokens, table, padding_idx=0, scale=math.sqrt(E))       # (L_i, E)
    h = nn.training.layer_norm(x, (E,), w, b)
    qkv = h.with_values(torch.nn.functional.linear(h.values(), w_in, b_in))           # (L_i, 3E)
    a = nn.training.self_attention(qkv, num_heads)                                    # (L_i, E)
    loss = a.values().float().square().mean()
    loss.backward()

The functions take and return NestedTensors; ``NestedTensor.values()`` is the packed ``[sum(L_i), ...]`` matrix that carries
the autograd graph, ``NestedTensor.with_values()`` puts a matrix of as many rows back into the ragged structure, so everything
between them (projections, activations, residuals, losses) is plain torch on unpadded rows.

Gradients flow to the values of the inputs, to weights and biases; first derivatives only.  All tensors of a call have one
device and one dtype (float32, float16 or bfloat16); statistics, sums and softmax denominators are fp32.  The gradients are
sums in a fixed order: the same inputs give the same bits.  Work runs on the current stream, the gradients on the stream of
their forward call; workspaces belong to the call.

Forward and backward may be captured into a CUDA graph, with two exceptions, which raise: an eager graph of the same leaves,
made on the default stream, is still alive; or attention needs the offsets of a nested tensor that are not on the device yet (a
pass over it before the capture puts them there, and every nested tensor made from it shares them).

The functions of ``nestedtensor_b200.nn`` itself are the inference forms: they do not track gradients, and refuse a NestedTensor
that does."""
from __future__ import annotations

from typing import Optional

import torch

from .. import _ops
from ..nested import NestedTensor


def _check(obj, name):
    if not isinstance(obj, NestedTensor):
        raise TypeError(name + " must be a NestedTensor")


def layer_norm(input: NestedTensor, normalized_shape, weight=None, bias=None, eps: float = 1e-5) -> NestedTensor:
    """``torch.nn.functional.layer_norm`` with gradients of the input, the weight and the bias.  As ``nn.layer_norm``, the last
    dimension must be regular and equal ``normalized_shape``, a singleton, and weight and bias come together; the dimensions
    between the first and the last must be regular here."""
    _check(input, "input")
    if isinstance(normalized_shape, int):
        normalized_shape = (normalized_shape,)
    x, sizes, features = input._tracked()
    shape = None if input.tensor_dim() == 2 else input.values().shape  # (L_i, ..., E): the operator's rows are finer
    out = _ops.ops().layer_norm_train(x, sizes, features, normalized_shape, weight, bias, eps)
    return input._with_rows(out if shape is None else out.view(shape))


def embedding(input: NestedTensor, weight: torch.Tensor, padding_idx: Optional[int] = None, max_norm=None, norm_type=2.0,
              scale_grad_by_freq=False, sparse=False, scale: float = 1.0) -> NestedTensor:
    """``scale * weight[input]`` for a NestedTensor of 1-D index sequences, with the dense gradient of ``weight``; row
    ``padding_idx`` of the gradient is zero.  ``scale`` is applied in fp32 before the one rounding to the weight's dtype.  An
    index out of range gives a row of zeros, contributes no gradient and raises bit 16 of ``device_error_flags()``.
    ``max_norm``, ``scale_grad_by_freq`` and ``sparse`` are not supported."""
    if max_norm is not None or scale_grad_by_freq or sparse:
        raise NotImplementedError("nestedtensor_b200: embedding with max_norm, scale_grad_by_freq or sparse is not supported")
    _check(input, "input")
    if input.dim() != 2 and len(input) > 0:
        raise NotImplementedError("nestedtensor_b200: embedding expects a nested tensor of 1-D index sequences")
    out = _ops.ops().embedding_train(weight, input._buffer, input._sizes, padding_idx, scale)
    return input._with_rows(out)


def self_attention(qkv: NestedTensor, num_heads: int, scaling: Optional[float] = None) -> NestedTensor:
    """softmax(scaling q k^T) v within every sequence, per head, for a NestedTensor of ``(L_i, 3 * E)`` rows q | k | v (the packed
    projection of ``torch.nn.MultiheadAttention``); ``(L_i, E)``.  ``scaling``, any finite number (the tensor-core kernels take
    positive ones), defaults to ``head_dim ** -0.5``.  The gradient of ``qkv`` has the same packed form."""
    _check(qkv, "qkv")
    if qkv.dim() != 3 and len(qkv) > 0:
        raise RuntimeError("query needs to be 3 dim.")
    x, sizes, features = qkv._tracked()
    meta, row_elems = qkv._row_offsets()
    out = _ops.ops().self_attention_train(x, sizes, features, meta, row_elems, num_heads, scaling)
    return qkv._with_rows(out)


def attention(query: NestedTensor, key: NestedTensor, value: NestedTensor, num_heads: int,
              scaling: Optional[float] = None) -> NestedTensor:
    """softmax(scaling q k^T) v of the queries of sequence b over the keys and values of sequence b, per head, for already projected
    NestedTensors ``(Lq_i, E)``, ``(Lk_i, E)``, ``(Lk_i, E)``; ``(Lq_i, E)``.  A sequence without keys gives zeros and passes no
    gradient.  ``scaling`` as in ``self_attention``."""
    for t, name in ((query, "query"), (key, "key"), (value, "value")):
        _check(t, name)
        if t.dim() != 3 and len(t) > 0:
            raise RuntimeError(name + " needs to be 3 dim.")
    if value is not key and not (key._packed is not None and value._packed is not None and key._ragged is value._ragged) \
            and not torch.equal(key._sizes, value._sizes):
        raise RuntimeError("nestedtensor_b200: key and value must have the same nested size")
    q, q_sizes, features = query._tracked()
    k, k_sizes, k_features = key._tracked()
    v = value._tracked()[0]
    q_meta, q_row = query._row_offsets()
    k_meta, k_row = key._row_offsets()
    out = _ops.ops().attention_train(q, k, v, q_sizes, features, q_meta, q_row, k_sizes, k_features, k_meta, k_row, num_heads, scaling)
    return query._with_rows(out)
