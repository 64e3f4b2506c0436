"""The training operators where a call could go wrong unseen: structures of any trailing sizes, what autograd sees of the caller's
tensors, captured graphs."""
import copy
import pickle

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


def test_capture_needs_the_offsets_on_the_device(cuda_device):
    """Made inside a capture, the offsets would be copied out of a host block that is no longer theirs at the replay: refused; and a
    nested tensor whose offsets were made before is taken, by training and inference operators alike."""
    sizes = torch.tensor([[3, 96], [50, 96]])
    x = torch.randn(53, 96, device="cuda")
    ready, late = nt.NestedTensor(x.view(-1), sizes), nt.NestedTensor(x.view(-1), sizes)
    want = training.self_attention(ready, 2).values()
    assert ready._meta is not None and late._meta is None
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            training.self_attention(late, 2)
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            training.attention(ready, late, late, 2)
    assert late._meta is None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = training.self_attention(ready, 2).values()
    # eager passes over other lengths take whatever host and device memory is free
    for n in range(1, 30):
        other = nt.NestedTensor(x[:n + 20].reshape(-1), torch.tensor([[n, 96], [20, 96]]))
        training.self_attention(other, 2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_offsets_made_inside_a_capture_are_not_kept(cuda_device):
    """An inference operator makes the offsets in its graph, where they hold nothing before the replay: an eager call makes its own."""
    sizes = torch.tensor([[3, 8], [50, 8]])
    x = torch.randn(53, 8, device="cuda")
    nested = nt.NestedTensor(x.view(-1), sizes)
    want = nt.NestedTensor(x.view(-1), sizes).to_padded_tensor(0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = nested.to_padded_tensor(0)
    assert nested._meta is None
    assert torch.equal(nested.to_padded_tensor(0), want)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def _in_a_capture(step):
    """`step` run eagerly on a side stream (no graph of it stays alive), then captured: (eager result, result of one replay)."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    return want, got


def test_capture_beside_an_eager_graph_of_a_leaf_behind_other_nodes(cuda_device):
    """The leaf whose eager graph is alive need not be an input of the operator itself: a projection and a view lie between."""
    sizes = torch.tensor([[3, 64], [5, 64]])
    x, p = (torch.randn(s, device="cuda", requires_grad=True) for s in ((8, 32), (32, 64)))
    w, b = (torch.randn(64, device="cuda", requires_grad=True) for _ in range(2))
    g = torch.randn(8, 64, device="cuda")

    def step(leaves=(x, p, w, b)):
        rows = (x @ p).view(-1)
        y = training.layer_norm(nt.NestedTensor(rows, sizes), 64, w, b).values()
        return torch.autograd.grad(y, leaves, g)

    want, got = _in_a_capture(step)  # no eager graph is alive (and cuBLAS is set up)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    for make in (lambda: x * 2, lambda: p.view(-1) * 3):
        eager = make()
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="eager graph of the same leaves"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                step()
        want, got = _in_a_capture(lambda: step((w, b)))  # a pass that does not reach the leaf
        assert all(torch.equal(a, c) for a, c in zip(got, want))
        eager.sum().backward()
        del eager
        x.grad = p.grad = None
    want, got = _in_a_capture(step)
    assert all(torch.equal(a, c) for a, c in zip(got, want))


def _hooked(x, sizes):
    """(leaf, the flat buffer made from it, a nested tensor over that buffer)"""
    x = x.detach().requires_grad_()
    buf = x.view(-1)
    return x, buf, nt.NestedTensor(buf, sizes)


def test_the_callers_buffer_is_in_the_graph(cuda_device):
    """Hooks on the buffer that a nested tensor was made of see and change its gradient; it can keep it, and be differentiated."""
    sizes = torch.tensor([[2, 96], [7, 96]])
    data, g = torch.randn(9, 96, device="cuda"), torch.randn(9, 96, device="cuda")
    ops = {"norm": lambda t: training.layer_norm(t, 96), "self": lambda t: training.self_attention(t, 2),
           "query": lambda t: training.attention(t, t.with_values(data), t.with_values(data), 2)}
    for name, op in ops.items():
        x, buf, nested = _hooked(data, sizes)
        y = op(nested).values()
        go = g[:, :y.size(1)]
        want, = torch.autograd.grad(y, x, go)
        x, buf, nested = _hooked(data, sizes)
        buf.register_hook(lambda t: t * 2)
        y = op(nested).values()
        y.backward(go)
        assert torch.equal(x.grad, want * 2), name
        x, buf, nested = _hooked(data, sizes)
        got, = torch.autograd.grad(op(nested).values(), buf, go)
        assert torch.equal(got, want.view(-1)), name
        buf.retain_grad()
        op(nested).values().backward(go)
        assert torch.equal(buf.grad, want.view(-1)) and torch.equal(x.grad, want), name


def test_a_buffer_cut_off_from_the_graph_stays_cut_off(cuda_device):
    """No gradient flows through a view made under no_grad to its base."""
    sizes = torch.tensor([[2, 64], [7, 64]])
    x = torch.randn(9, 64, device="cuda", requires_grad=True)
    w, b = (torch.randn(64, device="cuda", requires_grad=True) for _ in range(2))
    with torch.no_grad():
        buf = x.view(-1)
    y = training.layer_norm(nt.NestedTensor(buf, sizes), 64, w, b).values()
    y.sum().backward()
    assert x.grad is None and w.grad is not None


def test_inference_functions_refuse_a_tracked_buffer(cuda_device):
    """One answer for one object: what nn.training would track, the functions that track nothing refuse."""
    x = torch.randn(6, 32, device="cuda", requires_grad=True)
    nested = nt.NestedTensor(x.view(-1), torch.tensor([[2, 32], [4, 32]]))
    assert nested.requires_grad and nested.values().requires_grad
    for call in (lambda: nested.to_padded_tensor(0), lambda: nt.nn.layer_norm(nested, 32), lambda: nested.to_tensor_mask()):
        with pytest.raises(RuntimeError, match="does not track gradients"):
            call()
    with torch.no_grad():
        want = nt.nn.layer_norm(nested, 32)
    assert torch.equal(training.layer_norm(nested, 32).values().view(-1), want._buffer)
    assert torch.equal(nt.nn.layer_norm(nt.NestedTensor(x.detach().view(-1), nested._sizes), 32)._buffer, want._buffer)


def test_operators_that_read_lengths_alone_take_tracked_tensors(cuda_device):
    x = torch.randn(6, 32, device="cuda", requires_grad=True)
    nested = nt.NestedTensor(x.view(-1), torch.tensor([[2, 32], [4, 32]]))
    for t in (nested, nested.with_values(x * 1)):
        mask = torch.ops.nestedtensor.to_mask(t, 2)
        assert mask.tolist() == [[True, True, False, False], [True] * 4]
        padded = torch.randn(2, 4, 32, device="cuda")
        got = torch.ops.nestedtensor.from_padded_tensor(padded, t)
        assert torch.equal(got._buffer.view(6, 32), torch.cat([padded[0, :2], padded[1]]))


def test_channels_last_operators_refuse_a_tracked_buffer(cuda_device):
    x = torch.randn(8 * 6, device="cuda", requires_grad=True)
    images = nt.NestedTensor(x.view(-1), torch.tensor([[8, 2, 1], [8, 2, 2]]), channels_last=True)
    weight = torch.randn(4, 8, 1, 1, device="cuda", requires_grad=True)
    for call in (lambda: images.contiguous(), lambda: nt.nn.conv2d(images, weight), lambda: images.to_padded_tensor(0)):
        with pytest.raises(RuntimeError, match="does not track gradients"):
            call()
    with torch.no_grad():
        want = nt.nn.conv2d(images, weight)._buffer
    got = nt.nn.conv2d(nt.NestedTensor(x.detach(), images._sizes, channels_last=True), weight)  # (the weight's gradient is not offered)
    assert torch.equal(got._buffer, want) and not got.requires_grad
    assert torch.ops.nestedtensor.to_mask(images, 2).shape[0] == 2


def test_offsets_made_on_a_busy_stream_are_waited_for(cuda_device):
    """The first call puts the offsets' copy on its stream, behind what is queued there; a call on another stream, over values that are
    ready, does not run ahead of it."""
    sizes = torch.tensor([[30, 192], [7, 192], [200, 192]])
    x = torch.randn(237, 192, device="cuda")
    want = training.self_attention(nt.NestedTensor(x.view(-1), sizes), 1).values()
    padded = nt.NestedTensor(x.view(-1), sizes).to_padded_tensor(0)
    torch.cuda.synchronize()
    busy, other = torch.cuda.Stream(), torch.cuda.Stream()
    for irregular in (False, True):
        nested = nt.NestedTensor(x.view(-1), sizes)
        if irregular:
            nested = nt.NestedTensor(torch.zeros(37 * 3 + 200, device="cuda"), torch.tensor([[30, 3], [7, 3], [200, 1]])).with_values(x)
        torch.cuda.synchronize()
        with torch.cuda.stream(busy):
            torch.cuda._sleep(200_000_000)  # about a tenth of a second
            first = training.self_attention(nested, 1).values()
        with torch.cuda.stream(other):
            second = training.self_attention(nested, 1).values()
            third = nested.to_padded_tensor(0)
        torch.cuda.synchronize()
        assert torch.equal(first, want) and torch.equal(second, want) and torch.equal(third, padded)
        assert nested._row_offsets()[0].device == x.device and torch.equal(training.self_attention(nested, 1).values(), want)


def test_copies_and_pickles(cuda_device):
    """Of a nested tensor whose offsets have just been made, and of one made from it."""
    sizes = torch.tensor([[3, 96], [50, 96]])
    x = torch.randn(53, 96, device="cuda")
    a = nt.NestedTensor(x.view(-1), sizes)
    b = a.with_values(x * 2)
    want = [training.self_attention(t, 2).values() for t in (a, b)]
    padded = [t.to_padded_tensor(0) for t in (a, b)]
    for again in (copy.deepcopy((a, b)), pickle.loads(pickle.dumps((a, b)))):
        for t, w, p in zip(again, want, padded):
            assert torch.equal(training.self_attention(t, 2).values(), w) and torch.equal(t.to_padded_tensor(0), p)
