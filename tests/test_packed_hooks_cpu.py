"""What ``packed_activations`` does with tensors that it keeps as they are, on the CPU, where that is all of them."""
import gc
import weakref

import pytest
import torch

import hiscache


@pytest.mark.parametrize("op", (torch.exp, torch.sigmoid, torch.relu, lambda x: torch.softmax(x, 1)))
def test_a_graph_without_a_backward_pass_is_freed(op):
    x = torch.randn(6, 8, requires_grad=True)
    with hiscache.packed_activations(min_elements=1):
        y = op(x * 2)
    result = weakref.ref(y)
    del y
    gc.collect()
    assert result() is None


def test_gradients_through_what_is_kept():
    x, w = torch.randn(6, 8, requires_grad=True), torch.randn(8, 5, requires_grad=True)

    def loss():
        return (torch.tanh(x @ w).exp() * 2).sum()

    want = torch.autograd.grad(loss(), (x, w))
    with hiscache.packed_activations(min_elements=1):
        y = loss()
        g, = torch.autograd.grad((w * w * w).sum(), w, create_graph=True)
    for a, b in zip(torch.autograd.grad(y, (x, w)), want):
        assert torch.equal(a, b)
    assert torch.allclose(torch.autograd.grad(g.sum(), w)[0], 6 * w)          # a gradient of a gradient


@pytest.mark.parametrize("which", ("parameter", "result", "view", "data"))
def test_what_is_changed_in_place_before_the_backward_pass_is_noticed(which):
    x, w = torch.randn(6, 8), torch.randn(8, 8, requires_grad=True)
    with hiscache.packed_activations(min_elements=1):
        h = (x @ w).exp()
        y = (h.view(48) * 3).sum() + ((h @ w) ** 2).sum()
    with torch.no_grad():
        {"parameter": w, "result": h, "view": h[:1], "data": x}[which].mul_(100)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_operators_in_place_within_the_context():
    a = torch.randn(6, 8, requires_grad=True)
    with hiscache.packed_activations(min_elements=1):
        y = ((a * 2).exp_() + 1).sigmoid_()
    got, = torch.autograd.grad(y.sum(), a)
    assert torch.equal(got, torch.autograd.grad(((a * 2).exp() + 1).sigmoid().sum(), a)[0])


def test_what_counts_as_an_activation():
    is_activation = hiscache.experts._is_activation
    h = torch.randn(6, 8)
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        assert is_activation(h.to(dtype), 1) and is_activation(h.view(2, 3, 8).to(dtype), 48)
    for other in (h.view(-1), h.double(), h.long(), h.t(), h[:, ::2], h.clone().requires_grad_(True)):
        assert not is_activation(other, 1)
    assert not is_activation(h, 49)
    for empty in (h[:0], h[:, :0], torch.empty(0, 0)):
        assert not is_activation(empty, 0)


@pytest.mark.parametrize("layout", (torch.sparse_coo, torch.sparse_csr, torch.sparse_csc, torch.sparse_bsr))
def test_sparse_matrices_are_kept_as_they_are(layout):
    blocks = dict(blocksize=(2, 2)) if layout is torch.sparse_bsr else {}
    assert not hiscache.experts._is_activation(torch.eye(8).to_sparse(layout=layout, **blocks), 1)


class Twice(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        return x * 2

    @staticmethod
    def backward(ctx, g):
        return g * 2


P = torch.nn.Parameter
WEIGHTS = {
    "parameter": lambda w: w,
    "frozen": lambda w: P(w.detach(), requires_grad=False),
    "row block": lambda w: w[1],
    "flattened": lambda w: w.view(-1, 8),
    "frozen row block": lambda w: P(w.detach(), requires_grad=False)[1],
    "cast": lambda w: w.bfloat16(),
    "row block of a cast": lambda w: w.bfloat16()[1],
    "scaled": lambda w: w * 0.5,
    "scaled by a tensor": lambda w: w * torch.full((8,), 0.5),
    "a scaled row block": lambda w: w[1] * 0.5,
    "transposed copy": lambda w: w[0].t().contiguous(),
    "normalised": lambda w: torch.nn.functional.normalize(w, dim=-1),
    "sum of two": lambda w: w + P(torch.randn(3, 8, 2)) @ P(torch.randn(3, 2, 8)),
    "leaf": lambda w: w.detach().clone().requires_grad_(True),
    "view of a leaf": lambda w: w.detach().clone().requires_grad_(True).view(24, 8),
}
ACTIVATIONS = {
    "data": lambda x, w: x,
    "a row block of data": lambda x, w: x[:3],
    "product": lambda x, w: x @ w[0],
    "linear": lambda x, w: torch.nn.functional.linear(x, w[0], P(torch.zeros(8))),
    "relu": lambda x, w: torch.relu(x @ w[0]),
    "product by a cast": lambda x, w: x.bfloat16() @ w[0].bfloat16(),
    "rows times a vector": lambda x, w: x * P(torch.ones(8)),
    "embedding": lambda x, w: torch.nn.functional.embedding(torch.arange(5), P(torch.randn(9, 8))),
    "rows of a table": lambda x, w: P(torch.randn(9, 8))[torch.tensor([1, 1, 4])],
    "of an operator of one's own": lambda x, w: Twice.apply(w[0]),
    "rows over a norm": lambda x, w: (x @ w[0]) / (x @ w[0]).norm(),
    "masked": lambda x, w: (x @ w[0]) * torch.ones(7, 8),
    "of a leaf": lambda x, w: x.clone().requires_grad_(True) * 1,
    "deep": lambda x, w: torch.relu(torch.relu(torch.relu(x @ w[0]) @ w[1]) @ w[2]) + 1,
}


@pytest.mark.parametrize("name", WEIGHTS)
def test_weights_are_not_activations(name):
    assert not hiscache.experts._is_activation(WEIGHTS[name](P(torch.randn(3, 8, 8))), 1)


@pytest.mark.parametrize("name", ACTIVATIONS)
def test_activations_are(name):
    assert hiscache.experts._is_activation(ACTIVATIONS[name](torch.randn(7, 8), P(torch.randn(3, 8, 8))), 1)


@pytest.mark.parametrize("dtype,least", ((torch.float32, 2), (torch.float16, 5), (torch.bfloat16, 5)))
@pytest.mark.parametrize("group", (32, 64, 128))
def test_rows_too_narrow_to_get_smaller_are_kept_as_they_are(dtype, least, group):
    for width in (1, 2, 3, 4, 5, 6, 31, 33, 65, 129):
        t = torch.randn(9, width).to(dtype)
        smaller = width + 4 * -(-width // group) < width * t.element_size()
        assert hiscache.experts._is_activation(t, 1, group) == smaller == (width >= least)
