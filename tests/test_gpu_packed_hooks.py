"""``packed_activations`` around the layer of experts and around products by weights: what is not an activation goes into the
gradients exactly as it does outside the context."""
import math

import pytest
import torch

import hiscache
import hiscache_backend as be

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = (torch.float32, torch.float16, torch.bfloat16)


def both(forward, leaves, seed=0):
    """The gradients outside the context and inside, where the smallest matrix is kept in 8 bits."""
    grads = []
    for inside in (False, True):
        if inside:
            with hiscache.packed_activations(min_elements=1):
                out = forward()
        else:
            out = forward()
        g = torch.randn(out.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed)).to(out.dtype)
        grads.append(torch.autograd.grad(out, leaves, g))
    return zip(*grads)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("normalize", (True, False))
def test_routing_is_kept_exactly(dtype, normalize):
    l = 2 * torch.randn(300, 24, device=DEV)
    l[torch.rand(300, 24, device=DEV) < 0.2] = -math.inf
    l[7] = -math.inf
    a = l.to(dtype).requires_grad_(True)
    # (a leaf is never packed: what the router makes is not one)
    for outside, inside in both(lambda: be.route_rows(a * 1, 3, normalize=normalize)[1], (a,)):
        assert torch.equal(outside, inside) and bool(torch.isfinite(inside).all())


def same(a, b):
    """The same values, NaNs (of fp16 that has overflowed) in the same places."""
    return torch.allclose(a, b, rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_the_gate_s_scales_are_kept_exactly(dtype):
    gen = torch.Generator(device=DEV).manual_seed(0)
    x, w_in, w_out = (torch.randn(*s, device=DEV, generator=gen).to(dtype) for s in ((40, 64), (3, 512, 64), (3, 48, 256)))
    w_in[:, :64] *= 300                              # groups of very different size side by side
    leaves = [t.requires_grad_(True) for t in (x, w_in, w_out)]
    offset = torch.tensor([0, 10, 20, 40], device=DEV)
    (gx, gx2), (gi, gi2), (go, go2) = both(lambda: be.gated_experts(*leaves, offset), leaves)
    assert same(gx, gx2) and same(gi, gi2) and same(go, go2)


def test_the_weights_of_the_way_back_are_kept_exactly():
    gen = torch.Generator(device=DEV).manual_seed(0)
    order = be.expert_order(torch.randint(0, 3, (40, 2), device=DEV, generator=gen), 3)
    y, w = torch.randn(80, 24, device=DEV, generator=gen).requires_grad_(True), torch.rand(40, 2, device=DEV, generator=gen)
    w[:, 1] *= 1e-3
    (a, b), = both(lambda: be.rows_from_experts(y, order, w), (y,))
    assert torch.equal(a, b)


@pytest.mark.parametrize("normalize", (True, False))
@pytest.mark.parametrize("closed", (True, False))
def test_a_layer_of_experts_in_the_context(normalize, closed):
    torch.manual_seed(3)
    layer = hiscache.ExpertMLP(64, 96, 6, 2, normalize=normalize, device=DEV)
    x = torch.randn(500, 64, device=DEV, requires_grad=True)
    allowed = torch.rand(500, 6, device=DEV) < 0.7 if closed else None
    names = ["x", *dict(layer.named_parameters())]
    for name, (outside, inside) in zip(names, both(lambda: layer(x * 1, allowed=allowed), (x, *layer.parameters()))):
        assert bool(torch.isfinite(inside).all())
        # rows and results in 8 bits, a scale of 1 / 127 of 64 values' largest, half of it the most that one is off
        assert float((outside - inside).norm() / outside.norm()) <= 0.02, name


def test_the_statistics_of_a_normalisation_are_kept_exactly():
    gen = torch.Generator(device=DEV).manual_seed(5)
    x = torch.randn(700, 64, device=DEV, generator=gen) * torch.exp(2 * torch.randn(64, device=DEV, generator=gen))
    x.requires_grad_(True)
    bn = torch.nn.BatchNorm1d(64).to(DEV)
    from hiscache.history_model import bn_relu
    # (a leaf is not packed, so that all that could differ are the node's own statistics)
    for outside, inside in both(lambda: bn_relu(x, bn), (x, bn.weight, bn.bias)):
        assert torch.equal(outside, inside)


WEIGHTS = {
    "row block": lambda x, w, frozen: x @ w[1],
    "stack": lambda x, w, frozen: torch.matmul(x.expand(4, 64, 300), w).sum(0),
    "frozen": lambda x, w, frozen: x @ frozen,
    "scaled": lambda x, w, frozen: x @ (w[0] * 0.5),
    "normalised": lambda x, w, frozen: x @ torch.nn.functional.normalize(w[2], dim=0),
    "experts": lambda x, w, frozen: be.expert_linear(x, w * 2, torch.tensor([0, 20, 30, 50, 64], device=DEV)),
    "experts, cast": lambda x, w, frozen: be.expert_linear(x.bfloat16(), w.bfloat16(), torch.tensor([0, 20, 30, 50, 64], device=DEV)),
}


@pytest.mark.parametrize("name", WEIGHTS)
def test_a_gradient_of_rows_goes_by_the_weights_as_they_are(name):
    gen = torch.Generator(device=DEV).manual_seed(4)
    w = torch.nn.Parameter(torch.randn(4, 300, 300, device=DEV, generator=gen))
    frozen = torch.nn.Parameter(torch.randn(300, 300, device=DEV, generator=gen), requires_grad=False)
    x = torch.randn(64, 300, device=DEV, generator=gen).requires_grad_(True)
    for outside, inside in both(lambda: WEIGHTS[name](x, w, frozen), (x,)):
        assert torch.equal(outside, inside)
