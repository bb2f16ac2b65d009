"""The calls of the expert layer and of activations in 8 bits with operands that are not plain matrices in memory, inside
autograd's other modes, and at the ends of their documented ranges."""
import pytest
import torch
from torch.autograd import forward_ad

import hiscache
import hiscache_backend as be

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def operands(seed=0):
    """Every call of the layer by name, as a function of its floating-point operands, and those operands."""
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def draw(*shape):
        return torch.randn(*shape, device=DEV, generator=gen)

    order = be.expert_order(torch.randint(0, 3, (40, 2), device=DEV, generator=gen), 3)
    offset = torch.tensor([0, 10, 20, 40], device=DEV)
    kept = be.gated_pack(draw(40, 64))[1]
    return {
        "route": (lambda l: be.route_rows(l, 2)[1], [draw(40, 8)]),
        "route, not normalised": (lambda l: be.route_rows(l, 2, normalize=False)[1], [draw(40, 8)]),
        "to experts": (lambda x: be.rows_to_experts(x, order), [draw(40, 24)]),
        "from experts": (lambda y, w: be.rows_from_experts(y, order, w), [draw(80, 24), draw(40, 2)]),
        "from experts, unweighted": (lambda y: be.rows_from_experts(y, order), [draw(80, 24)]),
        "linear": (lambda x, w: be.expert_linear(x, w, offset), [draw(40, 64), draw(3, 32, 64)]),
        "linear_grad": (lambda g, x: be.expert_linear_grad(g, x, offset), [draw(40, 32), draw(40, 64)]),
        "pack": (lambda x: be.unpack_rows(be.pack_rows(x)), [draw(40, 64)]),
        "gated_pack": (lambda x: be.gated_pack(x, keep=False)[0], [draw(40, 64)]),
        "gated_grad": (lambda g: be.gated_grad(kept, g)[0], [draw(40, 32)]),
        "gated_experts": (lambda x, a, b: be.gated_experts(x, a, b, offset), [draw(40, 24), draw(3, 64, 24), draw(3, 16, 32)]),
    }


CALLS = ("route", "route, not normalised", "to experts", "from experts", "from experts, unweighted", "linear", "linear_grad", "pack",
         "gated_pack", "gated_grad", "gated_experts")
NODES = tuple(c for c in CALLS if c not in ("linear_grad", "pack", "gated_pack", "gated_grad"))


@pytest.mark.parametrize("name", CALLS)
def test_a_tangent_is_refused(name):
    call, args = operands()[name]
    want = call(*args)
    with forward_ad.dual_level():
        assert torch.equal(call(*args), want)                     # plain operands, whatever level there is
        for i, a in enumerate(args):
            dual = [*args[:i], forward_ad.make_dual(a, torch.ones_like(a)), *args[i + 1:]]
            with pytest.raises(NotImplementedError):
                call(*dual)
            with torch.no_grad(), pytest.raises(NotImplementedError):     # forward mode does not go by the grad mode
                call(*dual)


@pytest.mark.parametrize("name", NODES)
def test_a_tangent_of_a_gradient_is_refused(name):
    call, args = operands()[name]
    args = [a.requires_grad_(True) for a in args]
    out = call(*args)
    with forward_ad.dual_level():
        g = forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(out, args, g)


@pytest.mark.parametrize("name", CALLS)
def test_a_lazily_negated_operand_counts_with_its_sign(name):
    call, args = operands()[name]
    for i, a in enumerate(args):
        lazy = torch._neg_view(-a)
        assert lazy.is_neg() and torch.equal(call(*args[:i], lazy, *args[i + 1:]), call(*args))
        if name in NODES:
            leaf = (-a).requires_grad_(True)
            grad, = torch.autograd.grad(call(*args[:i], torch._neg_view(leaf), *args[i + 1:]).sum(), leaf)
            plain = a.clone().requires_grad_(True)
            want, = torch.autograd.grad(call(*args[:i], plain, *args[i + 1:]).sum(), plain)
            assert torch.equal(grad, -want)


@pytest.mark.parametrize("name", CALLS)
def test_zeros_that_were_never_written(name):
    call, args = operands()[name]
    for i, a in enumerate(args):
        lazy = torch._efficientzerotensor(a.shape, device=DEV)
        want = call(*args[:i], torch.zeros_like(a), *args[i + 1:])
        assert torch.equal(call(*args[:i], lazy, *args[i + 1:]), want)


@pytest.mark.parametrize("name", NODES)
def test_gradients_that_are_negated_or_never_written(name):
    call, args = operands()[name]
    args = [a.requires_grad_(True) for a in args]
    out = call(*args)
    g = torch.randn(out.shape, device=DEV)
    for lazy, plain in ((torch._neg_view(-g), g), (torch._efficientzerotensor(g.shape, device=DEV), torch.zeros_like(g))):
        got = torch.autograd.grad(out, args, lazy, retain_graph=True)
        for a, b in zip(got, torch.autograd.grad(out, args, plain, retain_graph=True)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("what", ("slot", "offset"))
@pytest.mark.parametrize("weighted", (True, False))
def test_an_order_changed_in_place_is_noticed(what, weighted):
    gen = torch.Generator(device=DEV).manual_seed(1)
    x, y = (torch.randn(n, 24, device=DEV, generator=gen).requires_grad_(True) for n in (40, 80))
    weight = torch.rand(40, 2, device=DEV, generator=gen) if weighted else None
    order = be.expert_order(torch.randint(0, 3, (40, 2), device=DEV, generator=gen), 3)
    outs = be.rows_to_experts(x, order), be.rows_from_experts(y, order, weight)
    getattr(order, what).fill_(0)
    for out, leaf in zip(outs, (x, y)):
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(out.sum(), leaf)


def test_an_order_that_does_not_fit_is_refused_by_the_calls():
    x, y, weight = torch.randn(6, 8, device=DEV), torch.randn(12, 8, device=DEV), torch.ones(6, 2, device=DEV)
    good = be.expert_order(torch.zeros(6, 2, dtype=torch.int64, device=DEV), 4)
    for slot, offset in ((good.slot[:11], good.offset), (good.slot, good.offset[:4]), (good.slot.long(), good.offset),
                         (good.slot.cpu(), good.offset), (good.slot, good.offset.cpu())):
        order = be.ExpertOrder(slot, good.pair, offset, 6, 2, 4)
        for call in (lambda: be.rows_to_experts(x, order), lambda: be.rows_from_experts(y, order),
                     lambda: be.rows_from_experts(y, order, weight)):
            with pytest.raises(ValueError):
                call()


def test_kept_rows_that_are_not_whole_are_refused_by_the_calls():
    x, g = torch.randn(6, 128, device=DEV), torch.randn(6, 64, device=DEV)
    plain, gated = be.pack_rows(x), be.gated_pack(x)[1]
    for kept, call in ((plain, be.unpack_rows), (gated, lambda k: be.gated_grad(k, g))):
        for codes, scale in ((kept.codes, kept.scale[:5]), (kept.codes[:, ::2], kept.scale), (kept.codes, kept.scale.cpu()),
                             (kept.codes, kept.scale.half()), (kept.codes.int(), kept.scale)):
            with pytest.raises(ValueError):
                call(be.PackedRows(codes, scale, 64, x.dtype))


def test_a_gate_that_would_lose_its_gradient_is_refused():
    x = torch.randn(6, 128, device=DEV, requires_grad=True)
    for of in (x, x * 2):
        with pytest.raises(RuntimeError, match="records no gradient"):
            be.gated_pack(of)
        with pytest.raises(RuntimeError, match="records no gradient"):
            be.gated_pack(of, keep=False)
    want, _ = be.gated_pack(x.detach())
    with torch.no_grad():
        assert torch.equal(be.gated_pack(x)[0], want)


def test_routing_under_autocast_and_in_half_precision():
    torch.manual_seed(2)
    layer = hiscache.ExpertMLP(64, 32, 8, 2, device=DEV)
    x = torch.randn(400, 64, device=DEV)
    expert, weight = layer.route(x)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        again, weight_again = layer.route(x)
    assert torch.equal(expert, again) and torch.equal(weight, weight_again)
    half = layer.bfloat16()
    rows = x.bfloat16().requires_grad_(True)
    out = half(rows)
    out.float().sum().backward()
    assert out.dtype == torch.bfloat16 and all(bool(torch.isfinite(p.grad).all()) for p in (rows, *half.parameters()))
    assert half.router.grad.dtype == torch.bfloat16


@pytest.mark.parametrize("n,k,E", ((1921, 1, 963), (256, 8, 1024), (2047, 1, 1024), (7681, 1, 1000), (1024, 8, 1024), (8191, 1, 1024)))
def test_an_order_by_one_block_with_many_experts(n, k, E):
    """Sixteen waves with a row of counters each: more than 64 KB of LDS."""
    gen = torch.Generator(device=DEV).manual_seed(n)
    expert = torch.randint(-1, E, (n, k), device=DEV, generator=gen)
    order, flat = be.expert_order(expert, E), expert.reshape(-1)
    live = int((flat >= 0).sum())
    pair = torch.sort(torch.where(flat < 0, E, flat), stable=True)[1]
    place = torch.empty_like(pair)
    place[pair] = torch.arange(n * k, device=DEV)
    assert torch.equal(order.pair[:live].long(), pair[:live]) and bool((order.pair[live:] == -1).all())
    assert torch.equal(order.slot.long(), torch.where(flat < 0, -1, place))
    assert torch.equal(order.offset, torch.searchsorted(torch.sort(flat)[0], torch.arange(E + 1, device=DEV)) - (n * k - live))


@pytest.mark.parametrize("dtype,most", ((torch.float32, 0.5001), (torch.float16, 0.57), (torch.bfloat16, 1.0)))
@pytest.mark.parametrize("group", (32, 64, 128))
def test_how_far_off_rows_in_8_bits_read_back(dtype, most, group):
    """Half a scale, 127 x 6 x 2^-24 scales of rounding in fp32, and half a unit of the type on up to 127 scales: 2^-11 of them in
    fp16 (0.0621), 2^-8 in bf16 (0.4961)."""
    gen = torch.Generator(device=DEV).manual_seed(group)
    x = (torch.randn(20_000, 2 * group + 7, device=DEV, generator=gen) * torch.exp(torch.randn(20_000, 1, device=DEV, generator=gen))).to(dtype)
    kept = be.pack_rows(x, group)
    off = (be.unpack_rows(kept).double() - x.double()).abs()
    scale = kept.scale.double().repeat_interleave(group, 1)[:, :x.shape[1]]
    assert bool((off <= most * scale).all())


def test_an_order_made_in_inference_mode():
    gen = torch.Generator(device=DEV).manual_seed(1)
    expert = torch.randint(0, 3, (40, 2), device=DEV, generator=gen)
    x, w = torch.randn(40, 24, device=DEV, generator=gen).requires_grad_(True), torch.rand(40, 2, device=DEV, generator=gen)
    with torch.inference_mode():
        made = be.expert_order(expert, 3)
    grads = []
    for order in (be.expert_order(expert, 3), made):
        out = be.rows_from_experts(be.rows_to_experts(x, order), order, w)
        grads.append(torch.autograd.grad(out.square().sum(), x)[0])
    assert torch.equal(*grads)
