"""Routing by scores: sigmoid or softmax, a bias in the choice, groups of experts; against the definition in 64 bits."""
import math

import pytest
import torch

import hiscache
import hiscache_backend as be

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def reference(logits, k, normalize=True, score="softmax", bias=None, num_group=1, top_group=1, scale=1.0):
    """(expert, weight) in fp64 on the CPU, and the weights as a differentiable function of the logits."""
    l = logits.detach().double().cpu()
    bias = None if bias is None else bias.detach().double().cpu()
    n, E = l.shape
    leaf = l.clone().requires_grad_(True)
    shut = torch.isneginf(l)
    whole = torch.where(shut.all(1, keepdim=True), torch.zeros_like(leaf), leaf)
    s = torch.sigmoid(leaf) if score == "sigmoid" else torch.softmax(whole, 1)
    c = s.detach() + (0 if bias is None else bias)
    c = torch.where(shut, -math.inf, c)
    shut = torch.isneginf(c)
    order = c if bias is not None else torch.where(shut, -math.inf, l)
    if num_group > 1:
        best = torch.sort(c.view(n, num_group, -1), dim=2, descending=True)[0][:, :, :2]
        rank = torch.where(torch.isneginf(best), 0.0, best).sum(2)
        rank = torch.where(torch.isneginf(best[:, :, 0]), -math.inf, rank)
        keep = torch.sort(rank, dim=1, descending=True, stable=True)[1][:, :top_group]
        out = torch.ones(n, num_group, dtype=torch.bool).scatter_(1, keep, False)
        order = torch.where(out.repeat_interleave(E // num_group, 1), -math.inf, order)
    value, expert = torch.sort(order, dim=1, descending=True, stable=True)
    value, expert = value[:, :k], expert[:, :k]
    none = torch.isneginf(value)
    picked = torch.where(none, 0.0, s.gather(1, expert))
    total = picked.sum(1, keepdim=True) if normalize else torch.ones(n, 1, dtype=torch.float64)
    weight = scale * picked / torch.where(total == 0, 1.0, total)
    return torch.where(none, -1, expert), weight, leaf


# Weights: exp and its argument's rounding (|l - max| <= 64: 64 * 2^-24), a sum of up to 1024 terms of that exactness added in 64 bits or
# up to 32 added in 32 (32 * 2^-24), a quotient and a factor (2^-23).
OFF = 100 * 2.0 ** -23


def check(logits, k, **how):
    expert, weight = be.route_rows(logits, k, **how)
    want, w, _ = reference(logits, k, **how)
    assert torch.equal(expert.cpu(), want)
    assert torch.equal(torch.isnan(weight.cpu()), torch.isnan(w))
    w = w.detach()
    off = torch.nan_to_num((weight.cpu().double() - w).abs() - OFF * w.abs())
    assert float(off.max() if off.numel() else 0) <= 2.0 ** -149
    return expert, weight


SHAPES = [(1, 1, 1, 1, 1), (1, 2, 1, 1, 2), (3, 7, 1, 1, 3), (70, 8, 2, 1, 2), (65, 16, 4, 2, 4), (129, 60, 6, 3, 6),
          (33, 64, 8, 4, 8), (500, 64, 1, 1, 4), (20, 64, 64, 9, 9), (40, 96, 32, 5, 12), (17, 250, 5, 2, 8),
          (300, 256, 8, 4, 8), (9, 511, 7, 3, 32), (5, 1024, 64, 10, 32), (2, 1023, 1, 1, 17), (6000, 40, 1, 1, 5),
          (140_001, 12, 3, 2, 3), (70_001, 66, 1, 1, 8), (20_000, 130, 2, 1, 2)]


@pytest.mark.parametrize("dtype", (torch.float32, torch.float16, torch.bfloat16))
@pytest.mark.parametrize("score", ("sigmoid", "softmax"))
@pytest.mark.parametrize("n,E,G,top,k", SHAPES)
def test_choices_and_weights(n, E, G, top, k, score, dtype):
    gen = torch.Generator(device=DEV).manual_seed(n + E)
    logits = (2 * torch.randn(n, E, generator=gen, device=DEV)).to(dtype)
    logits[torch.rand(n, E, generator=gen, device=DEV) < 0.1] = -math.inf
    logits[::7] = -math.inf
    bias = 0.1 * torch.randn(E, generator=gen, device=DEV)
    for b in (bias, None):
        for normalize, scale in ((True, 2.5), (False, 1.0)):
            check(logits, k, score=score, bias=b, num_group=G, top_group=top, normalize=normalize, scale=scale)


@pytest.mark.parametrize("score", ("sigmoid", "softmax"))
@pytest.mark.parametrize("G,top", ((1, 1), (4, 2)))
@pytest.mark.parametrize("sign", (1, -1))
def test_ties_go_to_the_lowest_index(score, G, top, sign):
    gen = torch.Generator(device=DEV).manual_seed(5)
    logits = sign * torch.randint(0, 4, (3000, 64), generator=gen, device=DEV).float() / 4       # zeros among them
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        for bias in (None, torch.zeros(64, device=DEV), torch.full((64,), -3.0, device=DEV),
                     torch.randint(0, 2, (64,), generator=gen, device=DEV).float() / 8):
            check(logits.to(dtype), 6, score=score, bias=bias, num_group=G, top_group=top)
    same = torch.full((7, 64), -0.0, device=DEV)
    same[:, ::2] = 0.0
    assert check(same, 6, score=score, bias=torch.zeros(64, device=DEV))[0][0].tolist() == list(range(6))
    assert check(same, 6, score=score, num_group=G, top_group=top)[0][0].tolist() == list(range(6))


def test_sums_that_32_bits_cannot_tell_apart():
    """Pairs of experts whose scores and biases add up to nearly the same, one way or the other by 2^-30 or so."""
    gen = torch.Generator(device=DEV).manual_seed(6)
    n, E = 4000, 64
    logits = torch.randn(n, E, generator=gen, device=DEV)
    s = torch.sigmoid(logits.double())
    bias = torch.zeros(E, device=DEV)
    # within a row experts come in twins: the second one's logit makes up for another bias
    bias[1::2] = 0.0625
    twin = torch.logit((s[:, ::2] - 0.0625).clamp(min=0.01)).float()
    logits[:, 1::2] = twin
    c = torch.sigmoid(logits.double()) + bias.double()
    gap = (c[:, ::2] - c[:, 1::2]).abs()
    assert float(((gap < 2.0 ** -24) & (gap > 0)).float().mean()) > 0.5
    for G, top in ((1, 1), (8, 3)):
        check(logits, 8, score="sigmoid", bias=bias, num_group=G, top_group=top)
        check(logits, 7, score="sigmoid", bias=bias, num_group=G, top_group=top)


def test_logits_that_differ_in_their_last_bits():
    """Without a bias every bit of an fp32 logit counts; lists of up to 1024 experts give ten of them to the index."""
    for E, k in ((64, 4), (256, 8), (1024, 32)):
        gen = torch.Generator(device=DEV).manual_seed(E)
        base = torch.randn(200, 1, generator=gen, device=DEV).abs() + 0.5
        step = torch.stack([torch.randperm(E, generator=gen, device=DEV) for _ in range(200)])
        for sign in (1, -1):
            logits = sign * (base.view(torch.int32) + step.to(torch.int32)).view(torch.float32)
            for score in ("sigmoid", "softmax"):
                check(logits, k, score=score, scale=2.0)
    tiny = (torch.randperm(64, device=DEV).to(torch.int32) + 1).view(1, 64).view(torch.float32)   # below fp32's normal numbers
    check(tiny, 8, score="sigmoid")


@pytest.mark.parametrize("dtype", (torch.float32, torch.float16, torch.bfloat16))
@pytest.mark.parametrize("score", ("sigmoid", "softmax"))
def test_masks_of_the_lowest_value_and_saturated_scores(score, dtype):
    gen = torch.Generator(device=DEV).manual_seed(7)
    logits = torch.randn(600, 32, generator=gen, device=DEV).to(dtype)
    logits[torch.rand(600, 32, generator=gen, device=DEV) < 0.9] = torch.finfo(dtype).min
    logits[:50] = torch.finfo(dtype).min
    logits[50:60, 3:] = -math.inf
    check(logits, 4, score=score, num_group=1)
    check(logits, 4, score=score, num_group=4, top_group=2, normalize=score == "softmax")
    for low in (-math.inf, torch.finfo(torch.float32).min):
        bias = torch.zeros(32, device=DEV)
        bias[::3] = low
        check(logits, 4, score=score, bias=bias)
        check(logits, 4, score=score, bias=bias, num_group=4, top_group=3)
    if score == "sigmoid":
        # scores of 0 and 1 to the last bit: with a bias they are equal numbers
        wide = (40 * torch.randn(600, 32, generator=gen, device=DEV)).to(dtype)
        check(wide, 4, score=score, normalize=False, bias=torch.linspace(0, 1, 32, device=DEV))
        expert, weight = be.route_rows(torch.full((3, 8), -200.0, device=DEV).to(dtype), 2, score=score)
        # sigma(-200) is 0 in 32 bits, but not its share: sigma(-200) / (2 sigma(-200)) = 1 / 2
        assert expert.tolist() == [[0, 1]] * 3 and weight.tolist() == [[0.5, 0.5]] * 3
        expert, weight = be.route_rows(torch.full((3, 8), -900.0, device=DEV).to(dtype), 2, score=score)
        assert expert.tolist() == [[0, 1]] * 3 and weight.tolist() == [[0.0, 0.0]] * 3     # exp(-900) is 0 in 64 bits


def test_infinities_and_nan():
    gen = torch.Generator(device=DEV).manual_seed(8)
    logits = torch.randn(40, 16, generator=gen, device=DEV)
    logits[3, 5] = math.nan
    logits[4, 2] = math.inf
    logits[5, [1, 9]] = math.inf
    logits[6, 7], logits[6, 8] = math.inf, math.nan
    logits[7, 3] = -torch.tensor(math.nan)
    logits[8, 4] = torch.tensor([-1], dtype=torch.int32).view(torch.float32)[0]        # a NaN of all bits
    bias = torch.zeros(16, device=DEV)
    for b in (None, bias):
        for G, top in ((1, 1), (4, 2)):
            expert, weight = be.route_rows(logits, 4, score="sigmoid", bias=b, num_group=G, top_group=top, normalize=False)
            assert expert[3, 0] == 5 and expert[4, 0] == 2 and expert[5, :2].tolist() == [1, 9]
            assert expert[6, :2].tolist() == [8, 7] and expert[7, 0] == 3 and expert[8, 0] == 4
            assert weight[4, 0] == 1 and weight[5, :2].tolist() == [1, 1] and bool(torch.isnan(weight[[3, 6, 7, 8], 0]).all())
            assert int(torch.isnan(weight).sum()) == 4
            w = be.route_rows(logits, 4, score="softmax", bias=b, num_group=G, top_group=top, scale=2.0)[1]
            assert bool(torch.isnan(w[3:9]).all()) and not bool(torch.isnan(w[9:]).any()) and not bool(torch.isnan(w[:3]).any())
    bias[6], bias[7] = math.inf, math.nan
    expert, weight = be.route_rows(logits[9:], 4, score="sigmoid", bias=bias, normalize=False)
    assert expert[:, :2].tolist() == [[7, 6]] * 31 and not bool(torch.isnan(weight).any())


@pytest.mark.parametrize("dtype", (torch.float32, torch.float16, torch.bfloat16))
@pytest.mark.parametrize("score,normalize", (("sigmoid", True), ("sigmoid", False), ("softmax", True), ("softmax", False)))
@pytest.mark.parametrize("n,E,G,top,k", ((1, 4, 1, 1, 2), (70, 64, 8, 4, 8), (301, 60, 6, 2, 7), (40, 250, 5, 5, 32), (4000, 9, 3, 2, 4)))
def test_gradient(n, E, G, top, k, score, normalize, dtype):
    gen = torch.Generator(device=DEV).manual_seed(n)
    logits = (2 * torch.randn(n, E, generator=gen, device=DEV)).to(dtype)
    logits[torch.rand(n, E, generator=gen, device=DEV) < 0.2] = -math.inf
    logits[::5] = -math.inf
    bias = 0.1 * torch.randn(E, generator=gen, device=DEV)
    g = torch.randn(n, k, generator=gen, device=DEV)
    leaf = logits.clone().requires_grad_(True)
    how = dict(score=score, normalize=normalize, bias=bias, num_group=G, top_group=top, scale=2.5)
    expert, weight = be.route_rows(leaf, k, **how)
    assert not expert.requires_grad and weight.requires_grad
    weight.backward(g)
    want, w, ref = reference(logits, k, **how)
    w.backward(torch.where(want < 0, 0.0, g.double().cpu()))
    want = torch.nan_to_num(ref.grad)
    assert leaf.grad.dtype == dtype
    # differences of numbers as large as scale * max |g|, each exact to OFF, times a factor of at most one (normalised: over S, of which s is
    # a part); rounded to the type
    most = 2.5 * g.abs().max(1, keepdim=True)[0].double().cpu()
    off = (leaf.grad.double().cpu() - want).abs()
    bound = 4 * OFF * most + torch.finfo(dtype).eps / 2 * want.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert bool((off <= bound).all()), float((off - bound).max())
    assert bool((leaf.grad[torch.isneginf(logits)] == 0).all())


@pytest.mark.parametrize("score,normalize", (("sigmoid", True), ("sigmoid", False), ("softmax", True), ("softmax", False)))
def test_gradient_against_differences(score, normalize):
    gen = torch.Generator(device=DEV).manual_seed(1)
    logits = torch.randn(3, 8, generator=gen, device=DEV)
    g = torch.randn(3, 3, generator=gen, device=DEV)
    how = dict(score=score, normalize=normalize, num_group=4, top_group=3, scale=1.5)
    leaf = logits.clone().requires_grad_(True)
    be.route_rows(leaf, 3, **how)[1].backward(g)
    h = 2.0 ** -6
    for i in range(3):
        for e in range(8):
            up, down = logits.clone(), logits.clone()
            up[i, e] += h
            down[i, e] -= h
            (eu, wu), (ed, wd) = be.route_rows(up, 3, **how), be.route_rows(down, 3, **how)
            assert torch.equal(eu, ed)                      # (no other choice within h)
            slope = float(((wu - wd).double() * g.double()).sum()) / (2 * h)
            # h^2 / 6 of a third derivative below 1.5 * 4 * 3 * max |g|, and the weights' own 2^-23 over h
            assert abs(slope - float(leaf.grad[i, e])) <= (h * h * 3 + 2.0 ** -16) * float(g.abs().max()) * 3


def test_other_views_streams_and_nothing_at_all():
    gen = torch.Generator(device=DEV).manual_seed(2)
    flat = torch.randn(1 + 500 * 64, generator=gen, device=DEV)
    logits = flat[1:].view(500, 64)                          # off every multiple of 16 bytes
    bias = torch.randn(65, generator=gen, device=DEV)[1:] / 8
    how = dict(score="sigmoid", bias=bias, num_group=8, top_group=4)
    want = be.route_rows(logits.clone(), 8, score="sigmoid", bias=bias.clone(), num_group=8, top_group=4)
    got = check(logits, 8, **how)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = be.route_rows(logits, 8, **how)
    side.synchronize()
    assert torch.equal(other[0], want[0]) and torch.equal(other[1], want[1])
    leaf = torch.zeros(0, 64, device=DEV, requires_grad=True)
    expert, weight = be.route_rows(leaf, 8, **how)
    assert expert.shape == weight.shape == (0, 8)
    weight.sum().backward()
    assert leaf.grad.shape == (0, 64)
    leaf = logits.clone().requires_grad_(True)
    assert be.route_rows(leaf, 8, **how)[0].grad_fn is None
    with pytest.raises(RuntimeError):
        _, weight = be.route_rows(leaf, 8, **how)
        torch.autograd.grad(torch.autograd.grad(weight.sum(), leaf, create_graph=True)[0].sum(), leaf)


def test_recorded_and_replayed():
    gen = torch.Generator(device=DEV).manual_seed(3)
    bias = torch.zeros(64, device=DEV)
    logits = torch.zeros(700, 64, device=DEV, requires_grad=True)
    g = torch.randn(700, 4, generator=gen, device=DEV)
    how = dict(score="sigmoid", bias=bias, num_group=8, top_group=3, scale=2.0)

    def step():
        expert, weight = be.route_rows(logits, 4, **how)
        return expert, weight, torch.autograd.grad(weight, logits, g)[0]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            logits.copy_(torch.randn(700, 64, generator=gen, device=DEV))
            bias.copy_(torch.randn(64, generator=gen, device=DEV) / 8)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


def test_refusals():
    logits = torch.zeros(4, 12, device=DEV)
    bias = torch.zeros(12, device=DEV)
    for bad in (dict(score="tanh"), dict(num_group=5), dict(num_group=4, top_group=5), dict(num_group=4, top_group=0),
                dict(num_group=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan),
                dict(bias=bias.half()), dict(bias=bias[:5]), dict(bias=bias.view(1, 12)), dict(bias=bias[::2]),
                dict(bias=bias.clone().requires_grad_(True)), dict(num_group=6, top_group=1)):
        with pytest.raises(ValueError):
            be.route_rows(logits, 3, **bad)
    with pytest.raises(RuntimeError, match="no CPU path"):
        be.route_rows(logits, 3, bias=bias.cpu())
    with pytest.raises(ValueError):
        be.route_rows(torch.zeros(4, 130, device=DEV), 3, score="sigmoid", num_group=65, top_group=3)
    with torch.no_grad():
        be.route_rows(logits, 3, bias=bias.clone().requires_grad_(True))


# ----------------------------------------------------------------------------- the layer
def test_a_balanced_layer():
    torch.manual_seed(0)
    layer = hiscache.ExpertMLP(32, 32, 8, 2, score="sigmoid", balance=True, scale=2.0, device=DEV)
    x = torch.randn(4000, 32, device=DEV) + 0.5              # rows that lean one way: some experts have far more than others
    with torch.no_grad():
        layer.router.mul_(2)

    def loads():
        order = be.expert_order(layer.route(x)[0], 8)
        return (order.offset[1:] - order.offset[:-1]).float()

    layer.balance_step(0.1)                                  # nothing has been routed yet
    assert bool((layer.balance_bias == 0).all())
    before = loads()
    layer.eval()
    layer(x)
    layer.balance_step(0.1)
    assert bool((layer.balance_bias == 0).all())             # (not by an evaluation)
    layer.train()
    for _ in range(60):
        layer(x)
        load, bias = loads(), layer.balance_bias.clone()
        layer.balance_step(0.01)
        assert torch.equal(layer.balance_bias, bias + 0.01 * torch.sign(load.mean() - load))
    after = loads()
    assert float(after.max() / after.mean()) < 1.1 < float(before.max() / before.mean())
    # no part of the weights, and no gradient
    expert, weight = layer.route(x)
    s = torch.sigmoid(x @ layer.router.t()).gather(1, expert)
    assert torch.allclose(weight, 2 * s / s.sum(1, keepdim=True), rtol=2.0 ** -16)
    layer(x).sum().backward()
    assert "balance_bias" in layer.state_dict() and all(p.grad is not None for p in layer.parameters())
    half = layer.bfloat16()
    assert half.balance_bias.dtype == torch.float32 and torch.equal(half.balance_bias, layer.balance_bias)
    assert half.w_in.dtype == torch.bfloat16
    half(x.bfloat16()).sum().backward()
    with pytest.raises(RuntimeError, match="balance=True"):
        hiscache.ExpertMLP(32, 32, 8, 2, device=DEV).balance_step()
    for bad in (dict(score="tanh"), dict(num_group=3), dict(num_group=4, top_group=5), dict(num_group=8, top_group=1), dict(scale=0)):
        with pytest.raises(ValueError):
            hiscache.ExpertMLP(32, 32, 8, 2, **bad)


def test_a_layer_of_groups():
    torch.manual_seed(1)
    layer = hiscache.ExpertMLP(32, 48, 12, 3, score="sigmoid", num_group=4, top_group=2, device=DEV)
    x = torch.randn(300, 32, device=DEV)
    allowed = torch.ones(12, dtype=torch.bool, device=DEV)
    allowed[3:6] = False                                     # a whole group
    expert, weight = layer.route(x, allowed)
    assert not bool(((expert >= 3) & (expert < 6)).any())
    assert int(torch.tensor([len(set(row)) for row in (expert // 3).tolist()]).max()) <= 2
    out = layer(x, allowed=allowed)
    h = torch.einsum("nc,ehc->neh", x, layer.w_in)
    h = torch.nn.functional.silu(h[..., :48]) * h[..., 48:]
    y = torch.einsum("neh,edh->ned", h, layer.w_out)
    want = (y.gather(1, expert.unsqueeze(2).expand(-1, -1, 32)) * weight.unsqueeze(2)).sum(1)
    assert torch.allclose(out, want, rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("k", (1, 4, 11))
def test_shares_of_scores_that_32_bits_do_not_hold(k):
    """Normalised sigmoid weights go by the formula down to logits of -700, in the gradient as well."""
    gen = torch.Generator(device=DEV).manual_seed(k)
    logits = torch.randn(700, 24, generator=gen, device=DEV) - torch.arange(700, device=DEV).unsqueeze(1) * 0.98
    logits[650:, 12:] = 3.0                                  # among others that are nothing to them
    check(logits, k, score="sigmoid", num_group=1, scale=2.0)
    check(logits, k, score="sigmoid", num_group=4, top_group=2, scale=2.0)
    g = torch.randn(700, k, generator=gen, device=DEV)
    leaf = logits.clone().requires_grad_(True)
    be.route_rows(leaf, k, score="sigmoid", scale=2.0)[1].backward(g)
    _, w, ref = reference(logits, k, score="sigmoid", scale=2.0)
    w.backward(g.double().cpu())
    off = (leaf.grad.double().cpu() - ref.grad).abs()
    assert bool((off <= 8 * OFF * g.abs().max(1, keepdim=True)[0].double().cpu()).all())


def test_shares_of_a_softmax_among_experts_that_are_nothing_to_its_largest():
    """A bias that sends rows to experts 90 to 690 below the largest logit: their shares, and their gradients."""
    gen = torch.Generator(device=DEV).manual_seed(2)
    logits = torch.randn(600, 16, generator=gen, device=DEV)
    logits[:, :8] += 90 + torch.arange(600, device=DEV).unsqueeze(1).float()
    bias = torch.zeros(16, device=DEV)
    bias[:8] = -2.0
    expert, weight = check(logits, 3, score="softmax", bias=bias)
    assert bool((expert >= 8).all()) and bool((weight > 0).all())
    g = torch.randn(600, 3, generator=gen, device=DEV)
    leaf = logits.clone().requires_grad_(True)
    be.route_rows(leaf, 3, bias=bias)[1].backward(g)
    _, w, ref = reference(logits, 3, bias=bias)
    w.backward(g.double().cpu())
    off = (leaf.grad.double().cpu() - ref.grad).abs()
    assert bool((off <= 8 * OFF * g.abs().max(1, keepdim=True)[0].double().cpu()).all())
    # masked ones have no shares
    logits[:, 8:] = torch.finfo(torch.float32).min
    leaf = logits.clone().requires_grad_(True)
    expert, weight = be.route_rows(leaf, 3, bias=bias)
    weight.backward(g)
    assert bool((expert >= 8).all()) and bool((weight == 0).all()) and bool((leaf.grad == 0).all())


@pytest.mark.parametrize("how", (dict(score="sigmoid"), dict(score="sigmoid", normalize=False), dict(scale=2.0), dict(scale=2.0, normalize=False)))
def test_what_reaches_the_weights_of_missing_experts_is_left_alone(how):
    gen = torch.Generator(device=DEV).manual_seed(8)
    logits = torch.randn(300, 20, generator=gen, device=DEV)
    logits[:, 3:] = -math.inf
    g = torch.randn(300, 12, generator=gen, device=DEV)
    grads = []
    for value in (0.0, math.nan, math.inf):
        leaf = logits.clone().requires_grad_(True)
        expert, weight = be.route_rows(leaf, 12, **how)
        assert bool((expert[:, 3:] == -1).all()) and not bool(weight[:, 3:].any())
        weight.backward(torch.where(expert < 0, value, g))
        grads.append(leaf.grad)
    assert bool(torch.isfinite(grads[0]).all()) and all(torch.equal(x, grads[0]) for x in grads[1:])


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("score", ("sigmoid", "softmax"))
def test_the_only_choice_of_a_row_has_weight_1_and_no_gradient(score, dtype):
    """Divided by itself a score is 1 whatever the logit is, to the last bit, in the gradient as well."""
    gen = torch.Generator(device=DEV).manual_seed(4)
    logits = (9 * torch.randn(4000, 40, generator=gen, device=DEV)).to(dtype)
    logits[2000:, :39] = -math.inf                           # of four choices three name no expert
    bias = torch.randn(40, generator=gen, device=DEV)
    for rows, k in ((logits[:2000], 1), (logits[2000:], 4)):
        leaf = rows.clone().requires_grad_(True)
        expert, weight = be.route_rows(leaf, k, score=score, bias=bias)
        weight.backward(torch.randn(2000, k, generator=gen, device=DEV))
        assert bool((weight[:, 0] == 1).all()) and not bool(weight[:, 1:].any()) and not bool(leaf.grad.any())
