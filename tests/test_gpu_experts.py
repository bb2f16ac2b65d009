"""Routing, the order by expert and the rows' way there and back, against plain implementations in 64 bits.

u is half a unit of fp32.  A result kept in a narrower type may be off by half a unit of that type besides."""
import math

import pytest
import torch

import hiscache_backend as be

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
TYPES = (torch.float32, torch.float16, torch.bfloat16)
# half a unit of the type's values near 1, and of its smallest ones
HALF = {torch.float32: (0.0, 2.0 ** -150), **{t: (torch.finfo(t).eps / 2, torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2) for t in TYPES[1:]}}


def close(got, want, bound):
    rel, least = HALF[got.dtype]
    off = (got.double() - want).abs()
    # the narrow rounding is of the computed value, which is off by up to the bound already
    assert bool((off <= bound + rel * (want.abs() + bound) + least).all()), float((off - bound - rel * want.abs()).max())


def route64(logits, k, normalize):
    """Experts, weights, and all probabilities, by the definition."""
    l = logits.double()
    p = torch.nan_to_num(torch.softmax(l, 1), nan=0.0) if not bool(torch.isnan(l).any()) else torch.softmax(l, 1)
    order = sorted_by_value(logits, k)
    on = ~torch.isneginf(l.gather(1, order))
    w = torch.where(on, p.gather(1, order), 0.0)
    if normalize:
        w = torch.where(on, w / w.sum(1, keepdim=True), 0.0)
    return torch.where(on, order, -1), w, p


def sorted_by_value(logits, k):
    return torch.sort(logits.double().cpu(), dim=1, descending=True, stable=True).indices[:, :k].to(logits.device)


def logits_for(gen, n, E, dtype, masked):
    l = 3 * torch.randn(n, E, device=DEV, generator=gen)
    l = (l * 4).round() / 4 if n % 2 else l                   # many equal values in a row
    l[torch.rand(n, E, device=DEV, generator=gen) < masked] = -math.inf
    if masked:
        l[0] = -math.inf
        l[-1, : E - 1] = -math.inf
    return l.to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,E,k", ((1, 1, 1), (5, 2, 2), (33, 7, 3), (64, 8, 8), (31, 9, 4), (257, 16, 2), (129, 33, 6), (1001, 64, 4),
                                   (65, 65, 32), (40, 100, 10), (17, 200, 8), (9, 300, 32), (6, 1000, 5), (3, 1024, 32)))
@pytest.mark.parametrize("normalize", (True, False))
@pytest.mark.parametrize("masked", (0.0, 0.4))
def test_route_and_its_gradient(dtype, n, E, k, normalize, masked):
    gen = torch.Generator(device=DEV).manual_seed(n * 1000 + E)
    logits = logits_for(gen, n, E, dtype, masked).requires_grad_(True)
    expert, weight = be.route_rows(logits, k, normalize=normalize)
    want_e, w, p = route64(logits.detach(), k, normalize)
    assert torch.equal(expert, want_e) and weight.dtype == torch.float32
    # the difference to the largest logit is rounded (up to 32 large here), the exponential is off by a unit, a sum of E
    # terms by E half units, the quotient by half a unit
    rel = (E + 2 * 32 + 8) * 2 * U
    close(weight.detach(), w, rel * w)
    g = torch.randn(n, k, device=DEV, generator=gen)
    grad, = torch.autograd.grad(weight, logits, g)
    on = want_e >= 0
    at, g64 = want_e.clamp(min=0), torch.where(on, g.double(), 0.0)
    t, size = (w * g64).sum(1, keepdim=True), (w * g64.abs()).sum(1, keepdim=True)
    dense_g = torch.zeros_like(p).scatter_add_(1, at, g64)
    dense_w = torch.zeros_like(p).scatter_add_(1, at, w)
    base = dense_w if normalize else p
    close(grad, base * (dense_g - t), 3 * rel * base * (dense_g.abs() + size))
    assert bool((grad[torch.isneginf(logits)] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_route_ties_lowest_values_and_zeros(dtype):
    low = torch.finfo(dtype).min
    l = torch.tensor([[0.0, -0.0, 0.0, -0.0], [low, low, low, low], [low, 1.0, low, -math.inf], [-0.0, 0.0, 2.0, 2.0]],
                     device=DEV, dtype=dtype)
    expert, weight = be.route_rows(l, 3)
    assert expert.tolist() == [[0, 1, 2], [0, 1, 2], [1, 0, 2], [2, 3, 0]]
    assert weight[2].tolist() == [1.0, 0.0, 0.0] and bool((weight[:2] == weight[0, 0]).all())


@pytest.mark.parametrize("bad", (math.nan, -math.nan, math.inf))
@pytest.mark.parametrize("normalize", (True, False))
@pytest.mark.parametrize("dtype", TYPES)
def test_route_shows_what_is_not_finite(bad, normalize, dtype):
    l = torch.zeros(3, 20, device=DEV, dtype=dtype)
    l[1, 7] = bad
    l.requires_grad_(True)
    expert, weight = be.route_rows(l, 2, normalize=normalize)
    assert expert.tolist() == [[0, 1], [7, 0], [0, 1]]
    assert bool(torch.isnan(weight[1]).all()) and bool(torch.isfinite(weight[::2]).all())
    grad, = torch.autograd.grad(weight, l, torch.ones_like(weight))
    assert bool(torch.isnan(grad[1]).any()) and bool(torch.isfinite(grad[::2]).all())


@pytest.mark.parametrize("normalize", (True, False))
def test_route_gradient_against_differences(normalize):
    gen = torch.Generator(device=DEV).manual_seed(5)
    l = torch.randn(200, 24, device=DEV, generator=gen)
    l += 0.5 * torch.arange(24, device=DEV)                   # far enough apart that a small step changes no choice
    d, g = torch.randn(200, 24, device=DEV, generator=gen), torch.randn(200, 4, device=DEV, generator=gen)
    step = 2.0 ** -9
    up, weight_up = be.route_rows(l + step * d, 4, normalize=normalize)
    down, weight_down = be.route_rows(l - step * d, 4, normalize=normalize)
    same = (up == down).all(1)
    assert int(same.sum()) > 150
    slope = ((weight_up.double() - weight_down.double()) * g).sum(1) / (2 * step)
    a = l.clone().requires_grad_(True)
    grad, = torch.autograd.grad(be.route_rows(a, 4, normalize=normalize)[1], a, g)
    # rounding of two weights of up to 1 over the step, and the third derivative (at most 1 for a softmax) times step^2 / 6
    size = g.abs().sum(1).double()
    bound = size * (2 * 100 * U / (2 * step) + (d.abs().amax(1).double() * 2) ** 3 * step ** 2)
    assert bool(((slope - (grad.double() * d).sum(1)).abs() <= bound)[same].all())


def order64(expert, E):
    flat = expert.reshape(-1).cpu()
    pairs = [torch.nonzero(flat == e).reshape(-1) for e in range(E)]
    offset = torch.tensor([0] + [p.numel() for p in pairs]).cumsum(0)
    live = torch.cat(pairs)
    pair = torch.full((flat.numel(),), -1, dtype=torch.int32)
    pair[: live.numel()] = live.int()
    slot = torch.full((flat.numel(),), -1, dtype=torch.int32)
    slot[live] = torch.arange(live.numel(), dtype=torch.int32)
    return slot, pair, offset


def choices(gen, n, k, E, dropped):
    e = torch.randint(0, E, (n, k), device=DEV, generator=gen)
    e[torch.rand(n, k, device=DEV, generator=gen) < dropped] = -1
    return e


@pytest.mark.parametrize("n,k,E", ((0, 2, 3), (1, 1, 1), (1, 3, 1024), (63, 1, 5), (64, 1, 64), (65, 3, 7), (1000, 2, 63), (4096, 2, 8),
                                   (4097, 2, 8), (2731, 3, 1024), (30_000, 4, 100), (40_001, 7, 1024), (700_001, 1, 2)))
@pytest.mark.parametrize("dropped", (0.0, 0.3, 1.0))
def test_order_is_the_stable_sort(n, k, E, dropped):
    gen = torch.Generator(device=DEV).manual_seed(n + E)
    expert = choices(gen, n, k, E, dropped)
    order = be.expert_order(expert, E)
    for got, want in zip((order.slot, order.pair, order.offset), order64(expert, E)):
        assert torch.equal(got.cpu(), want)
    assert (order.rows, order.top_k, order.experts, order.places) == (n, k, E, n * k)


@pytest.mark.parametrize("n", (100, 50_000))
def test_order_of_one_expert_and_of_numbers_out_of_range(n):
    one = be.expert_order(torch.full((n,), 3, dtype=torch.int64, device=DEV), 5)
    assert torch.equal(one.pair, torch.arange(n, dtype=torch.int32, device=DEV)) and one.offset.tolist() == [0, 0, 0, 0, n, n]
    e = torch.arange(n, device=DEV) % 7 - 1
    e[e == 5] = 1 << 40
    e[e == 4] = -(1 << 40)
    got = be.expert_order(e, 4)
    for a, b in zip((got.slot, got.pair, got.offset), order64(e, 4)):
        assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k,E,D", ((1, 1, 1, 1), (1, 2, 3, 5), (7, 3, 4, 47), (130, 2, 8, 64), (33, 5, 6, 100), (61, 8, 9, 172),
                                     (300, 4, 5, 602), (257, 9, 16, 128), (19, 2, 70, 1024), (5, 1, 2, 4100)))
@pytest.mark.parametrize("dropped", (0.0, 0.3, 1.0))
def test_rows_to_experts_and_back(dtype, n, k, E, D, dropped):
    gen = torch.Generator(device=DEV).manual_seed(n * 7 + D)
    order = be.expert_order(choices(gen, n, k, E, dropped), E)
    x, y, g_rows, g_out = (torch.randn(m, D, device=DEV, generator=gen).to(dtype) for m in (n, n * k, n * k, n))
    weight = torch.randn(n, k, device=DEV, generator=gen)
    live, kept = (order.pair >= 0).unsqueeze(1), (order.slot >= 0).view(n, k, 1)
    row, at = order.pair.clamp(min=0).long() // k, order.slot.clamp(min=0).long()

    x.requires_grad_(True)
    rows = be.rows_to_experts(x, order)
    assert torch.equal(rows, torch.where(live, x[row], 0.0).to(dtype))
    picked = torch.where(kept, g_rows.double()[at].view(n, k, D), 0.0)
    close(torch.autograd.grad(rows, x, g_rows)[0], picked.sum(1), k * U * picked.abs().sum(1))

    y.requires_grad_(True)
    weight.requires_grad_(True)
    out = be.rows_from_experts(y, order, weight)
    y64 = torch.where(kept, y.detach().double()[at].view(n, k, D), 0.0)
    term = y64 * weight.detach().double().unsqueeze(2)
    close(out.detach(), term.sum(1), k * U * term.abs().sum(1))
    g_y, g_w = torch.autograd.grad(out, (y, weight), g_out)
    w_at = weight.detach().double().reshape(-1)[order.pair.clamp(min=0).long()].unsqueeze(1)
    want = torch.where(live, w_at * g_out.double()[row], 0.0)
    close(g_y, want, U * want.abs())
    term = y64 * g_out.double().unsqueeze(1)
    close(g_w, term.sum(2), (D + 8) * U * term.abs().sum(2))

    plain = be.rows_from_experts(y, order)
    close(plain.detach(), y64.sum(1), k * U * y64.abs().sum(1))
    assert torch.equal(torch.autograd.grad(plain, y, g_out)[0], torch.where(live, g_out[row], 0.0).to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", (2, 3, 4, 6, 7, 8, 9, 12, 15, 17, 31, 65, 601))
def test_rows_of_every_width(dtype, D):
    """Rows shorter than a wide piece, of whole pieces, and with a last piece that reaches back over the one before."""
    test_rows_to_experts_and_back(dtype, 37, 3, 5, D, 0.3)


@pytest.mark.parametrize("dtype", TYPES)
def test_places_of_no_pair_may_hold_anything(dtype):
    n, k, E, D = 50, 3, 4, 72
    gen = torch.Generator(device=DEV).manual_seed(3)
    order = be.expert_order(choices(gen, n, k, E, 0.4), E)
    y, g = torch.randn(n * k, D, device=DEV, generator=gen).to(dtype), torch.randn(n, D, device=DEV, generator=gen).to(dtype)
    weight = torch.rand(n, k, device=DEV, generator=gen)
    weight[(order.slot < 0).view(n, k)] = math.nan
    clean = torch.where((order.pair >= 0).unsqueeze(1), y, 0.0).to(dtype)
    y[order.pair < 0] = math.nan
    results = []
    for rows in (y, clean):
        rows, w = rows.clone().requires_grad_(True), weight.clone().requires_grad_(True)
        out = be.rows_from_experts(rows, order, w)
        results.append((out.detach(), *torch.autograd.grad(out, (rows, w), g)))
    assert all(torch.equal(a, b) and bool(torch.isfinite(a).all()) for a, b in zip(*results))
    x = torch.randn(n, D, device=DEV).to(dtype).requires_grad_(True)
    grad, = torch.autograd.grad(be.rows_to_experts(x, order), x, y)
    assert bool(torch.isfinite(grad).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_off_the_alignment_of_wide_loads(dtype):
    n, k, E, D = 40, 2, 5, 64
    gen = torch.Generator(device=DEV).manual_seed(1)
    order = be.expert_order(choices(gen, n, k, E, 0.1), E)
    x, y, g = (torch.randn(m, D, device=DEV, generator=gen).to(dtype) for m in (n, n * k, n))
    w = torch.rand(n, k, device=DEV, generator=gen)

    def shifted(t):
        return torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)[1:].view(t.shape).copy_(t)

    def all_of(x, y, g):
        x, y, v = x.requires_grad_(True), y.requires_grad_(True), w.clone().requires_grad_(True)
        rows, out = be.rows_to_experts(x, order), be.rows_from_experts(y, order, v)
        return (rows, out, *torch.autograd.grad((rows, out), (x, y, v), (shifted(y.detach()), g)))

    for a, b in zip(all_of(x, y, g), all_of(shifted(x), shifted(y), shifted(g))):
        close(b.detach(), a.detach().double(), (D + 8) * 2 * U * (1 + a.detach().double().abs()))


def test_gradients_of_the_rows_way_against_differences():
    n, k, E, D = 60, 3, 5, 40
    gen = torch.Generator(device=DEV).manual_seed(8)
    order = be.expert_order(choices(gen, n, k, E, 0.2), E)
    y, w, dy, dw = (torch.randn(s, device=DEV, generator=gen) for s in ((n * k, D), (n, k), (n * k, D), (n, k)))
    g = torch.randn(n, D, device=DEV, generator=gen)
    a, b = y.clone().requires_grad_(True), w.clone().requires_grad_(True)
    gy, gw = torch.autograd.grad(be.rows_from_experts(a, order, b), (a, b), g)
    # linear in each: a step of one loses nothing but rounding
    for grad, d, up, down in ((gy, dy, be.rows_from_experts(y + dy, order, w), be.rows_from_experts(y - dy, order, w)),
                              (gw, dw, be.rows_from_experts(y, order, w + dw), be.rows_from_experts(y, order, w - dw))):
        slope = ((up.double() - down.double()) * g).sum() / 2
        size = (up.abs() + down.abs()).double().mul(g.abs()).sum() + (grad.abs() * d.abs()).double().sum()
        assert abs(float(slope - (grad.double() * d).sum())) <= 32 * U * float(size)


def test_refusals():
    x = torch.randn(6, 8, device=DEV)
    e = torch.zeros(6, 2, dtype=torch.int64, device=DEV)
    order = be.expert_order(e, 4)
    y = torch.randn(12, 8, device=DEV)
    for call in (lambda: be.route_rows(x, 0), lambda: be.route_rows(x, 9), lambda: be.route_rows(x.double(), 2),
                 lambda: be.route_rows(x[0], 1), lambda: be.route_rows(x.t(), 2),
                 lambda: be.route_rows(torch.zeros(2, 1025, device=DEV), 2), lambda: be.route_rows(torch.zeros(2, 64, device=DEV), 33),
                 lambda: be.expert_order(e.int(), 4), lambda: be.expert_order(e, 0), lambda: be.expert_order(e, 1025),
                 lambda: be.expert_order(e.view(3, 2, 2), 4), lambda: be.expert_order(e.t(), 4),
                 lambda: be.rows_to_experts(y, order), lambda: be.rows_to_experts(x.double(), order), lambda: be.rows_to_experts(x[:, :0], order),
                 lambda: be.rows_to_experts(x[:, ::2], order), lambda: be.rows_from_experts(x, order),
                 lambda: be.rows_from_experts(y, order, torch.ones(6, 3, device=DEV)),
                 lambda: be.rows_from_experts(y, order, torch.ones(6, 2, device=DEV).half())):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        be.rows_to_experts(x, e)
    with pytest.raises(RuntimeError):
        be.route_rows(x.cpu(), 2)
    with pytest.raises(RuntimeError):
        be.expert_order(e.cpu(), 4)


def test_no_rows():
    empty = torch.empty(0, 5, device=DEV, requires_grad=True)
    expert, weight = be.route_rows(empty, 2)
    assert expert.shape == weight.shape == (0, 2)
    assert torch.autograd.grad(weight, empty, torch.empty(0, 2, device=DEV))[0].shape == (0, 5)
    order = be.expert_order(expert, 5)
    assert order.offset.tolist() == [0] * 6
    x = torch.empty(0, 3, device=DEV, requires_grad=True)
    rows = be.rows_to_experts(x, order)
    out = be.rows_from_experts(rows, order, weight)
    assert rows.shape == out.shape == (0, 3) and torch.autograd.grad(out.sum(), x)[0].shape == (0, 3)


def test_the_gradients_have_no_gradient():
    x = torch.randn(4, 6, device=DEV, requires_grad=True)
    _, w = be.route_rows(x, 2)
    grad, = torch.autograd.grad(w[:, 0].sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


def test_on_another_stream_and_in_a_graph():
    n, k, E, D = 3000, 4, 16, 64
    gen = torch.Generator(device=DEV).manual_seed(2)
    logits, x = torch.randn(n, E, device=DEV, generator=gen), torch.randn(n, D, device=DEV, generator=gen)

    def layer():
        expert, weight = be.route_rows(logits, k)
        order = be.expert_order(expert, E)
        return be.rows_from_experts(be.rows_to_experts(x, order), order, weight)

    eager = layer()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(layer(), eager)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer()
    for seed in range(4):
        logits.copy_(torch.randn(n, E, device=DEV, generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, layer())


def test_places_that_are_not_there_count_as_none():
    n, k, E, D = 20, 2, 3, 40
    gen = torch.Generator(device=DEV).manual_seed(3)
    order = be.expert_order(choices(gen, n, k, E, 0.0), E)
    none, far = order.slot.clone(), order.slot.clone()
    none[5:8] = -1
    far[5:8] = torch.tensor([n * k, 1 << 30, -7], device=DEV)
    a, b = (be.ExpertOrder(s, order.pair, order.offset, n, k, E) for s in (none, far))
    y, weight, g = (torch.randn(*s, device=DEV, generator=gen) for s in ((n * k, D), (n, k), (n, D)))
    y.requires_grad_(True), weight.requires_grad_(True)
    outs = []
    for o in (a, b):
        out = be.rows_from_experts(y, o, weight)
        g_y, g_w = torch.autograd.grad(out, (y, weight), g)
        placed = o.slot[(o.slot >= 0) & (o.slot < n * k)].long()
        outs.append((out.detach(), g_y[placed], g_w, be.rows_to_experts(g, o)[placed]))
    for u, v in zip(*outs):
        assert torch.equal(u, v)
