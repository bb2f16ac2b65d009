"""hc_expert_linear and its gradients against products in float64: groups that are empty, end inside a tile or leave rows
over, every type, widths and addresses off the wide loads.

A sum of K products in fp32 is off by at most K units of 2^-23 of the sum of the magnitudes, whatever the order (the matrix
instructions may cut off where they add, hence a whole unit); a narrow result by half a unit of its type besides."""
import math

import pytest
import torch

import hiscache_backend as be

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
UNIT = 2.0 ** -23
TYPES = (torch.float32, torch.float16, torch.bfloat16)
HALF = {torch.float32: (0.0, 2.0 ** -150), **{t: (torch.finfo(t).eps / 2, torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2) for t in TYPES[1:]}}


def close(got, want, bound):
    rel, least = HALF[got.dtype]
    off = (got.double() - want).abs()
    assert bool((off <= bound + rel * (want.abs() + bound) + least).all()), float((off - bound - rel * want.abs()).max())


def offsets(sizes):
    return torch.tensor([0] + list(sizes), device=DEV).cumsum(0)


def check(sizes, S, N, K, dtype, seed=0, scale=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed + S + N * 3 + K)
    E, offset = len(sizes), offsets(sizes)
    x, w, g = (scale * torch.randn(s, device=DEV, generator=gen).to(dtype) for s in ((S, K), (E, N, K), (S, N)))
    x.requires_grad_(True)
    w.requires_grad_(True)
    y = be.expert_linear(x, w, offset)
    gx, gw = torch.autograd.grad(y, (x, w), g)
    assert y.shape == (S, N) and y.dtype == gx.dtype == gw.dtype == dtype
    x64, w64, g64, ends = x.detach().double(), w.detach().double(), g.double(), offset.tolist()
    for e in range(E):
        r = slice(ends[e], ends[e + 1])
        close(y[r].detach(), x64[r] @ w64[e].t(), (K + 1) * UNIT * (x64[r].abs() @ w64[e].abs().t()))
        close(gx[r], g64[r] @ w64[e], (N + 1) * UNIT * (g64[r].abs() @ w64[e].abs()))
        close(gw[e], g64[r].t() @ x64[r], (sizes[e] + 1) * UNIT * (g64[r].abs().t() @ x64[r].abs()))
    assert not y[ends[-1]:].any() and not gx[ends[-1]:].any()
    assert torch.equal(be.expert_linear_grad(g, x.detach(), offset), gw)
    return y, gx, gw


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,K", ((1, 1), (5, 3), (47, 64), (64, 47), (64, 64), (63, 65), (100, 172), (128, 256), (256, 128), (300, 96),
                                 (256, 256), (130, 520)))
def test_products_and_gradients(dtype, N, K):
    check((70, 0, 1, 129, 64, 0, 300), 600, N, K, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes,S", (((1,), 1), ((0,), 3), ((0, 0, 0), 0), ((1, 1, 1, 1), 4), ((0, 0, 5), 5), ((255, 256, 257), 768),
                                     ((511, 513), 1100), ((3,) * 70, 300), ((1,) * 1024, 1024), ((2000, 3, 1), 2004)))
def test_groups_of_any_size(dtype, sizes, S):
    check(sizes, S, 96, 80, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes,S,N,K", (((1500, 20, 0, 900, 4000), 6421, 512, 256), ((5000, 100), 5100, 320, 1024), ((17, 30_000), 30_020, 256, 256),
                                         ((9, 12, 3), 24, 2048, 1024), ((2100, 1900), 4000, 1000, 600)))
def test_larger_products(dtype, sizes, S, N, K):
    check(sizes, S, N, K, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes,S,N,K", (((9000, 20, 0, 3000, 4000), 16_030, 640, 70), ((9000, 20, 0, 3000, 4000), 16_030, 330, 602),
                                         ((7000, 33, 7900), 15_000, 1000, 72), ((7000, 33, 7900), 15_000, 90, 998),
                                         ((30_000, 1, 14_000), 44_010, 1000, 2006), ((300,) * 100 + (0, 7), 30_100, 640, 602),
                                         ((8000, 15_000, 9000), 32_020, 1024, 520), ((20_000, 14_000), 34_001, 512, 72)))
def test_products_of_every_tile(dtype, sizes, S, N, K):
    """Enough tiles for the wider ones, with widths that end inside a tile and inside a step."""
    check(sizes, S, N, K, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,K", ((64, 64), (256, 128), (100, 72)))
def test_operands_off_the_alignment_of_wide_loads(dtype, N, K):
    gen = torch.Generator(device=DEV).manual_seed(N)
    offset = offsets((100, 0, 60))
    x, w, g = (torch.randn(s, device=DEV, generator=gen).to(dtype) for s in ((170, K), (3, N, K), (170, N)))

    def shifted(t):
        return torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)[1:].view(t.shape).copy_(t)

    def all_of(x, w, g):
        x, w = x.requires_grad_(True), w.requires_grad_(True)
        y = be.expert_linear(x, w, offset)
        return (y.detach(), *torch.autograd.grad(y, (x, w), g))

    for a, b, n in zip(all_of(x, w, g), all_of(shifted(x), shifted(w), shifted(g)), (K, N, 100)):
        close(b, a.double(), 2 * n * UNIT * 8 * n ** 0.5 + 2 * HALF[dtype][0] * a.double().abs())


@pytest.mark.parametrize("dtype", TYPES)
def test_what_one_group_holds_does_not_reach_another(dtype):
    x, w = torch.ones(300, 64, device=DEV, dtype=dtype), torch.ones(3, 64, 64, device=DEV, dtype=dtype)
    g = torch.ones(300, 64, device=DEV, dtype=dtype)
    offset = offsets((100, 50, 130))
    x[100:150] = float("nan")
    g[280:] = float("inf")
    x[280:] = float("nan")
    w[1] = float("inf")
    a, b = x.requires_grad_(True), w.requires_grad_(True)
    y = be.expert_linear(a, b, offset)
    gx, gw = torch.autograd.grad(y, (a, b), g)
    rest = torch.cat([y[:100], y[150:280]])
    assert bool((rest == 64).all()) and not y[280:].any()
    assert bool((torch.cat([gx[:100], gx[150:280]]) == 64).all()) and not gx[280:].any()
    assert bool((gw[0] == 100).all()) and bool((gw[2] == 130).all()) and bool(torch.isnan(gw[1]).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,K,first", ((47, 47, 101), (33, 64, 101), (64, 33, 100), (1, 1, 7), (129, 65, 33)))
def test_what_one_group_holds_does_not_reach_another_at_odd_widths(dtype, N, K, first):
    """Where rows of 16-bit elements share a word with their neighbours, in tensors whose neighbours in memory are not finite."""
    def inside(*shape):
        whole = torch.full((math.prod(shape) + 66,), float("nan"), device=DEV, dtype=dtype)
        return whole[33:-33].view(shape).fill_(1)

    x, w, g = inside(300, K), inside(3, N, K), inside(300, N)
    offset, second = offsets((first, 50, 150 - first % 2)), first + 50
    end = int(offset[-1])
    x[first:second] = w[1] = float("nan")
    g[first:second] = x[end:] = float("inf")
    g[end:] = float("nan")
    a, b = x.requires_grad_(True), w.requires_grad_(True)
    y = be.expert_linear(a, b, offset)
    gx, gw = torch.autograd.grad(y, (a, b), g)
    for rows, n in ((y, K), (gx, N)):
        assert bool((torch.cat([rows[:first], rows[second:end]]) == n).all()) and not rows[end:].any()
    assert bool((gw[0] == first).all()) and bool((gw[2] == end - second).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_whole_numbers_are_summed_exactly(dtype):
    """Small whole numbers: every partial sum is exact in fp32, so a row or column left out, taken twice or rounded shows."""
    gen = torch.Generator(device=DEV).manual_seed(7)
    sizes = (700, 1, 0, 320)
    offset, S, N, K = offsets(sizes), 1030, 136, 200
    x, w, g = (torch.randint(-3, 4, s, device=DEV, generator=gen).to(dtype) for s in ((S, K), (4, N, K), (S, N)))
    x[:, 5:] *= torch.rand(S, K - 5, device=DEV, generator=gen) < 0.1              # small enough for 8 bits of mantissa
    w[:, :, 40:] *= torch.rand(4, N, K - 40, device=DEV, generator=gen) < 0.1
    g *= torch.rand(S, N, device=DEV, generator=gen) < 0.1
    a, b = x.requires_grad_(True), w.requires_grad_(True)
    y = be.expert_linear(a, b, offset)
    gx, gw = torch.autograd.grad(y, (a, b), g)
    x, w, ends = x.detach().double(), w.detach().double(), offset.tolist()
    for e in range(4):
        r = slice(ends[e], ends[e + 1])
        for got, want in ((y[r], x[r] @ w[e].t()), (gx[r], g[r].double() @ w[e]), (gw[e], g[r].double().t() @ x[r])):
            assert torch.equal(got.detach(), want.to(dtype))


def test_gradients_against_differences():
    gen = torch.Generator(device=DEV).manual_seed(11)
    offset = offsets((90, 0, 37, 200))
    x, dx = torch.randn(340, 72, device=DEV, generator=gen), torch.randn(340, 72, device=DEV, generator=gen)
    w, dw = torch.randn(4, 56, 72, device=DEV, generator=gen), torch.randn(4, 56, 72, device=DEV, generator=gen)
    g = torch.randn(340, 56, device=DEV, generator=gen)
    a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    gx, gw = torch.autograd.grad(be.expert_linear(a, b, offset), (a, b), g)
    # linear in each: a step of one loses nothing but rounding
    for grad, d, up, down in ((gx, dx, be.expert_linear(x + dx, w, offset), be.expert_linear(x - dx, w, offset)),
                              (gw, dw, be.expert_linear(x, w + dw, offset), be.expert_linear(x, w - dw, offset))):
        slope = ((up.double() - down.double()) * g).sum() / 2
        # sums of at most 200 products
        size = 8 * 200 ** 0.5 * g.abs().double().sum() + (grad.abs() * d.abs()).double().sum()
        assert abs(float(slope - (grad.double() * d).sum())) <= 200 * UNIT * float(size)


def test_offsets_out_of_order_or_range_touch_no_other_memory():
    x, w = torch.randn(50, 64, device=DEV), torch.randn(3, 64, 64, device=DEV)
    for off in ((0, 100, 20, 50), (-5, 10, 20, 1 << 40), (30, 20, 10, 0)):
        offset = torch.tensor(off, device=DEV)
        assert be.expert_linear(x, w, offset).shape == (50, 64)
        assert be.expert_linear_grad(x, x, offset).shape == (3, 64, 64)
    torch.cuda.synchronize()


@pytest.mark.parametrize("E", (3, 64, 65, 130))
def test_offsets_that_overlap_count_as_their_largest_so_far(E):
    """Also: the partial sums of a gradient stay in their workspace, however many parts such offsets would make."""
    S, N, K = 3000, 40, 64
    gen = torch.Generator(device=DEV).manual_seed(E)
    x, g = torch.randn(S, K, device=DEV, generator=gen), torch.randn(S, N, device=DEV, generator=gen)
    w = torch.randn(E, N, K, device=DEV, generator=gen)
    lib, size = be.load_library(), N * K
    there_and_back = torch.arange(E + 1, device=DEV) % 2 * S
    for offset in (there_and_back, torch.randint(-900, S + 900, (E + 1,), device=DEV, generator=gen)):
        ordered = offset.clamp(0, S).cummax(0).values
        assert torch.equal(be.expert_linear(x, w, offset), be.expert_linear(x, w, ordered))
        nbytes = lib.hc_expert_linear_grad_workspace_bytes(S, E, N, K, 0)
        assert nbytes > 0 and nbytes % 4 == 0
        room = torch.full((nbytes // 4 + 70 * size,), 7.0, device=DEV)
        gw = torch.empty(E, N, K, device=DEV)
        assert lib.hc_expert_linear_grad(g.data_ptr(), x.data_ptr(), 0, offset.data_ptr(), S, E, N, K, gw.data_ptr(), room.data_ptr(),
                                         nbytes, 0) == 0
        torch.cuda.synchronize()
        assert bool((room[nbytes // 4:] == 7).all())
        assert torch.equal(gw, be.expert_linear_grad(g, x, ordered))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("E", (2, 63, 64))
def test_some_of_the_experts(E, dtype):
    """A later part of a batch's offsets with its matrices: the rows of the other experts are zeros, and add nothing."""
    gen = torch.Generator(device=DEV).manual_seed(E)
    x, g = (torch.randn(700, d, device=DEV, generator=gen).to(dtype) for d in (72, 96))
    w = torch.randn(E + 2, 96, 72, device=DEV, generator=gen).to(dtype)
    offset = torch.randint(0, 700, (E + 3,), device=DEV, generator=gen).sort().values
    offset[0] = 0
    a, b = x.requires_grad_(True), w.requires_grad_(True)
    y = be.expert_linear(a, b, offset)
    gx, gw = torch.autograd.grad(y, (a, b), g)
    some = b.detach()[1:-1].contiguous().requires_grad_(True)
    part = be.expert_linear(a, some, offset[1:-1].contiguous())
    hx, hw = torch.autograd.grad(part, (a, some), g)
    mine = torch.zeros(700, 1, dtype=torch.bool, device=DEV)
    mine[int(offset[1]):int(offset[-2])] = True
    assert torch.equal(part, torch.where(mine, y, 0)) and torch.equal(hx, torch.where(mine, gx, 0)) and torch.equal(hw, gw[1:-1])


def test_refusals():
    x, w, off = torch.randn(10, 8, device=DEV), torch.randn(2, 4, 8, device=DEV), offsets((4, 6))
    for call in (lambda: be.expert_linear(x, w.half(), off), lambda: be.expert_linear(x.double(), w.double(), off),
                 lambda: be.expert_linear(x, w[:, :, :4].contiguous(), off), lambda: be.expert_linear(x, w, off[:2]),
                 lambda: be.expert_linear(x, w, off.int()), lambda: be.expert_linear(x, w.transpose(1, 2), off),
                 lambda: be.expert_linear(x[:, ::2], w, off), lambda: be.expert_linear(x[0], w, off),
                 lambda: be.expert_linear(x, w[0], off), lambda: be.expert_linear_grad(x[:5], x, off),
                 lambda: be.expert_linear_grad(x.half(), x, off),
                 lambda: be.expert_linear(x, torch.zeros(1025, 1, 8, device=DEV), torch.zeros(1026, dtype=torch.int64, device=DEV))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError):
        be.expert_linear(x.cpu(), w, off)


@pytest.mark.parametrize("dtype", TYPES)
def test_the_same_bits_every_time_and_in_a_graph(dtype):
    gen = torch.Generator(device=DEV).manual_seed(4)
    offset = offsets((700, 3000, 0, 120))
    x, w, g = (torch.randn(s, device=DEV, generator=gen).to(dtype) for s in ((3900, 128), (4, 192, 128), (3900, 192)))

    def step():
        a, b = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        y = be.expert_linear(a, b, offset)
        return (y.detach(), *torch.autograd.grad(y, (a, b), g))

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert all(torch.equal(p, q) for p, q in zip(step(), first))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        x.copy_(torch.randn(3900, 128, device=DEV, generator=gen))
        offset.copy_(offsets((1000, 2000, 500, 300)))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, step()))
