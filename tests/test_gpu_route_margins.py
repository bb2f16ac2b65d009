"""Routing by scores where 32 bits do not tell, and in rows that hold no numbers: against the definition in 64 bits."""
import math

import pytest
import torch

import hiscache_backend as be
from test_gpu_route_scores import check, reference

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("score", ("sigmoid", "softmax"))
@pytest.mark.parametrize("size", (64.0, 1024.0, 4096.0, 65536.0))
@pytest.mark.parametrize("E,G", ((4, 2), (32, 8), (256, 16)))
def test_groups_by_sums_of_large_numbers_of_both_signs(score, size, E, G):
    """A group's two largest are near +size and -size: their sum is near 0, and in 32 bits off by half a unit of size.  (In 64 bits a
    sum's own rounding, size 2^-53 or so, decides nothing here: the least of some 10^5 gaps is about 10^-6.)"""
    gen = torch.Generator(device=DEV).manual_seed(int(size))
    n = 400_000 // (E // 4)
    logits = torch.randn(n, E, generator=gen, device=DEV)
    bias = torch.full((E,), -4 * size, device=DEV)
    bias.view(G, -1)[:, 0], bias.view(G, -1)[:, 1] = size, -size
    check(logits, 1, score=score, bias=bias, num_group=G, top_group=1, normalize=False)
    check(logits, 2, score=score, bias=bias, num_group=G, top_group=1)
    if G > 2:
        check(logits, 3, score=score, bias=bias, num_group=G, top_group=3)


@pytest.mark.parametrize("normalize", (True, False))
@pytest.mark.parametrize("bias", (False, True))
@pytest.mark.parametrize("G,top", ((1, 1), (4, 2)))
def test_gradient_of_a_softmax_that_is_no_number(normalize, bias, G, top):
    """A row with an infinity or a NaN has no softmax: its weights are NaN, and what reaches its chosen logits is, too, whichever they are."""
    gen = torch.Generator(device=DEV).manual_seed(3)
    logits = torch.randn(40, 32, generator=gen, device=DEV)
    logits[:, 3] = -math.inf
    logits[4, 20], logits[5, 21], logits[6, [9, 30]] = math.inf, math.nan, math.inf
    bad = torch.zeros(40, dtype=torch.bool)
    bad[4:7] = True
    b = torch.randn(32, generator=gen, device=DEV) if bias else None
    leaf = logits.clone().requires_grad_(True)
    expert, weight = be.route_rows(leaf, 3, normalize=normalize, bias=b, num_group=G, top_group=top, scale=1.5)
    weight.backward(torch.randn(40, 3, generator=gen, device=DEV))
    assert torch.equal(torch.isnan(weight).any(1).cpu(), bad) and torch.equal(torch.isnan(weight).all(1).cpu(), bad)
    at_chosen = leaf.grad.gather(1, expert.clamp(min=0))
    assert torch.equal(torch.isnan(at_chosen).all(1).cpu(), bad) and torch.equal(torch.isnan(leaf.grad).any(1).cpu(), bad)
    # the other rows as without those
    clean = logits.clone()
    clean[4:7] = 0.0
    clean.requires_grad_(True)
    torch.manual_seed(0)
    g = torch.randn(40, 3, device=DEV)
    leaf.grad = None
    be.route_rows(leaf, 3, normalize=normalize, bias=b, num_group=G, top_group=top, scale=1.5)[1].backward(g)
    be.route_rows(clean, 3, normalize=normalize, bias=b, num_group=G, top_group=top, scale=1.5)[1].backward(g)
    assert torch.equal(leaf.grad[7:], clean.grad[7:]) and torch.equal(leaf.grad[:4], clean.grad[:4])


@pytest.mark.parametrize("score", ("sigmoid", "softmax"))
@pytest.mark.parametrize("G,top", ((1, 1), (4, 3)))
@pytest.mark.parametrize("n", (3, 3000))
def test_a_bias_closes_an_expert_whatever_its_logit_is(score, G, top, n):
    gen = torch.Generator(device=DEV).manual_seed(3)
    logits = torch.randn(n, 32, generator=gen, device=DEV)
    bias = 0.1 * torch.randn(32, generator=gen, device=DEV)
    closed = [0, 5, 8, 9, 10, 11, 12, 13, 14, 15]            # (of four groups one whole)
    bias[closed] = -math.inf
    for value in (math.nan, math.inf, torch.finfo(torch.float32).max, -math.inf, 1.0):
        for where in ([0], [5], [9], [5, 9], [0, 5, 20], [31]):
            l = logits.clone()
            l[1::2, where] = value
            expert, weight = be.route_rows(l, 6, score=score, bias=bias, num_group=G, top_group=top)
            assert not bool(torch.isin(expert, torch.tensor(closed, device=DEV)).any()) and bool((expert >= 0).all())
            still = [e for e in where if e not in closed]
            if score == "sigmoid" and math.isnan(value):     # an open one comes first, and makes the row's shares NaN
                assert all(expert[1::2, 0].eq(e).all() for e in still)
                assert bool(torch.isnan(weight[1::2]).all()) == bool(still)
            # rows without are as before
            assert torch.equal(expert[::2], be.route_rows(logits, 6, score=score, bias=bias, num_group=G, top_group=top)[0][::2])


@pytest.mark.parametrize("normalize", (True, False))
@pytest.mark.parametrize("n", ((1 << 17) - 1, 1 << 17))
def test_a_factor_alone_on_both_sides_of_the_size_from_which_it_is_a_call_of_its_own(n, normalize):
    gen = torch.Generator(device=DEV).manual_seed(3)
    logits = (2 * torch.randn(n, 64, generator=gen, device=DEV)).to(torch.bfloat16)
    logits[::9, 5:] = -math.inf
    logits[100], logits[101, 3], logits[102, 4] = -math.inf, math.nan, math.inf
    one, w = be.route_rows(logits, 6, normalize=normalize)
    two, v = be.route_rows(logits, 6, normalize=normalize, scale=2.5)
    leaf = logits.clone().requires_grad_(True)
    three, u = be.route_rows(leaf, 6, normalize=normalize, scale=2.5)
    assert torch.equal(one, two) and torch.equal(one, three)
    for x in (v, u.detach()):
        assert torch.equal(torch.isnan(x), torch.isnan(w))
        # (each within OFF of the definition, test_gpu_route_scores)
        assert float(torch.nan_to_num((x - 2.5 * w).abs() - 200 * 2.0 ** -23 * 2.5 * w).max()) <= 0
    check(logits[:100], 6, normalize=normalize, scale=2.5)


def test_a_factor_alone_for_more_rows_than_the_softmax_s_own_kernel_takes():
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GiB of free device memory")
    n = (1 << 29) + 3                                        # (eight lanes a row there, two here)
    logits = torch.zeros(n, 2, dtype=torch.bfloat16, device=DEV)
    logits[-1, 1] = 1.0
    expert, weight = be.route_rows(logits, 1, scale=2.0)
    assert expert[-2:, 0].tolist() == [0, 1] and bool((weight == 2.0).all())
