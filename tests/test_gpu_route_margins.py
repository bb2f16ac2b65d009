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
