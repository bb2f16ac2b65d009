"""The operators of a layer of experts on matrices of more than 2^31 elements and 2^32 bytes: whole numbers that every type
holds, so that a row from or at a wrong place shows."""
import pytest
import torch

import hiscache_backend as be

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
N, D = 2_097_411, 1024


def values(n):
    return torch.arange(n, device=DEV) % 251


def matrix(n, width):
    return values(n).to(torch.bfloat16).unsqueeze(1).expand(n, width).contiguous()


def holds(rows, value):
    """Is every row of a matrix its one value?  (a part at a time: the comparison is as long as the matrix)"""
    step = 1 << 18
    return all(bool((rows[i:i + step] == value[i:i + step].unsqueeze(1)).all()) for i in range(0, len(rows), step))


def test_rows_there_and_back():
    assert N * D > 2 ** 31
    x = matrix(N, D)
    order = be.expert_order(torch.arange(N, device=DEV) % 3, 3)
    rows = be.rows_to_experts(x, order)
    at_place = values(N)[order.pair.long()].to(torch.bfloat16)
    assert holds(rows, at_place)
    weight = torch.full((N, 1), 2.0, device=DEV)
    back = be.rows_from_experts(rows, order, weight)
    assert holds(back, values(N).to(torch.bfloat16) * 2)
    del back
    y, w = rows.requires_grad_(True), weight.requires_grad_(True)
    g = torch.zeros(N, D, device=DEV, dtype=torch.bfloat16)
    g[-9:] = 1
    gy, gw = torch.autograd.grad(be.rows_from_experts(y, order, w), (y, w), g)
    assert torch.equal(gw[-9:, 0], values(N)[-9:].float() * D) and not gw[:-9].any()
    last = torch.zeros(N, device=DEV, dtype=torch.bfloat16)
    last[order.slot[-9:].long()] = 2
    assert holds(gy, last)


def test_products():
    x = matrix(N, D)
    offset = torch.tensor([0, N // 2 + 1, N - 3], device=DEV)
    w = torch.ones(2, 8, D, device=DEV, dtype=torch.bfloat16)
    w[1] = 2
    expected = values(N).float() * D * torch.where(torch.arange(N, device=DEV) < N // 2 + 1, 1.0, 2.0)
    expected[N - 3:] = 0
    assert holds(be.expert_linear(x, w, offset), expected.to(torch.bfloat16))
    g = torch.zeros(N, 8, device=DEV, dtype=torch.bfloat16)
    g[N // 2 + 1 - 5:N // 2 + 1] = 1
    g[N - 8:] = 1                                   # five of them belong to an expert
    gw = be.expert_linear_grad(g, x, offset)
    for e, rows in ((0, slice(N // 2 + 1 - 5, N // 2 + 1)), (1, slice(N - 8, N - 3))):
        assert bool((gw[e] == values(N)[rows].sum().to(torch.bfloat16)).all())
    # and as the gradient of the rows: a result of that size
    rows = x.requires_grad_(True)
    (gx,) = torch.autograd.grad(be.expert_linear(rows, w, offset), rows, g)
    expected = g[:, 0].float() * 8
    expected[N // 2 + 1:] *= 2
    expected[N - 3:] = 0
    assert holds(gx, expected.to(torch.bfloat16))


def test_kept_in_8_bits():
    x = matrix(N, D)
    kept = be.pack_rows(x)
    assert holds(be.unpack_rows(kept), values(N).to(torch.bfloat16))
    h, kept = be.gated_pack(x)
    few = slice(N - 300, N)
    h2, kept2 = be.gated_pack(x[few].contiguous())
    assert torch.equal(h[few], h2) and torch.equal(kept.codes[few], kept2.codes) and torch.equal(kept.scale[few], kept2.scale)
    g = torch.ones(N, D // 2, device=DEV, dtype=torch.bfloat16)
    gx, again = be.gated_grad(kept, g)
    gx2, again2 = be.gated_grad(kept2, g[few].contiguous())
    assert torch.equal(gx[few], gx2) and torch.equal(again[few], again2)
