"""Activations kept in 8 bits, and the gate that computes its backward pass from them, against the definition: codes and scales
are those of fp32 arithmetic rounded operation by operation, bit for bit; what is computed from them is held to 64 bits."""
import math

import pytest
import torch

import hiscache_backend as be

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
TYPES = (torch.float32, torch.float16, torch.bfloat16)
HALF = {torch.float32: (0.0, 2.0 ** -149), **{t: (torch.finfo(t).eps / 2, torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2) for t in TYPES[1:]}}
SHAPES = ((1, 1), (1, 7), (3, 8), (5, 31), (4, 33), (9, 63), (8, 64), (7, 65), (130, 100), (33, 127), (20, 128), (6, 129), (50, 602),
          (11, 1000), (257, 256))


def close(got, want, bound):
    rel, least = HALF[got.dtype]
    off = (got.double() - want).abs()
    assert bool((off <= bound + rel * (want.abs() + bound) + least).all()), float((off - bound - rel * want.abs()).max())


def parts(F, group):
    return [slice(lo, min(lo + group, F)) for lo in range(0, F, group)]


def kept32(x, group):
    """Codes and scales of x (on the CPU, fp32)."""
    x = x.float().cpu()
    codes, scales = torch.zeros(x.shape, dtype=torch.int8), []
    for p in parts(x.shape[1], group):
        m = x[:, p].abs().amax(1, keepdim=True)
        zero = m < 2.0 ** -120
        inverse = torch.where(zero, 0.0, torch.tensor(1.0) / m * torch.tensor(127.0))
        codes[:, p] = torch.round(x[:, p] * inverse).to(torch.int8)
        scales.append(torch.where(zero, 0.0, m * (torch.tensor(1.0) / torch.tensor(127.0))))
    return codes, torch.cat(scales, 1)


def rows(gen, n, F, dtype):
    x = torch.randn(n, F, device=DEV, generator=gen) * torch.exp(2 * torch.randn(n, 1, device=DEV, generator=gen))
    x[torch.rand(n, F, device=DEV, generator=gen) < 0.02] *= 30
    return x.clamp_(-6e4, 6e4).to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,F", SHAPES)
@pytest.mark.parametrize("group", (32, 64, 128))
def test_codes_scales_and_what_reads_back(dtype, n, F, group):
    x = rows(torch.Generator(device=DEV).manual_seed(n + F), n, F, dtype)
    kept = be.pack_rows(x, group)
    codes, scale = kept32(x, group)
    assert torch.equal(kept.codes.cpu(), codes) and torch.equal(kept.scale.cpu(), scale)
    back = be.unpack_rows(kept, torch.float32)
    each = kept.scale.repeat_interleave(group, 1)[:, :F]
    assert torch.equal(back, codes.to(DEV).float() * each)
    # rounding to the nearest code, six operations on values of up to 127 scales
    assert bool(((back.double() - x.double()).abs() <= each.double() * (0.5 + 127 * 6 * U)).all())
    assert be.unpack_rows(kept).dtype == dtype and torch.equal(be.unpack_rows(kept), back.to(dtype))


def test_groups_that_are_zero_tiny_or_not_finite():
    x = torch.zeros(8, 192, device=DEV)
    x[1, 3] = 2.0 ** -121
    x[2, 3] = 2.0 ** -120
    x[3, 70] = math.inf
    x[4, 70] = -math.nan
    x[5] = torch.finfo(torch.float32).max
    x[6, 100] = -torch.finfo(torch.float32).max
    x[7] = -0.0
    back = be.unpack_rows(be.pack_rows(x, 64))
    assert not back[0].any() and not back[1].any() and not back[7].any()
    assert back[2, 3] == 2.0 ** -120 / 127 * 127 or abs(float(back[2, 3]) / 2.0 ** -120 - 1) < 4 * U
    for r in (3, 4):
        assert bool(torch.isnan(back[r, 64:128]).all()) and not back[r, :64].any() and not back[r, 128:].any()
    assert bool(torch.isfinite(back[5:7]).all()) and abs(float(back[5, 0] / x[5, 0]) - 1) < 4 * U


def gate64(a, b, g):
    s = torch.sigmoid(a)
    return a * s * b, g * b * (s * (1 + a * (1 - s))), g * a * s


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,F", SHAPES)
@pytest.mark.parametrize("group", (32, 64, 128))
def test_gate_and_its_gradient(dtype, n, F, group):
    gen = torch.Generator(device=DEV).manual_seed(n * 3 + F)
    x, g = rows(gen, n, 2 * F, dtype).clamp_(-100, 100), torch.randn(n, F, device=DEV, generator=gen).to(dtype)
    h, kept = be.gated_pack(x, group)
    a, b = x[:, :F].double(), x[:, F:].double()
    want = gate64(a, b, g.double())[0]
    # an exponential off by a unit (its argument is exact), a sum, a quotient and a product
    close(h, want, 8 * U * want.abs() + 2.0 ** -126 * b.abs())
    (ca, sa), (cb, sb) = kept32(x[:, :F], group), kept32(x[:, F:], group)
    assert torch.equal(kept.codes.cpu(), torch.cat([ca, cb], 1)) and torch.equal(kept.scale.cpu(), torch.cat([sa, sb], 1))
    gx, again = be.gated_grad(kept, g)
    a, b = ((c.float() * s.repeat_interleave(group, 1)[:, :F]).to(DEV).double() for c, s in ((ca, sa), (cb, sb)))
    want, ga, gb = gate64(a, b, g.double())
    least = 2.0 ** -126 * (1 + b.abs()) * (1 + g.double().abs())
    close(again, want, 8 * U * want.abs() + least)
    s = torch.sigmoid(a)
    # 1 - s and the sum behind it lose at most a few units of what is added
    close(gx[:, :F], ga, 24 * U * (g.double() * b).abs() * s * (1 + a.abs()) + least)
    close(gx[:, F:], gb, 8 * U * gb.abs() + least)
    only, none = be.gated_pack(x, group, keep=False)
    assert none is None and torch.equal(only, h)


def test_gate_gradient_against_differences():
    """The gradient is that of the gate at the values that were kept: at whole multiples of the scale nothing is lost."""
    gen = torch.Generator(device=DEV).manual_seed(9)
    x = torch.randint(-127, 128, (64, 128), device=DEV, generator=gen).float() / 32
    x[:, ::64] = 127 / 32                                        # the largest magnitude of every group: scale 1 / 32
    d, g = torch.randn(64, 128, device=DEV, generator=gen), torch.randn(64, 64, device=DEV, generator=gen)
    h, kept = be.gated_pack(x, 64)
    gx, again = be.gated_grad(kept, g)
    assert torch.equal(be.unpack_rows(be.pack_rows(x, 64)), x)
    step = 2.0 ** -8
    up, down = (be.gated_pack(x + s * d, 64, keep=False)[0].double() for s in (step, -step))
    slope = ((up - down) * g).sum(1) / (2 * step)
    # values of up to 16 rounded by 8 half units each; third derivatives of silu(a) b along d: below |d|^3 (|b| + 3)
    size = g.abs().double().sum(1)
    bound = size * (16 * 16 * U / (2 * step) + (d.abs().amax(1).double()) ** 3 * 7 * step ** 2)
    assert bool(((slope - (gx.double() * d).sum(1)).abs() <= bound).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_off_any_alignment(dtype):
    x = rows(torch.Generator(device=DEV).manual_seed(2), 21, 2 * 64, dtype)
    shifted = torch.empty(x.numel() + 1, dtype=dtype, device=DEV)[1:].view(x.shape).copy_(x)
    for a, b in zip((be.pack_rows(x), be.gated_pack(x)[1]), (be.pack_rows(shifted), be.gated_pack(shifted)[1])):
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scale, b.scale)
    assert torch.equal(be.gated_pack(x)[0], be.gated_pack(shifted)[0])


def test_no_rows_and_refusals():
    x, g = torch.randn(6, 64, device=DEV), torch.randn(6, 32, device=DEV)
    assert be.unpack_rows(be.pack_rows(x[:0])).shape == (0, 64)
    h, kept = be.gated_pack(x[:0])
    assert h.shape == (0, 32) and be.gated_grad(kept, g[:0])[0].shape == (0, 64)
    h, kept = be.gated_pack(x)
    plain = be.pack_rows(x)
    for call in (lambda: be.pack_rows(x, 48), lambda: be.pack_rows(x.double()), lambda: be.pack_rows(x.t()), lambda: be.pack_rows(x[0]),
                 lambda: be.pack_rows(x[:, :0]), lambda: be.gated_pack(x[:, :63].contiguous()), lambda: be.unpack_rows(plain, torch.float64),
                 lambda: be.unpack_rows(kept), lambda: be.gated_grad(plain, g), lambda: be.gated_grad(kept, g[:5]),
                 lambda: be.gated_grad(kept, g.half())):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError):
        be.pack_rows(x.cpu())
