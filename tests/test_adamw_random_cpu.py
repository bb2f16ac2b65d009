"""Moments of an AdamW step in 8 bits, rounded at random: the definition by itself, over many steps.

How far off it may be, in units of the right root.  A root moves by a = (1 - b2) / 2 |g g / v - 1| of itself a step and its codes lie at most
1/16 apart, so that one rounding has a variance of a / 16 at most.  Where v stands still on the whole, what is off fades by
1 - b2 a step: a variance of c / 64, c = mean |g g / v - 1| (1 for normally distributed gradients), 0.125 of the root; the mean of the
squares is c / 32 too large at most, the root's 1.6 %.  Where v only falls, T steps add up to T (1 - b2) / 32.  The mean over n
elements is off by another spread / sqrt(n)."""
import math

import pytest
import torch

from adamw_codes import hold, words

N = 128 * 8


def steps(gradient, count, b1=0.9, b2=0.999, random=True):
    """Moments held in 8 bits and in fp64 after ``count`` steps, and how far both have moved parameters."""
    index = torch.arange(N)
    m8, r8, far8 = torch.zeros(N), torch.zeros(N), torch.zeros(N, dtype=torch.float64)
    m, v, far = (torch.zeros(N, dtype=torch.float64) for _ in range(3))
    for t in range(1, count + 1):
        g = gradient(t)
        m8, v8 = b1 * m8 + (1 - b1) * g, b2 * (r8 * r8) + (1 - b2) * g * g
        r8 = v8.sqrt()
        m, v = b1 * m + (1 - b1) * g.double(), b2 * v + (1 - b2) * g.double() ** 2
        lift = math.sqrt(1 - b2 ** t)
        far8 += m8.double() / (1 - b1 ** t) / (r8.double() / lift + 1e-8)
        far += m / (1 - b1 ** t) / (v.sqrt() / lift + 1e-8)
        word = words(index, t) if random else None
        m8, r8 = hold(m8, 3, word)[2], hold(r8, 4, word)[2]
    return m8.double(), r8.double(), far8, m, v.sqrt(), far


def normal(seed, factor=lambda t: 1.0):
    gen = torch.Generator().manual_seed(seed)
    size = torch.exp(torch.randn(N, generator=gen))
    return lambda t: factor(t) * size * torch.randn(N, generator=gen)


@pytest.mark.parametrize("kind", ("constant", "normal", "shrinking", "growing"))
def test_moments_stay_right_in_the_mean(kind):
    gradient = {"constant": lambda t: torch.linspace(-1, 1, N), "normal": normal(1),
                "shrinking": normal(2, lambda t: 1.0 if t < 300 else 0.01), "growing": normal(3, lambda t: 1.0 if t < 300 else 100.0)}[kind]
    m8, r8, far8, m, r, far = steps(gradient, 1500)
    spread = math.sqrt(1200 * 0.001 / 32) if kind == "shrinking" else 0.0
    spread = math.hypot(spread, 0.125)
    ratio = r8 / r
    assert abs(float(ratio.mean()) - 1) <= 0.016 + 4 * spread / math.sqrt(N)
    assert float((ratio - 1).square().mean().sqrt()) <= 1.2 * spread
    # the moment's codes lie an eighth apart at most, it is unbiased
    assert abs(float((m8 * m).sum() / (m * m).sum()) - 1) <= 0.05
    assert abs(float((far8 * far).sum() / (far * far).sum()) - 1) <= 0.05


def test_the_nearest_code_would_stop_the_second_moment():
    """(Why a training run is not rounded so: the root ends where (1 - b2) / 2 (g g / v - 1) is half a code, 1/64 to 1/32 of it.)"""
    r8, r = steps(lambda t: torch.ones(N), 1500, random=False)[1::3]
    assert float((r8 / r).max()) < 0.25


def test_words_are_even():
    """Every bit of a word is set half the time, over elements and over steps, and flips half the time from a neighbour or a step to the next:
    a count of n fair bits is within 5 sqrt(n) / 2 of its half (once in two million for each of 200 counts)."""
    n = 1 << 16
    bits = torch.arange(32)
    over = words(torch.arange(n), 7)
    steps_ = torch.cat([words(torch.tensor([123]), t) for t in range(1, 4097)])
    for w in (over, steps_):
        for x in (w, w[1:] ^ w[:-1], (w[1:] >> 16 ^ w[:-1]) & 0xFFFF):
            count = ((x.view(-1, 1) >> bits) & 1).sum(0).double()
            top = 16 if int(x.max()) < 1 << 16 else 32
            assert bool(((count[:top] - x.numel() / 2).abs() <= 2.5 * math.sqrt(x.numel())).all())


def test_a_code_s_own_number_stays_as_it_is():
    value = torch.cat([torch.linspace(1, 2, 9)[:8] * 2.0 ** -k for k in range(16)])
    for t in range(1, 9):
        word = words(torch.arange(value.numel()), t)
        assert torch.equal(hold(value, 3, word)[2][:112], value[:112]) and torch.equal(hold(value, 4, word)[2][:112], value[:112])


def test_the_flag_at_the_c_entry():
    """8 | 256 is 8 with another rounding and wants what 8 wants; 32 | 256 and the flag alone are refused."""
    import ctypes

    import hiscache_backend as be
    lib = be.load_library()
    word = (ctypes.c_void_p * 1)(ctypes.addressof(ctypes.c_int64(0)))
    numel = (ctypes.c_int64 * 1)(4)

    def step(bits, scale):
        return lib.hc_adamw_step(1, word, word, 0, word, word, scale, None, word, numel, bits, 1e-3, None, 0.9, 0.999, 1e-8, 0.0, None)
    assert [step(b, None) for b in (8 | 256, 256, 32 | 256, 16 | 256)] == [1, 1, 1, 1]
    assert step(32 | 256, word) == 1 and step(8 | 512, word) == 1
