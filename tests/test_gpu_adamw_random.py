"""Moments in 8 bits, rounded at random: the kernel's codes against the definition, and long runs of the optimizer against one
in 32 bits (the bounds are derived in ``test_adamw_random_cpu``)."""
import copy
import math

import pytest
import torch

import hiscache
import hiscache_backend as be
from adamw_codes import hold, words

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HOW = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
SIZES = [(1,), (7,), (127,), (128,), (129,), (3, 43), (2047,), (2048,), (2049,), (64, 100), (5, 4099), (), (0,)]


@pytest.mark.parametrize("dtype", (torch.float32, torch.float16, torch.bfloat16))
@pytest.mark.parametrize("master", (False, True))
@pytest.mark.parametrize("start", (0, (5 << 32) + 17))
def test_codes_are_the_definition_s(dtype, master, start):
    if master and dtype == torch.float32:
        return
    gen = torch.Generator(device=DEV).manual_seed(1)
    ps = [torch.randn(s, generator=gen, device=DEV).to(dtype) for s in SIZES]
    states = [be.adamw_state(p, 8, master) for p in ps]
    twin = [p.clone() for p in ps]
    nearest = [be.adamw_state(p, 8, master) for p in ps]
    for s in states + nearest:
        s.step[0] = start
    b1, b2 = (torch.tensor(b, device=DEV) for b in HOW["betas"])
    c1, c2 = (torch.tensor(1 - b, device=DEV) for b in HOW["betas"])
    for t in range(start + 1, start + 5):
        gs = [(torch.randn(s, generator=gen, device=DEV) * torch.exp(2 * torch.randn(s, generator=gen, device=DEV))
               * (torch.rand(s, generator=gen, device=DEV) < 0.9)).to(dtype) for s in SIZES]
        held = be.adamw_moments(states)
        # (the step itself is the same whichever way its moments are kept)
        for p, q, s, z in zip(ps, twin, states, nearest):
            q.copy_(p)
            for part in ("exp_avg", "exp_avg_sq", "scale", "master"):
                if getattr(s, part) is not None:
                    getattr(z, part).copy_(getattr(s, part))
        be.adamw_step(ps, gs, states, rounding="random", **HOW)
        be.adamw_step(twin, gs, nearest, **HOW)
        for p, q, g, s, z, (m, r) in zip(ps, twin, gs, states, nearest, held):
            assert torch.equal(p, q) and s.step.tolist() == z.step.tolist() == [t, 0]
            m, r, g = m.view(-1), r.view(-1), g.float().view(-1)
            m = b1 * m + c1 * g
            r = torch.sqrt((b2 * (r * r) + c2 * g * g).double()).float()
            w = words(torch.arange(m.numel(), device=DEV), t)
            for x, bits, got, row in ((m, 3, s.exp_avg, 0), (r, 4, s.exp_avg_sq, 1)):
                code, E, value = hold(x, bits, w)
                assert torch.equal(got.view(-1), code) and torch.equal(s.scale[row], E)
                code, E, value = hold(x, bits, None)
                assert torch.equal((z.exp_avg, z.exp_avg_sq)[row].view(-1), code) and torch.equal(z.scale[row], E)


def test_groups_with_infinities_and_nan_and_numbers_near_fp32_s_ends():
    g = torch.full((640,), 0.5, device=DEV)
    g[130], g[300] = math.inf, math.nan
    g[384:512] = 0.0
    g[512:] = torch.linspace(1, 2, 128, device=DEV) * 2.0 ** -126
    state = be.adamw_state(g, 8)
    be.adamw_step([torch.ones(640, device=DEV)], [g], [state], betas=(0.0, 0.0), rounding="random")
    (m, r), = be.adamw_moments([state])
    nan = torch.zeros(640, dtype=torch.bool, device=DEV)
    nan[128:384] = True
    assert torch.equal(torch.isnan(m), nan) and torch.equal(torch.isnan(r), nan)
    assert bool((m[:128] == 0.5).all()) and bool((r[:128] == 0.5).all()) and not bool(m[384:512].any()) and not bool(r[384:512].any())
    assert bool(((m[512:] / g[512:] - 1).abs() < 1 / 8).all())


def test_recorded_and_repeated_steps_are_the_same():
    """What is random goes by element and count alone: an eager step, a replayed one and one beside other tensors keep the same codes."""
    gen = torch.Generator(device=DEV).manual_seed(2)
    p0, g = torch.randn(70_001, generator=gen, device=DEV), torch.randn(70_001, generator=gen, device=DEV)
    other = [torch.randn(300, generator=gen, device=DEV) for _ in range(3)]
    runs = [(p0.clone(), be.adamw_state(p0, 8)) for _ in range(3)]
    beside = [be.adamw_state(o, 8) for o in other]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        be.adamw_step([runs[1][0]], [g], [runs[1][1]], rounding="random")
    for _ in range(4):
        be.adamw_step([runs[0][0]], [g], [runs[0][1]], rounding="random")
        graph.replay()
        be.adamw_step([*other, runs[2][0]], [*other, g], [*beside, runs[2][1]], rounding="random")
        torch.cuda.synchronize()
        for p, s in runs[1:]:
            a = runs[0][1]
            assert torch.equal(p, runs[0][0]) and torch.equal(s.exp_avg, a.exp_avg) and torch.equal(s.exp_avg_sq, a.exp_avg_sq)
            assert torch.equal(s.scale, a.scale) and torch.equal(s.step, a.step)
    with pytest.raises(ValueError, match="rounding"):
        be.adamw_step([p0], [g], [be.adamw_state(p0, 8)], rounding="up")


@pytest.mark.parametrize("kind", ("constant", "normal", "shrinking", "growing"))
@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
def test_a_long_run_goes_where_one_in_32_bits_goes(kind, dtype):
    """3 000 steps at the default betas, 6 000 where gradients fall to a hundredth."""
    n, count = 128 * 128, 6000 if kind == "shrinking" else 3000
    gen = torch.Generator(device=DEV).manual_seed(3)
    size = torch.exp(torch.randn(n, generator=gen, device=DEV))
    ps = [torch.nn.Parameter(torch.zeros(n, device=DEV, dtype=dtype)) for _ in range(2)]
    opts = [hiscache.AdamW([p], lr=1e-3, weight_decay=0.0, state_bits=bits) for p, bits in zip(ps, (8, 32))]
    for p in ps:
        p.grad = torch.zeros_like(p)
    for t in range(1, count + 1):
        g = size if kind == "constant" else size * torch.randn(n, generator=gen, device=DEV)
        if t >= 1000 and kind in ("shrinking", "growing"):
            g = g * (0.01 if kind == "shrinking" else 100.0)
        for p, o in zip(ps, opts):
            p.grad.copy_(g)
            o.step()
    (m8, v8), (m, v) = (o.moments(p) for p, o in zip(ps, opts))
    assert opts[0].state[ps[0]]["exp_avg_sq"].dtype == torch.uint8
    m8, m, ratio = m8.double(), m.double(), (v8 / v).double().sqrt()
    spread = math.hypot(0.125, math.sqrt(5000 * 0.001 / 32) if kind == "shrinking" else 0.0)
    assert abs(float(ratio.mean()) - 1) <= 0.016 + 4 * spread / math.sqrt(n)
    assert float((ratio - 1).square().mean().sqrt()) <= 1.2 * spread
    assert abs(float((m8 * m).sum() / (m * m).sum()) - 1) <= 0.03
    far8, far = (o.state[p].get("master", p).detach().double() for p, o in zip(ps, opts))
    assert abs(float((far8 * far).sum() / (far * far).sum()) - 1) <= 0.03
    # an element's own way: the moment's roundings (0.09 of it) and the root's (0.125), more while it falls
    assert float((far8 - far).norm() / far.norm()) <= 0.25


def test_places_beyond_32_bits():
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GiB of free device memory")
    n, tail = (1 << 32) + 777, 4 * 128 + 777
    p, g = torch.zeros(n, device=DEV, dtype=torch.bfloat16), torch.zeros(n, device=DEV, dtype=torch.bfloat16)
    gen = torch.Generator(device=DEV).manual_seed(8)
    g[-tail:] = torch.randn(tail, generator=gen, device=DEV).to(torch.bfloat16)
    s = be.adamw_state(p, 8)
    be.adamw_step([p], [g], [s], betas=(0.0, 0.0), rounding="random")
    w = words(torch.arange(n - tail, n, device=DEV), 1)
    for x, bits, got, row in ((g[-tail:].float(), 3, s.exp_avg, 0), (g[-tail:].float().abs(), 4, s.exp_avg_sq, 1)):
        code, E, _ = hold(x, bits, w)
        assert torch.equal(got[-tail:], code) and torch.equal(s.scale[row, -E.numel():], E)


def test_a_part_of_a_state_goes_with_one_parameter():
    """Two states with one moment, one scale, one copy or two views of one count: refused before anything is written."""
    ps = [torch.zeros(300, device=DEV, dtype=torch.bfloat16) for _ in range(2)]
    gs = [torch.ones_like(p) for p in ps]
    for part in ("exp_avg", "exp_avg_sq", "step", "scale", "master"):
        a, b = (be.adamw_state(p, 8, True) for p in ps)
        shared = getattr(a, part)
        setattr(b, part, shared.view(shared.shape))
        with pytest.raises(ValueError, match="one parameter"):
            be.adamw_step(ps, gs, [a, b])
        assert not bool(a.step.any()) and not bool(b.step.any()) and not bool(a.exp_avg.any())
    q = torch.zeros(300, device=DEV)
    s = be.adamw_state(q)
    with pytest.raises(ValueError, match="part of a state"):
        be.adamw_step([q], [q + 1], [be.AdamWState(s.exp_avg, q.view(300), s.step)])
    none = [torch.zeros(0, device=DEV) for _ in range(2)]
    be.adamw_step(none, none, [be.adamw_state(p) for p in none])


@pytest.mark.parametrize("most", (1.0, 2.0 ** 40, 2.0 ** -30))
def test_small_codes_are_rounded_once(most):
    """Numbers beside the middle between two of the smallest codes, nearer to it than fp32's smallest steps are where the largest of the group has
    been scaled to the codes' own exponent: the side that they lie on counts, a tie is even."""
    for bits in (3, 4):
        unit = most * 2.0 ** (-14 - bits)
        k = torch.arange(8, device=DEV).double() + 0.5
        x = torch.cat([k * (1 + s * 2.0 ** -e) for e in (21, 22, 23) for s in (-1, 0, 1)] + [k * 0 + 0.25, k * 0, -k]).float() * unit
        g = torch.zeros(128, device=DEV)
        g[0], g[1:1 + x.numel()] = most, x
        state = be.adamw_state(g, 8)
        be.adamw_step([torch.zeros_like(g)], [g], [state], betas=(0.0, 0.0))
        if bits == 3:
            code = state.exp_avg[1:25].tolist()
            assert code[:8] == [0, 1, 2, 3, 4, 5, 6, 7]      # just below the middle: down
            assert code[8:16] == [0, 2, 2, 4, 4, 6, 6, 8] and code[16:] == [1, 2, 3, 4, 5, 6, 7, 8]
            assert torch.equal(state.exp_avg, hold(g, 3, None)[0])
        else:                                                # (b2 = 0: the root of the gradient's square)
            assert torch.equal(state.exp_avg_sq, hold((g * g).double().sqrt().float(), 4, None)[0])


def test_a_copied_optimizer_takes_weights_that_were_loaded_before_its_first_step():
    """The fp32 copies that came with it are of the weights as they were."""
    torch.manual_seed(0)
    model = torch.nn.Linear(64, 64).to(DEV, torch.bfloat16)
    opt = hiscache.AdamW(model.parameters(), lr=1e-3)
    for p in model.parameters():
        p.grad = torch.randn_like(p)
    opt.step()
    twin, other = copy.deepcopy((model, opt))
    kept = other.state[twin.weight]["master"].clone()
    with torch.no_grad():
        twin.weight[3] = 2.0
    for p in twin.parameters():
        p.grad = torch.zeros_like(p)
    other.param_groups[0].update(lr=0.0)
    other.step()
    master = other.state[twin.weight]["master"]
    assert bool((master[3] == 2.0).all()) and torch.equal(master[:3], kept[:3]) and torch.equal(master[4:], kept[4:])
    assert torch.equal(twin.weight, master.to(torch.bfloat16)) and torch.equal(opt.state[model.weight]["master"], kept)
