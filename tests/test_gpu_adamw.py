"""The AdamW step over many tensors, and the optimizer around it: against the formula in 64 bits, states in 32 and in 8 bits."""
import copy
import math

import pytest
import torch

import hiscache
import hiscache_backend as be

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HOW = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
SIZES = [(1,), (7,), (127,), (128,), (129,), (3, 43), (2047,), (2048,), (2049,), (64, 100), (5, 4099), ()]


def draw(gen, shape, dtype, scale=1.0):
    return (scale * torch.randn(shape, generator=gen, device=DEV)).to(dtype)


def exact_step(p, g, m, v, t, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2):
    """The formula in fp64; t: the step that is made."""
    p, g, m, v = (x.double() for x in (p, g, m, v))
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    move = m / (1 - betas[0] ** t) / (torch.sqrt(v / (1 - betas[1] ** t)) + eps)
    return p * (1 - lr * weight_decay) - lr * move, m, v


def near_step(p, want, old, lr):
    """Is p what a step in fp32 from `old` to `want` may give?  Two roundings of numbers up to |p| + lr (2^-24 each), and the move, of at
    most 10 lr here, exact to eight roundings and two units of a reciprocal and a root (2^-20 of it)."""
    bound = 2.0 ** -23 * (old.abs().double() + want.abs()) + 10 * lr * 2.0 ** -20
    return bool(((p.double() - want).abs() <= bound).all())


def units(x, most, bits):
    """The step of 8 bits around x in a group whose largest magnitude is `most`: 2^-bits of its binade, at least 2^-14 of the largest's."""
    e = torch.floor(torch.log2(torch.where(x == 0, torch.full_like(x, 2.0 ** -300), x.abs())))
    top = torch.floor(torch.log2(most))
    return torch.exp2(torch.maximum(e, top - 14) - bits)


def groups_of(x):
    flat = x.reshape(-1).double()
    pad = -flat.numel() % be.ADAMW_GROUP
    most = torch.nn.functional.pad(flat.abs(), (0, pad)).view(-1, be.ADAMW_GROUP).amax(1)
    return most.repeat_interleave(be.ADAMW_GROUP)[:flat.numel()].view(x.shape)


def held_near(value, x, bits):
    """Does 8 bits' `value` hold x to half a step (and fp32's rounding of x)?  The largest may have rounded up a binade."""
    most = groups_of(x)
    step = units(x.double(), torch.clamp(most * (1 + 2.0 ** -bits), min=2.0 ** -200), bits)
    # a root (four bits) above 0 and below half the smallest code is held as that code, a step: 0 < x < step / 2 gives |step - x| < step
    up = (x.double() > 0) & (x.double() < step / 2) if bits == 4 else torch.zeros_like(x, dtype=torch.bool)
    bound = torch.where(up, step, step * (0.5 + 2.0 ** -10))
    return bool(((value.double() - x.double()).abs() <= bound + 2.0 ** -126).all())


@pytest.mark.parametrize("dtype", (torch.float32, torch.float16, torch.bfloat16))
@pytest.mark.parametrize("master", (False, True))
def test_32_bits(dtype, master):
    if master and dtype == torch.float32:
        with pytest.raises(ValueError):
            be.adamw_state(torch.zeros(4, device=DEV), 32, True)
        return
    gen = torch.Generator(device=DEV).manual_seed(1)
    ps = [draw(gen, s, dtype) for s in SIZES]
    states = [be.adamw_state(p, 32, master) for p in ps]
    for t in range(1, 6):
        gs = [draw(gen, s, dtype, 10.0 ** (-t)) for s in SIZES]
        before = [(p.clone(), s.exp_avg.clone(), s.exp_avg_sq.clone(), None if s.master is None else s.master.clone())
                  for p, s in zip(ps, states)]
        be.adamw_step(ps, gs, states, **HOW)
        for p, g, s, (p0, m0, v0, copy0) in zip(ps, gs, states, before):
            start = copy0 if master else p0
            want, m, v = exact_step(start, g, m0, v0, t, **HOW)
            # three roundings of sums of numbers of one sign or of the two terms' size
            assert bool(((s.exp_avg - m).abs() <= 2.0 ** -22 * (m0.abs() + g.float().abs())).all())
            assert bool(((s.exp_avg_sq - v).abs() <= 2.0 ** -22 * v + 2.0 ** -149).all())
            assert s.step.tolist() == [t, 0]
            if master:
                assert near_step(s.master, want, start.float(), HOW["lr"]) and torch.equal(p, s.master.to(dtype))
            elif dtype == torch.float32:
                assert near_step(p, want, start, HOW["lr"])
            else:
                bound = torch.finfo(dtype).eps / 2 * want.abs() + 10 * HOW["lr"] * 2.0 ** -18 + torch.finfo(dtype).tiny
                assert bool(((p.double() - want).abs() <= bound + 2.0 ** -20 * want.abs()).all())


@pytest.mark.parametrize("dtype", (torch.float32, torch.float16, torch.bfloat16))
@pytest.mark.parametrize("master", (False, True))
def test_8_bits(dtype, master):
    if master and dtype == torch.float32:
        return
    gen = torch.Generator(device=DEV).manual_seed(2)
    ps = [draw(gen, s, dtype) for s in SIZES]
    states = [be.adamw_state(p, 8, master) for p in ps]
    for t in range(1, 7):
        # gradients of very uneven size inside a group, zeros among them
        gs = [(draw(gen, s, torch.float32) * torch.exp(2 * torch.randn(s, generator=gen, device=DEV))
               * (torch.rand(s, generator=gen, device=DEV) < 0.9)).to(dtype) for s in SIZES]
        held = be.adamw_moments(states)
        before = [(s.master if master else p).clone() for p, s in zip(ps, states)]
        be.adamw_step(ps, gs, states, **HOW)
        for p, g, s, start, (m0, r0), (m1, r1) in zip(ps, gs, states, before, held, be.adamw_moments(states)):
            want, m, v = exact_step(start, g, m0, r0.double() ** 2, t, **HOW)
            assert held_near(m1, m, 3) and held_near(r1, v.sqrt(), 4)
            assert bool((r1[v > 0] > 0).all()) and bool((r1[v == 0] == 0).all())
            got = s.master if master else p
            if got.dtype == torch.float32:
                assert near_step(got, want, start.float(), HOW["lr"])
            if master:
                assert torch.equal(p, s.master.to(dtype))
            assert s.step.tolist() == [t, 0]
        for d in (torch.float16, torch.bfloat16):
            assert all(torch.equal(a, b.to(d)) for x, y in zip(be.adamw_moments(states, d), be.adamw_moments(states)) for a, b in zip(x, y))


def test_every_code_reads_back_as_itself():
    """All codes under all exponents a state can have: reading and holding them again (betas that leave a moment as it is) changes none."""
    exps = torch.tensor([1, 2, 15, 16, 100, 127, 128, 200, 253, 254], dtype=torch.uint8, device=DEV)
    n = exps.numel() * 256
    code = torch.arange(256, dtype=torch.uint8, device=DEV).repeat(exps.numel())
    scale = exps.repeat_interleave(2).repeat(2, 1).contiguous()
    state = be.AdamWState(code.clone(), code.clone(), torch.zeros(2, dtype=torch.int64, device=DEV), scale)
    (m, root), = be.adamw_moments([state])
    field = code.double() % 128
    low = torch.where(field < 8, field / 8 * 2.0 ** -14, (1 + field % 8 / 8) * torch.exp2(torch.floor(field / 8) - 15))
    e = scale[0].repeat_interleave(128).double() - 127
    want = torch.where(code >= 128, -low, low) * torch.exp2(e)
    assert torch.equal(m.double(), want.float().double())
    c = code.double()
    want = torch.where(c < 16, c / 16 * 2.0 ** -14, (1 + c % 16 / 16) * torch.exp2(torch.floor(c / 16) - 15)) * torch.exp2(e)
    assert torch.equal(root.double(), want.float().double())
    assert n == m.numel()


def test_groups_with_infinities_and_nan_and_groups_of_zeros():
    p = torch.ones(512, device=DEV)
    g = torch.full((512,), 0.5, device=DEV)
    g[130], g[300], g[384:] = math.inf, math.nan, 0.0
    state = be.adamw_state(p, 8)
    be.adamw_step([p], [g], [state], **HOW)
    bad = torch.zeros(512, dtype=torch.bool, device=DEV)
    bad[[130, 300]] = True
    assert torch.equal(torch.isnan(p), bad)                                   # (inf / inf)
    (m, r), = be.adamw_moments([state])
    nan = torch.zeros(512, dtype=torch.bool, device=DEV)
    nan[128:384] = True
    assert torch.equal(torch.isnan(m), nan) and torch.equal(torch.isnan(r), nan)
    assert bool((m[384:] == 0).all()) and bool((r[384:] == 0).all()) and bool((m[:128] == m[0]).all()) and float(m[0]) > 0
    assert bool((p[384:] == 1 - HOW["lr"] * HOW["weight_decay"]).all())        # no gradient ever: decay alone
    g.fill_(0.5)
    be.adamw_step([p], [g], [state], **HOW)
    assert torch.equal(torch.isnan(p), nan)
    # the same in 32 bits stays with the element
    p, state = torch.ones(512, device=DEV), be.adamw_state(torch.ones(512, device=DEV), 32)
    g[130] = math.nan
    be.adamw_step([p], [g], [state], **HOW)
    g.fill_(0.5)
    be.adamw_step([p], [g], [state], **HOW)
    assert torch.isnan(p).nonzero().view(-1).tolist() == [130]


@pytest.mark.parametrize("bits", (8, 32))
def test_tensors_at_any_place_in_memory(bits):
    """Slices of larger tensors, off every alignment; what lies beside them stays as it is."""
    gen = torch.Generator(device=DEV).manual_seed(3)
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        for n in (1, 5, 127, 130, 2050, 5001):
            flat, grad = draw(gen, (n + 8,), dtype), draw(gen, (n + 8,), dtype)
            whole = flat.clone()
            p, g = flat[3:3 + n], grad[1:1 + n]
            q, h = p.clone(), g.clone()
            kind = torch.uint8 if bits == 8 else torch.float32
            m, v = torch.zeros(n + 3, dtype=kind, device=DEV), torch.zeros(n + 5, dtype=kind, device=DEV)
            scale = torch.zeros(2 * -(-n // 128) + 1, dtype=torch.uint8, device=DEV) if bits == 8 else None
            a = be.AdamWState(m[1:1 + n], v[3:3 + n], torch.zeros(2, dtype=torch.int64, device=DEV),
                              None if bits == 32 else scale[1:].view(2, -1))
            b = be.adamw_state(q, bits)
            for _ in range(3):
                be.adamw_step([p], [g], [a], **HOW)
                be.adamw_step([q], [h], [b], **HOW)
            assert torch.equal(p, q) and torch.equal(a.exp_avg, b.exp_avg) and torch.equal(a.exp_avg_sq, b.exp_avg_sq)
            assert torch.equal(flat[:3], whole[:3]) and torch.equal(flat[3 + n:], whole[3 + n:])
            assert int(m[0]) == 0 and bool((m[1 + n:] == 0).all()) and bool((v[:3] == 0).all()) and bool((v[3 + n:] == 0).all())
            if bits == 8:
                assert int(scale[0]) == 0 and torch.equal(a.scale, b.scale)


def test_more_tensors_than_a_launch_takes_and_counts_of_their_own():
    gen = torch.Generator(device=DEV).manual_seed(4)
    shapes = [(int(n),) for n in torch.randint(1, 700, (110,), generator=torch.Generator().manual_seed(1))]
    shapes[17] = (0,)
    shapes[60] = (3_000_001,)
    ps, gs = [draw(gen, s, torch.float32) for s in shapes], [draw(gen, s, torch.float32) for s in shapes]
    one = [p.clone() for p in ps]
    states, alone = [be.adamw_state(p, 8 if i % 3 else 32) for i, p in enumerate(ps)], []
    for i, s in enumerate(states):
        s.step[0] = i * i                                   # a long history, a short one
        alone.append(copy.copy(s))
    for a, p in zip(alone, one):
        a.exp_avg, a.exp_avg_sq, a.step = a.exp_avg.clone(), a.exp_avg_sq.clone(), a.step.clone()
        a.scale = None if a.scale is None else a.scale.clone()
    be.adamw_step(ps, gs, states, **HOW)
    for i in range(110):
        be.adamw_step([one[i]], [gs[i]], [alone[i]], **HOW)
        assert torch.equal(one[i], ps[i]) and torch.equal(states[i].exp_avg, alone[i].exp_avg)
        assert states[i].step.tolist() == [i * i + 1, 0]
    be.adamw_step([], [], [])
    be.adamw_step([torch.zeros(0, device=DEV)], [torch.zeros(0, device=DEV)], [be.adamw_state(torch.zeros(0, device=DEV))])


def test_a_long_history_and_other_betas():
    for t in (1, 2, 1000, 10 ** 6, 2 ** 40):
        for betas in ((0.0, 0.0), (0.9, 0.999), (0.99, 0.99999)):
            p, g = torch.ones(300, device=DEV), torch.full((300,), 0.25, device=DEV)
            s = be.adamw_state(p)
            s.step[0] = t - 1
            be.adamw_step([p], [g], [s], lr=0.5, betas=betas, eps=1e-3, weight_decay=0.0)
            want = exact_step(torch.ones(300), torch.full((300,), 0.25), torch.zeros(300), torch.zeros(300), t, 0.5, betas, 1e-3, 0.0)[0]
            # (1 - beta as fp32 is off by 2^-24 of it)
            assert abs(float(p[0]) - float(want[0])) <= 2.0 ** -20 * (1 + 0.5 * abs(float(want[0]) - 1))


def test_a_rate_on_the_device_and_another_stream():
    gen = torch.Generator(device=DEV).manual_seed(5)
    p, g = draw(gen, (1000,), torch.float32), draw(gen, (1000,), torch.float32)
    q, a, b = p.clone(), be.adamw_state(p), be.adamw_state(p)
    rate = torch.tensor([0.03], device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        be.adamw_step([p], [g], [a], lr=rate)
    side.synchronize()
    be.adamw_step([q], [g], [b], lr=float(rate))
    assert torch.equal(p, q)
    be.adamw_step([q], [g], [b], lr=torch.tensor(0.03))
    with pytest.raises(ValueError):
        be.adamw_step([q], [g], [b], lr=rate.double())
    with pytest.raises(ValueError):
        be.adamw_step([q], [g], [b], lr=torch.ones(2, device=DEV))


def test_gradients_that_are_no_plain_memory():
    gen = torch.Generator(device=DEV).manual_seed(6)
    p = draw(gen, (40, 30), torch.float32)
    grad = draw(gen, (30, 40), torch.float32)
    for g in (grad.t(), draw(gen, (80, 30), torch.float32)[::2], torch.ones(1, 1, device=DEV).expand(40, 30),
              torch.view_as_complex(draw(gen, (40, 30, 2), torch.float32)).conj().imag):
        q, a, b = p.clone(), be.adamw_state(p), be.adamw_state(p)
        x = p.clone()
        be.adamw_step([x], [g], [a])
        be.adamw_step([q], [g.clone(memory_format=torch.contiguous_format).resolve_neg()], [b])
        assert torch.equal(x, q)


def test_refusals_of_the_step():
    p, g = torch.zeros(6, 4, device=DEV), torch.zeros(6, 4, device=DEV)
    s = be.adamw_state(p)
    for bad in (dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1.0)):
        with pytest.raises(ValueError):
            be.adamw_step([p], [g], [s], **bad)
    cases = [([p], [g], []), ([p, p], [g, g], [s, be.adamw_state(p)]), ([p], [g[:5]], [s]), ([p], [g.half()], [s]),
             ([p], [g.view(4, 6)], [s]), ([p.t()], [g.t()], [s]), ([p], [g.to_sparse()], [s]), ([p.double()], [g.double()], [s]),
             ([p], [g], [be.adamw_state(p.view(-1))]),
             ([p], [g], [be.AdamWState(s.exp_avg, s.exp_avg_sq, s.step[:1])]),
             ([p], [g], [be.AdamWState(s.exp_avg, s.exp_avg_sq.half(), s.step)]),
             ([p], [g], [be.AdamWState(s.exp_avg, s.exp_avg_sq, s.step, torch.zeros(2, 1, dtype=torch.uint8, device=DEV))]),
             ([p], [g], [be.AdamWState(s.exp_avg, s.exp_avg_sq, s.step, None, torch.zeros(6, 4, device=DEV))]),
             ([p], [g], [be.AdamWState(s.exp_avg.t().contiguous().t(), s.exp_avg_sq, s.step)])]
    for ps, gs, ss in cases:
        with pytest.raises((ValueError, RuntimeError)):
            be.adamw_step(ps, gs, ss)
    b = be.adamw_state(p, 8)
    b.scale = torch.zeros(2, 2, dtype=torch.uint8, device=DEV)
    with pytest.raises(ValueError):
        be.adamw_step([p], [g], [b])
    with pytest.raises(RuntimeError, match="no CPU path"):
        be.adamw_step([p.cpu()], [g.cpu()], [s])
    with pytest.raises(ValueError):
        be.adamw_step([p], [g.cpu()], [s])
    with pytest.raises(ValueError):
        be.adamw_moments([s])
    with pytest.raises(ValueError):
        be.adamw_state(p, 16)
    assert bool((p == 0).all()) and s.step.tolist() == [0, 0]


def test_what_was_saved_of_a_parameter_is_out_of_date_after_a_step():
    w = torch.randn(8, 8, device=DEV, requires_grad=True)
    x = torch.randn(3, 8, device=DEV, requires_grad=True)
    loss = (x @ w).square().sum()
    be.adamw_step([w.detach().requires_grad_(False)], [torch.ones_like(w)], [be.adamw_state(w)])
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()


# ----------------------------------------------------------------------------- the optimizer
def net(dtype=torch.float32, seed=0):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Linear(64, 128), torch.nn.ReLU(), torch.nn.Linear(128, 64), torch.nn.LayerNorm(64)).to(DEV, dtype)


def train(model, opt, steps, seed=1):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dtype = next(model.parameters()).dtype
    for _ in range(steps):
        x = torch.randn(32, 64, generator=gen, device=DEV).to(dtype)
        opt.zero_grad()
        (model(x) - x).float().square().mean().backward()
        opt.step()


def test_it_is_torch_s_adamw():
    a, b = net(), net()
    train(a, hiscache.AdamW(a.parameters(), lr=3e-3, weight_decay=0.05), 10)
    train(b, torch.optim.AdamW(b.parameters(), lr=3e-3, weight_decay=0.05), 10)
    for p, q in zip(a.parameters(), b.parameters()):
        # ten steps, each of at most lr or so and exact to 2^-18 of it; what one is off moves the next gradients as much again
        assert float((p - q).detach().abs().max()) <= 10 * 10 * 3e-3 * 2.0 ** -10
    groups = [dict(params=list(a[0].parameters()), lr=1e-3), dict(params=list(a[2].parameters()), weight_decay=0.0)]
    opt = hiscache.AdamW(groups, lr=5e-3, state_bits=8)
    sched = torch.optim.lr_scheduler.LambdaLR(opt, lambda i: 0.5 ** i)
    train(a, opt, 2)
    sched.step()
    assert [g["lr"] for g in opt.param_groups] == [5e-4, 2.5e-3]


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
def test_states_by_size_and_type(dtype):
    model = net(dtype)
    opt = hiscache.AdamW(model.parameters(), state_bits=8)
    for p in model[3].parameters():
        p.requires_grad_(False)                              # some have no gradient at first
    train(model, opt, 2)
    weight, bias = model[0].weight, model[0].bias
    assert opt.state[weight]["exp_avg"].dtype == torch.uint8 and opt.state[bias]["exp_avg"].dtype == torch.float32
    assert ("master" in opt.state[weight]) == (dtype == torch.bfloat16) and model[3].weight not in opt.state
    for p in model[3].parameters():
        p.requires_grad_(True)
    train(model, opt, 1)
    assert opt.state[weight]["step"].tolist() == [3, 0] and opt.state[model[3].weight]["step"].tolist() == [1, 0]
    m, v = opt.moments(weight)
    assert m.shape == v.shape == weight.shape and m.dtype == torch.float32 and bool((v >= 0).all())
    assert opt.moments(bias)[0] is opt.state[bias]["exp_avg"]


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("bits", (8, 32))
def test_a_checkpoint_goes_on_as_if_nothing_had_been(dtype, bits, tmp_path):
    whole = net(dtype)
    opt = hiscache.AdamW(whole.parameters(), lr=1e-2, state_bits=bits)
    train(whole, opt, 3)
    torch.save({"model": whole.state_dict(), "opt": opt.state_dict()}, tmp_path / "c.pt")
    saved = torch.load(tmp_path / "c.pt", weights_only=True)
    again = net(dtype, seed=5)
    more = hiscache.AdamW(again.parameters(), lr=1e-2, state_bits=bits)
    train(again, more, 1)
    again.load_state_dict(saved["model"])
    more.load_state_dict(saved["opt"])
    for p in again.parameters():
        assert more.state[p]["exp_avg"].dtype in (torch.uint8, torch.float32) and more.state[p]["step"].dtype == torch.int64
    twin = copy.deepcopy(again)
    other = hiscache.AdamW(twin.parameters(), lr=1e-2, state_bits=bits)
    other.load_state_dict(copy.deepcopy(more.state_dict()))
    for model, o in ((whole, opt), (again, more), (twin, other)):
        train(model, o, 3, seed=9)
    for a, b, c in zip(whole.parameters(), again.parameters(), twin.parameters()):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_weights_that_something_else_changed_are_taken_as_they_are():
    model = net(torch.bfloat16)
    opt = hiscache.AdamW(model.parameters(), lr=1e-4)
    train(model, opt, 3)
    w, master = model[0].weight, opt.state[model[0].weight]["master"]
    kept = master.clone()
    with torch.no_grad():
        w[5:9] = 3.0
    model.zero_grad()
    w.grad = torch.zeros_like(w)
    opt.param_groups[0].update(lr=0.0)
    opt.step()
    assert bool((master[5:9] == 3.0).all()) and torch.equal(master[:5], kept[:5]) and torch.equal(master[9:], kept[9:])
    # small steps add up in the copy, where the parameter itself would never move
    lone = torch.nn.Parameter(torch.ones(4096, device=DEV, dtype=torch.bfloat16))
    o = hiscache.AdamW([lone], lr=1e-4, weight_decay=0.0)
    lone.grad = torch.ones_like(lone)
    for _ in range(60):
        o.step()
    assert float(lone.detach()[0]) < 1


@pytest.mark.parametrize("bits", (8, 32))
def test_recorded_steps(bits):
    """A step in a graph, replayed, is the same as one by itself; two optimizers in graphs of their own do not disturb each other."""
    gen = torch.Generator(device=DEV).manual_seed(7)
    shapes = [(300, 70), (129,), (5000,)]

    def make():
        torch.manual_seed(3)
        ps = [torch.nn.Parameter(torch.randn(s, device=DEV)) for s in shapes]
        for p in ps:
            p.grad = torch.zeros_like(p)
        return ps, hiscache.AdamW(ps, lr=1e-2, state_bits=bits, min_elements=128)

    pairs = [make() for _ in range(3)]
    with pytest.raises(RuntimeError, match="recorded"):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            pairs[0][1].step()
    torch.cuda.synchronize()
    for _, opt in pairs:
        opt.step()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for g, (_, opt) in zip(graphs, pairs):
        with torch.cuda.graph(g):
            opt.step()
    for i in range(5):
        new = [torch.randn(s, generator=gen, device=DEV) for s in shapes]
        for ps, _ in pairs:
            for p, g in zip(ps, new):
                p.grad.copy_(g)
        for g in graphs:
            g.replay()
        pairs[2][1].step()
        torch.cuda.synchronize()
        for a, b, c in zip(*(ps for ps, _ in pairs)):
            assert torch.equal(a, c) and torch.equal(b, c)
    assert [opt.state[ps[0]]["step"].tolist() for ps, opt in pairs] == [[6, 0]] * 3


def test_refusals_of_the_optimizer():
    w = torch.nn.Parameter(torch.zeros(4, device=DEV))
    for bad in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1), dict(weight_decay=-1), dict(state_bits=4)):
        with pytest.raises(ValueError):
            hiscache.AdamW([w], **bad)
    host = torch.nn.Parameter(torch.zeros(4))
    host.grad = torch.zeros(4)
    with pytest.raises(RuntimeError, match="GPU"):
        hiscache.AdamW([host]).step()
    crossed = torch.nn.Parameter(torch.zeros(6, 4, device=DEV).t())
    crossed.grad = torch.zeros(4, 6, device=DEV)
    with pytest.raises(ValueError):
        hiscache.AdamW([crossed]).step()
    assert hiscache.AdamW([w]).step(lambda: 3.0) == 3.0       # nothing has a gradient


def test_tensors_of_more_than_2_31_elements():
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GiB of free device memory")
    n, tail = (1 << 31) + 5003, 9000
    p, g = torch.ones(n, device=DEV, dtype=torch.bfloat16), torch.zeros(n, device=DEV, dtype=torch.bfloat16)
    gen = torch.Generator(device=DEV).manual_seed(8)
    first = n - tail - (n - tail) % 128                      # (from the start of a group on)
    p[first:], g[first:] = draw(gen, (n - first,), torch.bfloat16), draw(gen, (n - first,), torch.bfloat16)
    q, h = p[first:].clone(), g[first:].clone()
    a, b = be.adamw_state(p, 8), be.adamw_state(q, 8)
    for _ in range(2):
        be.adamw_step([p], [g], [a], **HOW)
        be.adamw_step([q], [h], [b], **HOW)
    assert torch.equal(p[first:], q) and torch.equal(a.exp_avg[first:], b.exp_avg) and torch.equal(a.scale[:, first // 128:], b.scale)
    assert bool((p[:first] == p[0]).all()) and int(a.exp_avg[:first].max()) == 0 and a.step.tolist() == [2, 0]
    (m, _), = be.adamw_moments([a], torch.bfloat16)
    assert torch.equal(m[first:], be.adamw_moments([b], torch.bfloat16)[0][0])


@pytest.mark.parametrize("dtype", ("fp32", "bf16"))
def test_the_example_of_experts_runs_with_all_of_it(dtype):
    import importlib.util
    import os
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "history-cache_amd", "example", "experts.py")
    spec = importlib.util.spec_from_file_location("hiscache_example_experts", at)
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    losses = ex.run(ex.parse(["--nodes", "2000", "--steps", "4", "--score", "sigmoid", "--balance", "0.01", "--state-bits", "8",
                              "--dtype", dtype]), say=lambda *_: None)
    assert len(losses) == 4 and all(math.isfinite(v) for v in losses)


def test_a_state_goes_with_one_parameter():
    a, b = torch.zeros(300, device=DEV), torch.zeros(300, device=DEV)
    state, other = be.adamw_state(a), be.adamw_state(a)
    with pytest.raises(ValueError, match="one parameter"):
        be.adamw_step([a, b], [a + 1, b + 1], [state, state])
    with pytest.raises(ValueError, match="one parameter"):
        be.adamw_step([a, b], [a + 1, b + 1], [state, be.AdamWState(other.exp_avg, other.exp_avg_sq, state.step)])
    assert not bool(a.any()) and not bool(state.step.any())


@pytest.mark.parametrize("bits", (32, 8))
def test_steps_on_two_streams_at_once(bits):
    gen = torch.Generator(device=DEV).manual_seed(5)
    made = [[draw(gen, (700_001,), torch.float32), draw(gen, (33,), torch.float32)] for _ in range(2)]
    grads = [[draw(gen, p.shape, torch.float32) for p in ps] for ps in made]
    alone = [[p.clone() for p in ps] for ps in made]
    for ps, gs in zip(alone, grads):
        states = [be.adamw_state(p, bits) for p in ps]
        for _ in range(4):
            be.adamw_step(ps, gs, states, **HOW)
    kept = [[be.adamw_state(p, bits) for p in ps] for ps in made]
    streams = [torch.cuda.Stream() for _ in made]
    torch.cuda.synchronize()
    for _ in range(4):
        for st, ps, gs, states in zip(streams, made, grads, kept):
            with torch.cuda.stream(st):
                be.adamw_step(ps, gs, states, **HOW)
    torch.cuda.synchronize()
    for ps, want, states in zip(made, alone, kept):
        assert all(torch.equal(a, b) for a, b in zip(ps, want))
        assert all(s.step.tolist() == [4, 0] for s in states)
