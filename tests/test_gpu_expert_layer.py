"""The layer of experts as a whole: gated_experts and ExpertMLP against a loop over the experts in 64 bits, activations kept in
8 bits through autograd's hooks, and the example that runs them together."""
import importlib.util
import os

import pytest
import torch

import hiscache
import hiscache_backend as be

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EXAMPLE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "history-cache_amd", "example", "experts.py")


def gated64(rows, w_in, w_out, ends, kept=None):
    """The experts' results and the hidden rows' argument; ``kept``: the argument's values to compute from."""
    y, pre = rows.new_zeros(rows.shape[0], w_out.shape[1]), rows.new_zeros(rows.shape[0], w_in.shape[1])
    H = w_out.shape[2]
    for e in range(w_in.shape[0]):
        r = slice(ends[e], ends[e + 1])
        pre[r] = rows[r] @ w_in[e].t()
        p = pre[r] if kept is None else kept[r]
        y[r] = (torch.nn.functional.silu(p[:, :H]) * p[:, H:]) @ w_out[e].t()
    return y, pre


def rel(a, b):
    a, b = a.detach().double(), b.detach().double()
    return float((a - b).norm() / b.norm())


# rounding of the rows' type at every one of the few operations behind one another
LIMIT = {torch.float32: 1e-5, torch.float16: 8 * 2.0 ** -11, torch.bfloat16: 8 * 2.0 ** -8}


@pytest.mark.parametrize("dtype", tuple(LIMIT))
@pytest.mark.parametrize("C,H,D,group", ((64, 96, 64, 64), (47, 33, 20, 32), (128, 256, 128, 128)))
def test_gated_experts_forward_and_gradients(dtype, C, H, D, group):
    gen = torch.Generator(device=DEV).manual_seed(C)
    sizes = (70, 0, 200, 33)
    offset = torch.tensor((0,) + sizes, device=DEV).cumsum(0)
    ends, S = offset.tolist(), 320
    rows, w_in, w_out, g = (torch.randn(s, device=DEV, generator=gen) for s in ((S, C), (4, 2 * H, C), (4, D, H), (S, D)))
    rows, w_in, w_out, g = (t.to(dtype) for t in (rows, w_in / C ** 0.5, w_out / H ** 0.5, g))
    a = [t.detach().requires_grad_(True) for t in (rows, w_in, w_out)]
    y = be.gated_experts(*a, offset, group)
    grads = torch.autograd.grad(y, a, g)
    r64, i64, o64, g64 = (t.double() for t in (rows, w_in, w_out, g))
    want, pre = gated64(r64, i64, o64, ends)
    assert rel(y.detach(), want) <= LIMIT[dtype] and not y[ends[-1]:].any()
    # the gradients of the same loop at the argument as it was kept
    h, kept = be.gated_pack(be.expert_linear(rows, w_in, offset), group)
    leaf = torch.cat([be.unpack_rows(be.PackedRows(c.contiguous(), s.contiguous(), group, dtype), torch.float32) for c, s in
                      zip(kept.codes.split(H, 1), kept.scale.chunk(2, 1))], 1).double().requires_grad_(True)
    o64.requires_grad_(True)
    g_pre, g_o = torch.autograd.grad(gated64(r64, i64, o64, ends, leaf)[0], (leaf, o64), g64)
    want_rows, want_in = torch.zeros_like(r64), torch.zeros_like(i64)
    for e in range(4):
        r = slice(ends[e], ends[e + 1])
        want_rows[r], want_in[e] = g_pre[r] @ i64[e], g_pre[r].t() @ r64[r]
    for got, ref in zip(grads, (want_rows, want_in, g_o)):
        assert rel(got, ref) <= LIMIT[dtype]
    # and near those of the unrounded argument: a scale is 1 / 127 of a group's largest value, a few times its typical one
    leaf2 = pre.detach().requires_grad_(True)
    exact, = torch.autograd.grad(gated64(r64, i64, o64.detach(), ends, leaf2)[0], leaf2, g64)
    assert rel(g_pre, exact) <= 0.03
    with torch.no_grad():
        assert torch.equal(be.gated_experts(rows, w_in, w_out, offset, group), y)


@pytest.mark.parametrize("dtype", tuple(LIMIT))
@pytest.mark.parametrize("top_k,normalize", ((1, True), (2, True), (3, False)))
def test_expert_mlp(dtype, top_k, normalize):
    torch.manual_seed(top_k)
    layer = hiscache.ExpertMLP(64, 96, 6, top_k, normalize=normalize, device=DEV, dtype=dtype)
    x = torch.randn(500, 64, device=DEV).to(dtype).requires_grad_(True)
    out = layer(x)
    expert, weight = layer.route(x)
    want = torch.zeros(500, 64, dtype=torch.float64, device=DEV)
    x64, w_in, w_out = x.detach().double(), layer.w_in.detach().double(), layer.w_out.detach().double()
    for j in range(top_k):
        for e in range(6):
            r = expert[:, j] == e
            p = x64[r] @ w_in[e].t()
            want[r] += weight[r, j].double().unsqueeze(1) * ((torch.nn.functional.silu(p[:, :96]) * p[:, 96:]) @ w_out[e].t())
    assert rel(out.detach(), want) <= LIMIT[dtype]
    out.float().square().sum().backward()
    assert all(bool(torch.isfinite(p.grad).all()) for p in (x, *layer.parameters()))
    assert all(bool(p.grad.any()) for p in (x, layer.w_in, layer.w_out))
    # a single weight that is normalised is one whatever the router says
    assert bool(layer.router.grad.any()) == (top_k > 1 or not normalize)


def test_expert_mlp_by_given_experts_and_masks():
    torch.manual_seed(0)
    layer = hiscache.ExpertMLP(32, 64, 4, 2, device=DEV)
    x, types = torch.randn(90, 32, device=DEV), torch.arange(90, device=DEV) % 5 - 1
    out = layer(x, types)
    assert not out[types < 0].any() and out[types >= 0].any(1).all()
    assert torch.allclose(out, layer(x, types.unsqueeze(1), torch.ones(90, 1, device=DEV)))
    allowed = torch.zeros(90, 4, dtype=torch.bool, device=DEV)
    allowed[:30, 2] = True
    expert, weight = layer.route(x, allowed)
    assert expert[:30].tolist() == [[2, -1]] * 30 and bool((expert[30:] == -1).all()) and not weight[30:].any()
    assert not layer(x, allowed=allowed)[30:].any() and torch.equal(layer(x, allowed=allowed)[:30], layer(x[:30], torch.full((30,), 2, device=DEV)))
    with pytest.raises(ValueError):
        hiscache.ExpertMLP(32, 64, 4, 5)
    with pytest.raises(ValueError):
        be.gated_experts(x, layer.w_in[:, :100].contiguous(), layer.w_out, torch.zeros(5, dtype=torch.int64, device=DEV))


def test_packed_activations_keep_a_quarter():
    torch.manual_seed(1)
    net = torch.nn.Sequential(torch.nn.Linear(256, 512), torch.nn.GELU(), torch.nn.Linear(512, 256)).to(DEV)
    x = torch.randn(4096, 256, device=DEV)

    def step(context):
        net.zero_grad()
        before = torch.cuda.memory_allocated()
        with context:
            y = net(x)
        kept = torch.cuda.memory_allocated() - before - y.numel() * 4
        y.square().mean().backward()
        return kept, [p.grad.clone() for p in net.parameters()]

    import contextlib
    full, want = step(contextlib.nullcontext())
    packed, got = step(hiscache.packed_activations())
    # x is alive anyway, so that packing it adds a copy of a quarter; the two hidden matrices shrink to one byte and 1 / 16
    assert packed < 0.45 * full
    for a, b in zip(got, want):
        assert 0 < rel(a, b) < 0.03 or torch.equal(a, b)


def test_packed_activations_leave_small_and_whole_things_alone():
    with hiscache.packed_activations():
        w = torch.randn(300, 300, device=DEV, requires_grad=True)
        small = torch.randn(10, 300, device=DEV, requires_grad=True)
        y = (small @ w).sum()
    a, b = torch.autograd.grad(y, (small, w))
    assert torch.allclose(a, w.sum(1).expand(10, 300), rtol=1e-4, atol=1e-4) and torch.allclose(b, small.sum(0).unsqueeze(1).expand(300, 300), rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("dtype", ("fp32", "bf16"))
def test_the_example_learns(dtype):
    spec = importlib.util.spec_from_file_location("hiscache_example_experts", EXAMPLE)
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    said = []
    losses = ex.run(ex.parse(["--nodes", "3000", "--steps", "25", "--dtype", dtype]), said.append)
    assert len(losses) == 25 and losses[-1] < 0.8 * losses[0] and said
    full = ex.run(ex.parse(["--nodes", "3000", "--steps", "25", "--dtype", dtype, "--full-width"]), said.append)
    assert abs(full[0] - losses[0]) < 1e-5 and abs(full[-1] - losses[-1]) < 0.1 * full[0]
