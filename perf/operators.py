"""Cases of the expert layer's operators: routing, sorting rows by expert and back, the experts' products, and
activations kept in 8 bits.

``listed()`` names the cases that are always timed, ``draw(rng)`` gives further cases of the same ranges.
``prepare(case, seed)`` makes what a program has in hand before the call, ``run(state)`` is one pass: through the
public entry points of ``hiscache_backend`` where ``own`` is true, in elementary torch operations in 32 bits where it
is false. ``work(case)`` gives the bytes and operations that the pass cannot do without, ``exact(case, seed)`` the
outputs by the definitions in 64 bits.

The kinds of case:

* ``route``    logits of a row over the experts to its ``top_k`` experts and their weights (softmax, masked experts at
               -inf), in training with the gradient of the logits;
* ``sort``     (row, choice) pairs in expert order, rows copied there, the experts' results weighted and added up row by
               row, in training with all gradients; some choices name no expert (-1);
* ``product``  every row times its expert's matrix, in training with the gradients of rows and matrices;
* ``pack``     a matrix kept in 8 bits with a scale for each group of columns, and read back;
* ``gated``    silu(a) * b of [a | b], kept in 8 bits, and its gradient from what was kept.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"fp32": 4, "fp16": 2, "bf16": 2}
# Row widths in use around these operators, multiples of 64 and others.
WIDTHS = (47, 64, 100, 128, 172, 200, 256, 300, 384, 512, 602, 768, 1024, 1280)
SMALLEST = 2.0 ** -120      # a group of columns whose largest magnitude is below this is kept as zeros


def listed():
    return [
        # the next few rows of a model that answers, one row a request: latency of one small launch
        dict(name="route_step", kind="route", rows=8, experts=64, top_k=8, dtype="fp32", normalize=True, masked=0.0,
             train=False),
        # a training batch of half a million nodes over many experts, some of them closed to some rows
        dict(name="route_train", kind="route", rows=500_009, experts=64, top_k=4, dtype="bf16", normalize=True,
             masked=0.1, train=True),
        # the same few rows on their way to the experts and back
        dict(name="sort_step", kind="sort", rows=4, experts=16, top_k=2, width=1024, dtype="bf16", dropped=0.0, skew=0.5,
             train=False),
        # a training batch with many experts a row, wide half-precision rows
        dict(name="sort_train", kind="sort", rows=16_411, experts=64, top_k=4, width=1024, dtype="bf16", dropped=0.02,
             skew=1.0, train=True),
        # the nodes of a large sampled block, fp32 rows of a hidden width, few and unevenly loaded experts
        dict(name="sort_block", kind="sort", rows=200_003, experts=8, top_k=2, width=256, dtype="fp32", dropped=0.1,
             skew=1.5, train=True),
        # a few rows at their experts: every matrix that a row names is read for it
        dict(name="product_step", kind="product", rows=16, experts=16, inner=1024, outer=2048, dtype="bf16", dropped=0.0,
             skew=0.0, train=False),
        # a training batch through wide half-precision experts
        dict(name="product_train", kind="product", rows=32_771, experts=16, inner=1024, outer=2048, dtype="bf16",
             dropped=0.0, skew=0.7, train=True),
        # the nodes of a block through one fp32 map for each of five node types
        dict(name="product_block", kind="product", rows=60_007, experts=5, inner=256, outer=256, dtype="fp32", dropped=0.0,
             skew=1.0, train=True),
        # widths off every tile, uneven experts, rows that go nowhere
        dict(name="product_odd", kind="product", rows=20_011, experts=7, inner=172, outer=300, dtype="fp16", dropped=0.1,
             skew=1.0, train=True),
        # the input features of a block of odd width as a checkpoint
        dict(name="pack_features", kind="pack", rows=150_001, width=602, dtype="fp32", group=64),
        # the gate of a small batch: latency of two launches
        dict(name="gated_small", kind="gated", rows=96, width=512, dtype="bf16", group=64),
        # the gate inside wide experts, forward and backward of a training batch
        dict(name="gated_train", kind="gated", rows=65_537, width=1024, dtype="bf16", group=64),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("route", "sort", "product", "pack", "gated"))
    listed_work = [work(c) for c in listed() if c["kind"] == kind]
    most = {k: max(w[k] for w in listed_work) for k in ("bytes", "flops")}
    while True:
        dtype = rng.choice(sorted(DTYPES))
        if kind == "route":
            experts = _log_uniform(rng, 2, 256)
            c = dict(kind=kind, rows=_log_uniform(rng, 1, 1_000_000), experts=experts,
                     top_k=rng.randint(1, min(8, experts)), dtype=dtype, normalize=rng.random() < 0.5,
                     masked=rng.choice((0.0, 0.1, 0.5)), train=rng.random() < 0.7)
        elif kind == "sort":
            experts = _log_uniform(rng, 2, 256)
            c = dict(kind=kind, rows=_log_uniform(rng, 1, 400_000), experts=experts, top_k=rng.randint(1, min(8, experts)),
                     width=rng.choice(WIDTHS), dtype=dtype, dropped=rng.choice((0.0, 0.02, 0.3)),
                     skew=rng.choice((0.0, 1.0, 2.0)), train=rng.random() < 0.7)
        elif kind == "product":
            c = dict(kind=kind, rows=_log_uniform(rng, 1, 200_000), experts=_log_uniform(rng, 1, 64),
                     inner=rng.choice(WIDTHS), outer=rng.choice(WIDTHS), dtype=dtype, dropped=rng.choice((0.0, 0.1)),
                     skew=rng.choice((0.0, 1.0, 2.0)), train=rng.random() < 0.7)
        else:
            c = dict(kind=kind, rows=_log_uniform(rng, 1, 200_000), width=rng.choice(WIDTHS), dtype=dtype,
                     group=rng.choice((32, 64, 128)))
        w = work(c)
        # single precision multiplies at a small part of the half-precision rate
        dear = 8 if kind == "product" and dtype == "fp32" else 1
        if w["bytes"] <= most["bytes"] and dear * w["flops"] <= most["flops"]:
            return c


# ----------------------------------------------------------------------------- inputs
def _rand(gen, *shape):
    return torch.rand(shape, generator=gen, device=DEV)


def _randn(gen, dtype, *shape):
    return torch.randn(shape, generator=gen, device=DEV).to(dtype)


def _popularity(gen, experts, skew):
    """Log weights of the experts; the busiest half are a few times busier, and with eight and more one has no rows."""
    p = skew * torch.randn(experts, generator=gen, device=DEV)
    if experts >= 8:
        p[experts // 2] = -math.inf
    return p


def prepare(case, seed):
    if own:
        _backend()
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dtype, n, kind = DTYPES[case["dtype"]], case["rows"], case["kind"]
    s = dict(case=dict(case))
    if kind == "route":
        E, k = case["experts"], case["top_k"]
        logits = 2 * torch.randn(n, E, generator=gen, device=DEV)
        if case["masked"]:
            logits[_rand(gen, n, E) < case["masked"]] = -math.inf
            logits[:: 1001] = -math.inf                       # rows with no expert at all
        s.update(logits=logits.to(dtype), g_weight=_randn(gen, torch.float32, n, k))
    elif kind == "sort":
        E, k, D = case["experts"], case["top_k"], case["width"]
        noise = -torch.log(-torch.log(_rand(gen, n, E).clamp_(1e-20, 1 - 1e-6)))
        score, expert = torch.topk(noise + _popularity(gen, E, case["skew"]), k, dim=1)
        expert[torch.isneginf(score) | (_rand(gen, n, k) < case["dropped"])] = -1
        weight = torch.softmax(_randn(gen, torch.float32, n, k), dim=1)
        s.update(expert=expert.contiguous(), weight=weight * (expert >= 0), x=_randn(gen, dtype, n, D),
                 y=_randn(gen, dtype, n * k, D))
        if case["train"]:
            s.update(g_rows=_randn(gen, dtype, n * k, D), g_out=_randn(gen, dtype, n, D))
    elif kind == "product":
        E, K, N = case["experts"], case["inner"], case["outer"]
        share = torch.softmax(_popularity(gen, E, case["skew"]), 0).double()
        end = (torch.cumsum(share / share.sum(), 0) * (n * (1 - case["dropped"]))).round().to(torch.int64)
        s.update(offset=torch.cat([end.new_zeros(1), end.clamp_(max=n)]), x=_randn(gen, dtype, n, K),
                 w=(torch.randn(E, N, K, generator=gen, device=DEV) / math.sqrt(K)).to(dtype))
        if case["train"]:
            s.update(g=_randn(gen, dtype, n, N))
    else:
        F = case["width"] * (2 if kind == "gated" else 1)
        # activations of uneven size: a factor for each row and some columns that stand out
        x = torch.randn(n, F, generator=gen, device=DEV) * torch.exp(0.5 * torch.randn(n, 1, generator=gen, device=DEV))
        x *= 1 + 5 * (_rand(gen, 1, F) < 0.01)
        s.update(x=x.to(dtype))
        if kind == "gated":
            s.update(g=_randn(gen, dtype, n, case["width"]))
    return s


# ----------------------------------------------------------------------------- the framework's operators
def _backend():
    at = os.path.join(os.getcwd(), "history-cache_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import hiscache_backend
    return hiscache_backend


def _run_own(s):
    be, c = _backend(), s["case"]
    if c["kind"] == "route":
        if not c["train"]:
            return be.route_rows(s["logits"], c["top_k"], normalize=c["normalize"])
        logits = s["logits"].detach().requires_grad_(True)
        expert, weight = be.route_rows(logits, c["top_k"], normalize=c["normalize"])
        return expert, weight.detach(), torch.autograd.grad(weight, logits, s["g_weight"])[0]
    if c["kind"] == "sort":
        order = be.expert_order(s["expert"], c["experts"])
        if not c["train"]:
            rows = be.rows_to_experts(s["x"], order)
            out = be.rows_from_experts(s["y"], order, s["weight"])
            return order.slot, order.pair, order.offset, rows, out
        x, y, weight = (s[k].detach().requires_grad_(True) for k in ("x", "y", "weight"))
        rows = be.rows_to_experts(x, order)
        out = be.rows_from_experts(y, order, weight)
        grads = torch.autograd.grad((rows, out), (x, y, weight), (s["g_rows"], s["g_out"]))
        return (order.slot, order.pair, order.offset, rows.detach(), out.detach(), *grads)
    if c["kind"] == "product":
        if not c["train"]:
            return be.expert_linear(s["x"], s["w"], s["offset"])
        x, w = (s[k].detach().requires_grad_(True) for k in ("x", "w"))
        y = be.expert_linear(x, w, s["offset"])
        return (y.detach(), *torch.autograd.grad(y, (x, w), s["g"]))
    if c["kind"] == "pack":
        return be.unpack_rows(be.pack_rows(s["x"], c["group"]))
    h, kept = be.gated_pack(s["x"], c["group"])
    g_x, h_again = be.gated_grad(kept, s["g"])
    return h, g_x, h_again


# ----------------------------------------------------------------------------- plain forms
def _plain_route(s):
    c = s["case"]
    dtype, k = s["logits"].dtype, c["top_k"]
    logits = s["logits"].float()
    value, expert = torch.sort(logits, dim=1, descending=True, stable=True)      # ties: the lowest index first
    value, expert = value[:, :k], expert[:, :k]
    top = value[:, :1]
    none = torch.isneginf(value)
    e = torch.where(none, 0.0, torch.exp(value - top))
    if c["normalize"]:
        total = e.sum(1, keepdim=True)
    else:
        all_e = torch.where(torch.isneginf(logits), 0.0, torch.exp(logits - top))
        total = all_e.sum(1, keepdim=True)
    weight = torch.where(none, 0.0, e / total)
    out = (torch.where(none, -1, expert), weight)
    if not c["train"]:
        return out
    g = torch.where(none, 0.0, s["g_weight"])
    inner = (weight * g).sum(1, keepdim=True)
    if c["normalize"]:
        grad = torch.zeros_like(logits).scatter_(1, expert, weight * (g - inner))
    else:
        p = torch.where(torch.isneginf(logits), 0.0, all_e / total)
        grad = p * (torch.zeros_like(logits).scatter_(1, expert, g) - inner)
    return (*out, grad.to(dtype))


def _places(s):
    c = s["case"]
    E, flat = c["experts"], s["expert"].reshape(-1)
    kept = flat >= 0
    _, pair = torch.sort(torch.where(kept, flat, E), stable=True)
    count = torch.zeros(E + 1, dtype=torch.int64, device=DEV).index_add_(0, torch.where(kept, flat, E), torch.ones_like(flat))
    offset = torch.cat([count.new_zeros(1), torch.cumsum(count[:E], 0)])
    place = torch.empty_like(pair)
    place[pair] = torch.arange(pair.numel(), device=DEV)
    live = kept[pair]
    return torch.where(kept, place, -1).to(torch.int32), torch.where(live, pair, -1).to(torch.int32), offset


def _plain_sort(s):
    c = s["case"]
    n, k, D, dtype = c["rows"], c["top_k"], c["width"], s["x"].dtype
    slot, pair, offset = _places(s)
    live, kept = (pair >= 0).unsqueeze(1), (slot >= 0).view(n, k, 1)
    row, at = pair.clamp(min=0).long() // k, slot.clamp(min=0).long()
    rows = torch.where(live, s["x"].float()[row], 0.0)
    y = torch.where(kept, s["y"].float()[at].view(n, k, D), 0.0)
    out = (y * s["weight"].unsqueeze(2)).sum(1)
    first = (slot, pair, offset, rows.to(dtype), out.to(dtype))
    if not c["train"]:
        return first
    g_x = torch.where(kept, s["g_rows"].float()[at].view(n, k, D), 0.0).sum(1)
    g_out = s["g_out"].float()
    share = s["weight"].reshape(-1)[pair.clamp(min=0).long()].unsqueeze(1)
    g_y = torch.where(live, g_out[row] * share, 0.0)
    g_weight = (y * g_out.unsqueeze(1)).sum(2)
    return (*first, g_x.to(dtype), g_y.to(dtype), g_weight)


def _plain_product(s):
    dtype = s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    ends = s["offset"].tolist()
    y = torch.zeros(x.shape[0], w.shape[1], device=DEV)
    train = s["case"]["train"]
    if train:
        g, g_x, g_w = s["g"].float(), torch.zeros_like(x), torch.zeros_like(w)
    # one matrix product an expert: its rows are as many as it has, and the sizes of products are the host's to give
    for e in range(w.shape[0]):
        rows = slice(ends[e], ends[e + 1])
        y[rows] = x[rows] @ w[e].t()
        if train:
            g_x[rows] = g[rows] @ w[e]
            g_w[e] = g[rows].t() @ x[rows]
    return (y.to(dtype), g_x.to(dtype), g_w.to(dtype)) if train else y.to(dtype)


def _kept(x, group):
    """What rows kept in 8 bits stand for: x [n, F] in 32 bits."""
    n, F = x.shape
    groups = -(-F // group)
    x = torch.cat([x, x.new_zeros(n, groups * group - F)], 1).view(n, groups, group)
    most = x.abs().amax(2, keepdim=True)
    zero = most < SMALLEST
    code = torch.round(x * torch.where(zero, 0.0, 127.0 / most))
    return (code * torch.where(zero, 0.0, most / 127.0)).reshape(n, groups * group)[:, :F]


def _plain_gated(s):
    c, x, g = s["case"], s["x"].float(), s["g"].float()
    F, dtype = c["width"], s["x"].dtype
    a, b = x[:, :F], x[:, F:]
    h = a * (1 / (1 + torch.exp(-a))) * b
    a, b = _kept(a, c["group"]), _kept(b, c["group"])
    sig = 1 / (1 + torch.exp(-a))
    g_a, g_b = g * b * (sig * (1 + a * (1 - sig))), g * (a * sig)
    return h.to(dtype), torch.cat([g_a, g_b], 1).to(dtype), (a * sig * b).to(dtype)


def run(state):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    if kind == "pack":
        return _kept(state["x"].float(), state["case"]["group"]).to(state["x"].dtype)
    return {"route": _plain_route, "sort": _plain_sort, "product": _plain_product, "gated": _plain_gated}[kind](state)


# ----------------------------------------------------------------------------- what a pass needs
def work(case):
    n, b, kind = case["rows"], SIZES[case["dtype"]], case["kind"]
    if kind == "route":
        E, k, train = case["experts"], case["top_k"], case["train"]
        return dict(bytes=n * E * b * (1 + train) + n * k * (8 + 4 + 4 * train), flops=n * E * (4 + 4 * train))
    if kind == "sort":
        k, D, train = case["top_k"], case["width"], case["train"]
        P = n * k
        size = P * 8 + P * 4 + P * 8 + 8 * (case["experts"] + 1) + (2 * n + 2 * P) * D * b
        if train:
            size += (2 * n + 2 * P) * D * b + P * 4
        return dict(bytes=size, flops=P * D * (2 + 4 * train))
    if kind == "product":
        E, K, N, train = case["experts"], case["inner"], case["outer"], case["train"]
        live = n * (1 - case["dropped"])
        matrices = min(E - (E >= 8), n)               # at most: a matrix whose expert has no row need not be read
        size = (n * (K + N) + matrices * K * N) * b
        if train:
            size += (n * (K + N) + E * K * N) * b
        return dict(bytes=size, flops=2 * live * K * N * (3 if train else 1))
    F = case["width"] * (2 if kind == "gated" else 1)
    kept = n * (F + 4 * (F // case["width"]) * -(-case["width"] // case["group"]))        # codes and scales
    if kind == "pack":
        return dict(bytes=2 * n * F * b + 2 * kept, flops=6 * n * F)
    # [a | b] in, h out; the gradient of h in, the gradients of a and b and h again out
    return dict(bytes=n * F * b * 2 + 3 * n * case["width"] * b + 2 * kept, flops=40 * n * F)


# ----------------------------------------------------------------------------- definitions in 64 bits
def _exact_kept(x, group):
    n, F = x.shape
    out = torch.zeros_like(x)
    for lo in range(0, F, group):
        part = x[:, lo:lo + group]
        most = part.abs().max(dim=1, keepdim=True).values
        fine = most >= SMALLEST
        step = torch.where(fine, most, 1.0) / 127
        out[:, lo:lo + group] = torch.where(fine, torch.round(part / step) * step, 0.0)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind, n = case["kind"], case["rows"]
    if kind == "route":
        k, l = case["top_k"], s["logits"].double()
        p = torch.nan_to_num(torch.softmax(l, 1), nan=0.0)               # rows without any expert: nothing
        chosen, left = [], l.clone()
        index = torch.arange(case["experts"], device=DEV)
        for _ in range(k):
            best = left.max(1, keepdim=True).values
            at = torch.where(left == best, index, case["experts"]).min(1, keepdim=True).values
            chosen.append(torch.where(torch.isneginf(best), -1, at))
            # out of the running, without becoming a masked one: those are told from the logits
            left.scatter_(1, at, -math.inf)
        expert = torch.cat(chosen, 1)
        on = expert >= 0
        pick = torch.where(on, p.gather(1, expert.clamp(min=0)), 0.0)
        total = pick.sum(1, keepdim=True)
        weight = torch.where(on, pick / total, 0.0) if case["normalize"] else pick
        if not case["train"]:
            return expert, weight
        g = torch.where(on, s["g_weight"].double(), 0.0)
        dense_g = torch.zeros_like(l).scatter_add_(1, expert.clamp(min=0), g)
        dense_w = torch.zeros_like(l).scatter_add_(1, expert.clamp(min=0), weight)
        base = dense_w if case["normalize"] else p
        return expert, weight, base * (dense_g - (dense_w * dense_g).sum(1, keepdim=True))
    if kind == "sort":
        E, k, D = case["experts"], case["top_k"], case["width"]
        flat = s["expert"].reshape(-1)
        pairs = [torch.nonzero(flat == e).reshape(-1) for e in range(E)]
        count = torch.tensor([p.numel() for p in pairs], device=DEV)
        offset = torch.cat([count.new_zeros(1), torch.cumsum(count, 0)])
        pair = torch.cat(pairs)
        live = pair.numel()
        slot = torch.full_like(flat, -1)
        slot[pair] = torch.arange(live, device=DEV)
        all_pair = torch.cat([pair, pair.new_full((n * k - live,), -1)])
        rows, row = torch.zeros(n * k, D, dtype=torch.float64, device=DEV), pair // k
        rows[:live] = s["x"].double()[row]
        w = s["weight"].double().reshape(-1)
        out = torch.zeros(n, D, dtype=torch.float64, device=DEV)
        out.index_add_(0, row, s["y"][:live].double() * w[pair].unsqueeze(1))
        whole = (slot.to(torch.int32), all_pair.to(torch.int32), offset)
        if not case["train"]:
            return (*whole, rows, out)
        g_x = torch.zeros(n, D, dtype=torch.float64, device=DEV).index_add_(0, row, s["g_rows"][:live].double())
        g_y = torch.zeros(n * k, D, dtype=torch.float64, device=DEV)
        g_row = s["g_out"].double()[row]
        g_y[:live] = g_row * w[pair].unsqueeze(1)
        g_w = torch.zeros(n * k, dtype=torch.float64, device=DEV)
        g_w[pair] = (g_row * s["y"][:live].double()).sum(1)
        return (*whole, rows, out, g_x, g_y, g_w.view(n, k))
    if kind == "product":
        ends = s["offset"].tolist()
        x, w = s["x"].double(), s["w"].double()
        groups = [slice(ends[e], ends[e + 1]) for e in range(w.shape[0])]
        rest = x.new_zeros(n - ends[-1], 1)
        y = torch.cat([x[r] @ w[e].t() for e, r in enumerate(groups)] + [rest.expand(-1, w.shape[1])])
        if not case["train"]:
            return y
        g = s["g"].double()
        g_x = torch.cat([g[r] @ w[e] for e, r in enumerate(groups)] + [rest.expand(-1, w.shape[2])])
        return y, g_x, torch.stack([g[r].t() @ x[r] for r in groups])
    x = s["x"].double()
    if kind == "pack":
        return _exact_kept(x, case["group"])
    F, g = case["width"], s["g"].double()
    h = torch.nn.functional.silu(x[:, :F]) * x[:, F:]
    a, b = _exact_kept(x[:, :F], case["group"]), _exact_kept(x[:, F:], case["group"])
    sig = torch.sigmoid(a)
    silu = a * sig
    return h, torch.cat([g * b * (sig + silu * (1 - sig)), g * silu], 1), silu * b
