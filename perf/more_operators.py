"""Cases of three further operators: routing by scores with a bias for balance and groups of experts, a ring cache of
embeddings held in 8 bits (written by admission, read back by lookup), and an AdamW step over many tensors at once with
states in 8 or in 32 bits.

``listed()`` names the cases that are always timed, ``draw(rng)`` gives further cases of the same ranges.
``prepare(case, seed)`` makes what a program has in hand before the call, ``run(state)`` is one pass: through the
public entry points of ``hiscache_backend`` where ``own`` is true, in elementary torch operations where it is false
(32 bits; 64 where two scores are compared). ``work(case)`` gives the bytes and operations that the pass cannot do
without, ``exact(case, seed)`` the outputs by the definitions in 64 bits.

The kinds of case:

* ``route``  logits of a row over the experts to its ``top_k`` experts and their weights: sigmoid or softmax scores, a bias
             that takes part in the choice alone, the best ``top_group`` of ``groups`` groups of experts, in training with the
             gradient of the logits;
* ``ring``   one batch's admission to a ring of embeddings (rows under a threshold take the next slots, in 8 bits with a scale
             for each group of columns) and the next batch's lookup (slots, and the rows of the hits read back);
* ``adamw``  one step over a list of tensors; states in 8 bits are read back as the values that they stand for.
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
WIDTHS = (47, 64, 100, 128, 172, 200, 256, 300, 384, 512, 602, 768, 1024)
SMALLEST = 2.0 ** -120      # a group of columns whose largest magnitude is below this is kept as zeros
ADAM = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2)
ADAM_GROUP = 128            # adjacent elements that share an exponent where states are held in 8 bits
AGE_LIMIT = 1000            # iterations after which an entry of the ring counts as absent


def listed():
    return [
        # the next few rows of a model that answers, one row a request: latency of one small launch
        dict(name="route_step", kind="route", rows=8, experts=256, groups=8, top_group=4, top_k=8, score="sigmoid", dtype="fp32",
             bias=True, normalize=True, scale=2.5, masked=0.0, train=False),
        # a training batch of half a million nodes over many experts that a bias keeps in balance
        dict(name="route_train", kind="route", rows=500_009, experts=64, groups=1, top_group=1, top_k=4, score="sigmoid",
             dtype="bf16", bias=True, normalize=True, scale=1.0, masked=0.0, train=True),
        # a training batch over experts that lie in groups, of which a row may take half
        dict(name="route_groups", kind="route", rows=65_537, experts=256, groups=8, top_group=4, top_k=8, score="sigmoid",
             dtype="fp32", bias=True, normalize=True, scale=2.5, masked=0.0, train=True),
        # softmax weights as they are, experts off every power of two, some closed to some rows
        dict(name="route_odd", kind="route", rows=200_003, experts=60, groups=6, top_group=3, top_k=6, score="softmax",
             dtype="fp16", bias=False, normalize=False, scale=1.0, masked=0.1, train=True),
        # the plumbing configuration's batch: 100 000 nodes, hidden width 128
        dict(name="ring_step", kind="ring", nodes=100_000, capacity=60_000, rows=1_500, lookups=1_500, width=128, group=64,
             admitted=0.5, hits=0.35),
        # the 1-hop nodes of a batch from a large graph, hidden width 256
        dict(name="ring_batch", kind="ring", nodes=8_000_000, capacity=3_000_000, rows=8_661, lookups=8_661, width=256, group=64,
             admitted=0.5, hits=0.35),
        # a block of many batches at once, and their lookups
        dict(name="ring_block", kind="ring", nodes=6_000_000, capacity=2_500_000, rows=1_000_003, lookups=1_000_003, width=256,
             group=64, admitted=0.4, hits=0.4),
        # a width off every group of columns
        dict(name="ring_odd", kind="ring", nodes=2_000_000, capacity=700_001, rows=200_003, lookups=150_001, width=172, group=32,
             admitted=0.3, hits=0.5),
        # a two-layer model of width 128: a dozen small tensors, latency
        dict(name="adamw_small", kind="adamw", tensors="128x128,128x128,128,128,128,128x10,10x128,10", dtype="fp32", bits=32,
             master=False),
        # the matrices of wide experts in half precision beside a router, states in 8 bits
        dict(name="adamw_experts", kind="adamw", tensors="16x2048x1024,16x1024x1024,64x1024,1024", dtype="bf16", bits=8,
             master=True),
        # a large model's fp32 matrices, states in 8 bits
        dict(name="adamw_large", kind="adamw", tensors="64x2048x1024,64x1024x1024,1024x602,1024", dtype="fp32", bits=8,
             master=False),
        # odd sizes in half precision, states in 32 bits
        dict(name="adamw_odd", kind="adamw", tensors="7x300x172,300x7,47,1,602x129,1000003", dtype="fp16", bits=32, master=True),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("route", "ring", "adamw"))
    most = max(work(c)["bytes"] for c in listed() if c["kind"] == kind)
    while True:
        if kind == "route":
            groups = rng.choice((1, 1, 2, 4, 6, 8))
            experts = groups * _log_uniform(rng, 2, 256 // groups)
            top_group = rng.randint(1, groups)
            c = dict(kind=kind, rows=_log_uniform(rng, 1, 1_000_000), experts=experts, groups=groups, top_group=top_group,
                     top_k=rng.randint(1, min(8, experts // groups * top_group)), score=rng.choice(("sigmoid", "softmax")),
                     dtype=rng.choice(sorted(DTYPES)), bias=rng.random() < 0.7, normalize=rng.random() < 0.6,
                     scale=rng.choice((1.0, 2.5)), masked=rng.choice((0.0, 0.1, 0.5)), train=rng.random() < 0.7)
        elif kind == "ring":
            nodes = _log_uniform(rng, 50_000, 6_000_000)
            c = dict(kind=kind, nodes=nodes, capacity=int(nodes * rng.uniform(0.2, 0.7)), rows=_log_uniform(rng, 1, nodes // 6),
                     lookups=_log_uniform(rng, 1, nodes // 6), width=rng.choice(WIDTHS), group=rng.choice((32, 64, 128)),
                     admitted=rng.choice((0.05, 0.3, 0.65)), hits=rng.choice((0.1, 0.35, 0.7)))
        else:
            shapes = []
            for _ in range(rng.randint(1, 10)):
                n = _log_uniform(rng, 1, 20_000_000)
                cols = rng.choice(WIDTHS)
                shapes.append(str(n) if n < 2 * cols else f"{n // cols}x{cols}")
            dtype = rng.choice(sorted(DTYPES))
            c = dict(kind=kind, tensors=",".join(shapes), dtype=dtype, bits=rng.choice((8, 32)),
                     master=dtype != "fp32" and rng.random() < 0.7)
        if work(c)["bytes"] <= most:
            return c


# ----------------------------------------------------------------------------- states of 8 bits
def _binade(x):
    """The exponent e of 2^e <= |x| < 2^(e + 1) (int32; of zeros: far below every other)."""
    return torch.where(x == 0, -1000, torch.frexp(x)[1] - 1)


def _rounded(x, e, bits):
    """x to ``bits`` binary places behind the point in units of 2^e, ties to even (64 bits inside: scaling is exact there)."""
    step = torch.exp2((e - bits).double())
    return torch.round(x.double() / step) * step


def _kept_moment(x, bits, keep):
    """What a moment [elements] held in 8 bits stands for, and the exponent of each group: four bits of exponent under the group's
    largest magnitude, ``bits`` of mantissa; a value above zero stays above it where ``keep``."""
    n = x.numel()
    groups = -(-n // ADAM_GROUP)
    x = torch.cat([x, x.new_zeros(groups * ADAM_GROUP - n)]).view(groups, ADAM_GROUP)
    most = x.abs().amax(1, keepdim=True)
    top = _binade(_rounded(most, _binade(most), bits).float())
    dead = top < -126                                   # below the smallest normal number: zeros
    low = torch.where(dead, 0, top - 14)                # the binade of the smallest normal code; under it, its steps
    value = _rounded(x, torch.maximum(_binade(x), low), bits)
    if keep:
        value = torch.where((x > 0) & (value == 0), torch.exp2((low - bits).double()), value)
    return torch.where(dead, 0.0, value).float(), torch.where(dead, 0, top + 127).to(torch.uint8).view(-1)


def _codes(value, exponent, bits):
    """The codes of values that :func:`_kept_moment` gave, uint8 [elements]."""
    low = (exponent.to(torch.int32) - 127 - 14).view(-1, 1)
    e = torch.maximum(_binade(value), low)
    units = torch.round(value.abs().double() / torch.exp2((e - bits).double())).to(torch.int32)     # from 2^bits on: a normal code
    code = torch.where(units >= 1 << bits, (e - low + 1) * (1 << bits) + (units - (1 << bits)), units)
    if bits == 3:
        code = code + 128 * torch.signbit(value).to(torch.int32) * (value != 0)
    return torch.where(exponent.view(-1, 1) == 0, 0, code).to(torch.uint8).view(-1)


def _read_codes(code, exponent, bits):
    """The values that codes stand for, fp32 [elements]."""
    n, groups = code.numel(), exponent.numel()
    c = torch.cat([code, code.new_zeros(groups * ADAM_GROUP - n)]).view(groups, ADAM_GROUP).to(torch.int32)
    sign = torch.where(c >= 128, -1.0, 1.0) if bits == 3 else 1.0
    field = c & 127 if bits == 3 else c
    units = torch.where(field < 1 << bits, field, (field & ((1 << bits) - 1)) + (1 << bits))
    e = torch.clamp(field >> bits, min=1) - 1 + exponent.to(torch.int32).view(-1, 1) - 127 - 14 - bits
    value = sign * units.double() * torch.exp2(e.double())
    return torch.where(exponent.view(-1, 1) == 0, 0.0, value).float().view(-1)[:n]


# ----------------------------------------------------------------------------- inputs
def _rand(gen, *shape):
    return torch.rand(shape, generator=gen, device=DEV)


def _randn(gen, dtype, *shape):
    return torch.randn(shape, generator=gen, device=DEV).to(dtype)


def _shapes(case):
    return [tuple(int(v) for v in t.split("x")) for t in case["tensors"].split(",")]


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    kind = case["kind"]
    s = dict(case=dict(case))
    if kind == "route":
        n, E, k = case["rows"], case["experts"], case["top_k"]
        logits = 2 * torch.randn(n, E, generator=gen, device=DEV)
        if case["masked"]:
            logits[_rand(gen, n, E) < case["masked"]] = -math.inf
            logits[:: 1001] = -math.inf                       # rows with no expert at all
        s.update(logits=logits.to(DTYPES[case["dtype"]]), g_weight=_randn(gen, torch.float32, n, k),
                 bias=0.1 * _randn(gen, torch.float32, E) if case["bias"] else None)
    elif kind == "ring":
        N, cap, n, m, F = (case[k] for k in ("nodes", "capacity", "rows", "lookups", "width"))
        groups = -(-F // case["group"])
        # a ring that has gone round: every slot has a node, its row, and the iteration that brought it
        node = torch.randperm(N, generator=gen, device=DEV)
        held, absent = node[:cap], node[cap:]
        full2slot = torch.full((N,), -1, dtype=torch.int64, device=DEV)
        full2slot[held] = torch.arange(cap, device=DEV)
        codes = torch.randint(-127, 128, (cap, F), generator=gen, device=DEV, dtype=torch.int8)
        scale = torch.exp(0.5 * torch.randn(cap, groups, generator=gen, device=DEV)) / 127
        # the batch: a part of its rows was served from the ring, the others may enter it where their score is low
        known = int(n * 0.3)
        ids = torch.cat([held[torch.randperm(cap, generator=gen, device=DEV)[:known]], absent[:n - known]])
        ids = ids[torch.randperm(ids.numel(), generator=gen, device=DEV)].contiguous()
        emb = torch.randn(n, F, generator=gen, device=DEV) * torch.exp(0.5 * torch.randn(n, 1, generator=gen, device=DEV))
        emb = torch.relu(emb)                                 # embeddings behind a layer's activation: half of them zeros
        # the next batch: nodes of the ring, of this batch, and others
        old = int(m * case["hits"])
        pool = torch.cat([held[torch.randperm(cap, generator=gen, device=DEV)[:old]], ids[: (m - old) // 2]])
        new = absent[torch.randperm(absent.numel(), generator=gen, device=DEV)[: m - pool.numel()]]
        pool = torch.cat([pool, new])
        s.update(ids=ids, slot=full2slot[ids].contiguous(), emb=emb, score=_rand(gen, n),
                 thres=torch.full((1,), min(1.0, case["admitted"] / 0.7), device=DEV), codes=codes, scale=scale,
                 full2slot=full2slot, slot2full=held.clone(),
                 checkin=torch.randint(0, 1200, (cap,), generator=gen, device=DEV), header=torch.full((1,), cap - n // 5, device=DEV) % cap,
                 lookup=pool[torch.randperm(pool.numel(), generator=gen, device=DEV)].contiguous(), it=1200)
    else:
        dtype, tensors = DTYPES[case["dtype"]], []
        step = torch.zeros(len(_shapes(case)), 2, dtype=torch.int64, device=DEV)
        for i, shape in enumerate(_shapes(case)):
            numel = math.prod(shape)
            p = torch.randn(shape, generator=gen, device=DEV) / math.sqrt(shape[-1])
            # gradients of uneven size: a factor for each row
            size = 0.01 * torch.exp(torch.randn(shape[:-1] + (1,), generator=gen, device=DEV))
            g = (size * torch.randn(shape, generator=gen, device=DEV)).to(dtype)
            m = (0.3 * size * torch.randn(shape, generator=gen, device=DEV)).view(-1)
            r = (size * (0.2 + _rand(gen, *shape))).view(-1)
            step[i, 0] = 7 + 100 * i
            t = dict(p=p.to(dtype), g=g, step=step[i], scale=None, master=None)
            if case["master"]:
                t["master"] = p
            if case["bits"] == 8:
                value, em = _kept_moment(m, 3, False)
                root, er = _kept_moment(r, 4, True)
                t.update(m=_codes(value, em, 3)[:numel].view(shape), v=_codes(root, er, 4)[:numel].view(shape),
                         scale=torch.stack([em, er]))
            else:
                t.update(m=m.view(shape), v=(r * r).view(shape))
            tensors.append(t)
        s.update(tensors=tensors, steps=step)
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
        how = dict(normalize=c["normalize"], score=c["score"], bias=s["bias"], num_group=c["groups"], top_group=c["top_group"],
                   scale=c["scale"])
        if not c["train"]:
            return be.route_rows(s["logits"], c["top_k"], **how)
        logits = s["logits"].detach().requires_grad_(True)
        expert, weight = be.route_rows(logits, c["top_k"], **how)
        return expert, weight.detach(), torch.autograd.grad(weight, logits, s["g_weight"])[0]
    if c["kind"] == "ring":
        if "table" not in s:                                  # a program keeps these handles beside the tensors
            s["table"] = be.PackedRows(s["codes"], s["scale"], c["group"], torch.float32)
        table = s["table"]
        mask, _ = be.grad_check(None, s["emb"], s["slot"], s["ids"], s["thres"], table, s["full2slot"], s["slot2full"],
                                s["header"], s["it"], checkin=s["checkin"], score=s["score"])
        slot, rows = be.ring_lookup(s["full2slot"], s["lookup"], table, checkin=s["checkin"], now=s["it"] + 1,
                                    age_limit=AGE_LIMIT)
        return mask, s["header"], s["full2slot"], s["slot2full"], s["checkin"], slot, rows
    if "states" not in s:
        s["states"] = [be.AdamWState(t["m"], t["v"], t["step"], t["scale"], t["master"]) for t in s["tensors"]]
    states = s["states"]
    be.adamw_step([t["p"] for t in s["tensors"]], [t["g"] for t in s["tensors"]], states, **ADAM)
    if c["bits"] == 32:
        moments = [(t["m"], t["v"]) for t in s["tensors"]]
    else:
        moments = be.adamw_moments(states, torch.bfloat16)
    return s["steps"], [(t["p"], t["master"], *mv) for t, mv in zip(s["tensors"], moments)]


# ----------------------------------------------------------------------------- plain forms
def _plain_route(s):
    c, dtype = s["case"], s["logits"].dtype
    n, E, k, G = c["rows"], c["experts"], c["top_k"], c["groups"]
    # which is larger is decided in 64 bits
    l = s["logits"].double()
    closed = torch.isneginf(l)
    if c["score"] == "sigmoid":
        score = 1 / (1 + torch.exp(-l))
    else:
        e = torch.where(closed, 0.0, torch.exp(l - l.amax(1, keepdim=True)))
        score = torch.where(closed, 0.0, e / e.sum(1, keepdim=True))
    choice = score if s["bias"] is None else score + s["bias"].double()
    choice = torch.where(closed, -math.inf, choice)
    if G > 1:
        best = torch.sort(choice.view(n, G, E // G), dim=2, descending=True).values[:, :, :2]
        rank = torch.where(torch.isneginf(best), 0.0, best).sum(2)
        rank = torch.where(torch.isneginf(best[:, :, 0]), -math.inf, rank)
        group = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :c["top_group"]]
        open_ = torch.zeros(n, G, dtype=torch.bool, device=DEV).scatter_(1, group, True)
        choice = torch.where(open_.repeat_interleave(E // G, 1), choice, -math.inf)
    value, expert = torch.sort(choice, dim=1, descending=True, stable=True)          # ties: the lowest index first
    value, expert = value[:, :k], expert[:, :k]
    none = torch.isneginf(value)
    score = score.float()
    picked = torch.where(none, 0.0, score.gather(1, expert))
    total = picked.sum(1, keepdim=True) if c["normalize"] else torch.ones(n, 1, device=DEV)
    total = torch.where(total == 0, 1.0, total)
    share = picked / total
    out = (torch.where(none, -1, expert), c["scale"] * share)
    if not c["train"]:
        return out
    g = torch.where(none, 0.0, c["scale"] * s["g_weight"])
    inner = (share * g).sum(1, keepdim=True)
    grad = torch.zeros(n, E, device=DEV)
    if c["score"] == "sigmoid":
        l = l.float().gather(1, expert)
        slope = torch.where(none, 0.0, picked * (1 / (1 + torch.exp(l))))
        grad.scatter_(1, expert, slope * ((g - inner) / total if c["normalize"] else g))
    elif c["normalize"]:
        grad.scatter_(1, expert, share * (g - inner))
    else:
        grad = score * (grad.scatter_(1, expert, g) - inner)
    return (*out, grad.to(dtype))


def _plain_ring(s):
    c = s["case"]
    n, F, cap, group = c["rows"], c["width"], c["capacity"], c["group"]
    groups = -(-F // group)
    full2slot, slot2full, checkin, header = s["full2slot"], s["slot2full"], s["checkin"], s["header"]
    mask = (s["score"] < s["thres"]) & (s["slot"] == -1)
    # admitted rows take the next slots in the order of the rows
    row = torch.nonzero(mask).view(-1)
    at = (header + torch.arange(row.numel(), device=DEV)) % cap
    header.add_(row.numel()).remainder_(cap)
    before, node = slot2full[at], s["ids"][row]
    # (more rows than slots: the ring keeps the last ones; no case has that)
    gone = before[(before >= 0) & (full2slot[before.clamp(min=0)] == at)]
    full2slot[gone] = -1
    full2slot[node] = at
    slot2full[at] = node
    checkin[at] = s["it"]
    x = s["emb"][row]
    x = torch.cat([x, x.new_zeros(row.numel(), groups * group - F)], 1).view(-1, groups, group)
    most = x.abs().amax(2, keepdim=True)
    zero = most < SMALLEST
    code = torch.round(x * torch.where(zero, 0.0, 1.0 / most * 127.0))
    s["codes"][at] = code.view(-1, groups * group)[:, :F].to(torch.int8)
    s["scale"][at] = torch.where(zero, 0.0, most * torch.tensor(1.0 / 127.0, device=DEV)).view(-1, groups)
    # the next batch's lookup
    slot = full2slot[s["lookup"]]
    slot = torch.where((slot >= 0) & (s["it"] + 1 - checkin[slot.clamp(min=0)] < AGE_LIMIT), slot, -1)
    hit = slot.clamp(min=0)
    rows = s["codes"][hit].float() * s["scale"][hit].repeat_interleave(group, 1)[:, :F]
    return mask, header, full2slot, slot2full, checkin, slot, torch.where((slot >= 0).unsqueeze(1), rows, 0.0)


def _plain_adamw_one(t, bits, a):
    shape, dtype = t["p"].shape, t["p"].dtype
    b1, b2 = a["betas"]
    p = (t["p"].float() if t["master"] is None else t["master"]).view(-1)
    g = t["g"].float().view(-1)
    if bits == 32:
        m, v = t["m"].view(-1), t["v"].view(-1)
    else:
        m = _read_codes(t["m"].view(-1), t["scale"][0], 3)
        root = _read_codes(t["v"].view(-1), t["scale"][1], 4)
        v = root * root
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    count = t["step"][:1] + 1
    t["step"][:1] = count
    size = (a["lr"] / (1 - b1 ** count.double())).float()
    lift = (1 / torch.sqrt(1 - b2 ** count.double())).float()
    root = torch.sqrt(v)
    p = p * (1 - a["lr"] * a["weight_decay"]) - size * (m / (root * lift + a["eps"]))
    if t["master"] is not None:
        t["master"].copy_(p.view(shape))
    t["p"].copy_(p.view(shape).to(dtype))
    if bits == 32:
        t["m"].copy_(m.view(shape))
        t["v"].copy_(v.view(shape))
        return t["p"], t["master"], t["m"], t["v"]
    n = p.numel()
    m, em = _kept_moment(m, 3, False)
    root, er = _kept_moment(root, 4, True)
    t["m"].copy_(_codes(m, em, 3)[:n].view(shape))
    t["v"].copy_(_codes(root, er, 4)[:n].view(shape))
    t["scale"][0], t["scale"][1] = em, er
    return (t["p"], t["master"], m.view(-1)[:n].view(shape).to(torch.bfloat16), root.view(-1)[:n].view(shape).to(torch.bfloat16))


def run(state):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    if kind == "route":
        return _plain_route(state)
    if kind == "ring":
        return _plain_ring(state)
    # one tensor after the other: their sizes differ
    return state["steps"], [_plain_adamw_one(t, state["case"]["bits"], ADAM) for t in state["tensors"]]


# ----------------------------------------------------------------------------- what a pass needs
def work(case):
    kind = case["kind"]
    if kind == "route":
        n, E, k, b, train = case["rows"], case["experts"], case["top_k"], SIZES[case["dtype"]], case["train"]
        return dict(bytes=n * E * b * (1 + train) + n * k * (8 + 4 + 4 * train) + 4 * E, flops=n * E * (6 + 4 * train))
    if kind == "ring":
        n, m, F = case["rows"], case["lookups"], case["width"]
        packed = F + 4 * -(-F // case["group"])
        admitted, found = n * case["admitted"], m * case["hits"]
        # scores, slots and masks of the batch; the admitted rows in and out, with their ids and maps; the lookup's ids and
        # slots, its hits' ages and rows in, all its rows out
        return dict(bytes=int(n * 13 + admitted * (4 * F + packed + 8 * 6) + m * (8 + 8 + 8 + 4 * F) + found * (8 + packed)),
                    flops=int(admitted * F * 4 + found * F))
    n = sum(math.prod(s) for s in _shapes(case))
    b = SIZES[case["dtype"]]
    kept = (2 if case["bits"] == 8 else 8) + (4 if case["master"] else 0)
    # gradient in; parameter out (and in, where it has no copy in 32 bits); states and copies in and out; 8 bits as values out
    return dict(bytes=n * (b + b + (0 if case["master"] else b) + 2 * kept + (4 if case["bits"] == 8 else 0)), flops=n * 16)


# ----------------------------------------------------------------------------- definitions in 64 bits
def _exact_route(case, s):
    n, E, k, G = case["rows"], case["experts"], case["top_k"], case["groups"]
    l = s["logits"].double().requires_grad_(case["train"])
    masked = torch.isneginf(s["logits"])
    if case["score"] == "sigmoid":
        score = torch.sigmoid(l)
    else:
        score = torch.softmax(torch.where(masked.all(1, keepdim=True), 0.0, l), 1)
    left = score.detach().clone()
    if s["bias"] is not None:
        left += s["bias"].double()
    left[masked] = -math.inf
    if G > 1:
        parts = left.view(n, G, E // G)
        first = parts.max(2).values
        second = parts.scatter(2, parts.max(2, keepdim=True).indices, -math.inf).max(2).values
        rank = first + torch.where(second > -math.inf, second, 0.0)
        # a group is in where fewer than top_group others are ahead of it
        ahead = torch.zeros(n, G, dtype=torch.int64, device=DEV)
        for j in range(G):
            before = (rank[:, j:j + 1] > rank) | ((rank[:, j:j + 1] == rank) & (torch.arange(G, device=DEV) > j))
            ahead += before
        out = (ahead >= case["top_group"]).unsqueeze(2).expand(n, G, E // G).reshape(n, E)
        left[out] = -math.inf
    chosen, index = [], torch.arange(E, device=DEV)
    for _ in range(k):
        best = left.max(1, keepdim=True).values
        at = torch.where(left == best, index, E).min(1, keepdim=True).values
        chosen.append(torch.where(torch.isneginf(best), -1, at))
        left.scatter_(1, at, -math.inf)
    expert = torch.cat(chosen, 1)
    on = expert >= 0
    pick = torch.where(on, score.gather(1, expert.clamp(min=0)), 0.0)
    weight = pick
    if case["normalize"]:
        total = pick.sum(1, keepdim=True)
        weight = pick / torch.where(total > 0, total, 1.0)
    weight = case["scale"] * weight
    if not case["train"]:
        return expert, weight
    grad, = torch.autograd.grad(weight, l, s["g_weight"].double())
    return expert, weight.detach(), torch.where(masked, 0.0, grad)


def _exact_ring(case, s):
    cap, group, F = case["capacity"], case["group"], case["width"]
    mask = torch.logical_and(torch.lt(s["score"], s["thres"]), s["slot"] < 0)
    count = int(mask.sum())
    start = int(s["header"])
    rank = torch.cumsum(mask.to(torch.int64), 0) - 1
    slot_of_row = torch.where(mask, (start + rank) % cap, -1)
    full2slot, slot2full, checkin = (s[k].clone() for k in ("full2slot", "slot2full", "checkin"))
    taken = torch.zeros(cap, dtype=torch.bool, device=DEV)
    taken[slot_of_row[mask]] = True
    # nodes whose slot is taken lose it, the admitted ones have theirs
    lost = (full2slot >= 0) & taken[full2slot.clamp(min=0)]
    full2slot[lost] = -1
    full2slot[s["ids"][mask]] = slot_of_row[mask]
    slot2full[slot_of_row[mask]] = s["ids"][mask]
    checkin[taken] = s["it"]
    table = torch.zeros(cap, F, dtype=torch.float64, device=DEV)
    x, where = s["emb"][mask], slot_of_row[mask]
    for lo in range(0, F, group):
        cols = slice(lo, min(lo + group, F))
        table[:, cols] = s["codes"][:, cols].double() * s["scale"][:, lo // group].double().unsqueeze(1)
        part = x[:, cols]
        most = part.abs().max(dim=1, keepdim=True).values
        fine = most >= SMALLEST
        # the codes are whole numbers by definition, and which ones goes by 32 bits: rint(x * (1 / m * 127))
        per_unit = torch.reciprocal(torch.where(fine, most, 1.0)) * 127
        code = torch.round(part * per_unit).double()
        table[where, cols] = torch.where(fine, code * (most.double() / 127), 0.0)
    slot = full2slot[s["lookup"]]
    stale = (slot >= 0) & (s["it"] + 1 - checkin[slot.clamp(min=0)] >= AGE_LIMIT)
    slot = torch.where(stale, -1, slot)
    rows = table[slot.clamp(min=0)]
    rows[slot < 0] = 0.0
    return mask, torch.tensor([(start + count) % cap], device=DEV), full2slot, slot2full, checkin, slot, rows


def _exact_values(code, exponent, bits):
    """By a table of all 256 codes, in units of the top binade's 2^0."""
    all_codes = torch.arange(256, dtype=torch.float64, device=DEV)
    field = all_codes % 128 if bits == 3 else all_codes
    power, mantissa = torch.floor(field / 2 ** bits), (field % 2 ** bits) / 2 ** bits
    unit = torch.where(power == 0, mantissa * 2.0 ** -14, (1 + mantissa) * torch.exp2(power - 15))
    if bits == 3:
        unit = torch.where(all_codes >= 128, -unit, unit)
    e = exponent.double().repeat_interleave(ADAM_GROUP)[:code.numel()]
    return torch.where(e == 0, 0.0, unit[code.view(-1).long()] * torch.exp2(e - 127))


def _nearest(x, bits):
    """The nearest values among those that codes of x's groups can stand for."""
    n = x.numel()
    groups = -(-n // ADAM_GROUP)
    x = torch.nn.functional.pad(x, (0, groups * ADAM_GROUP - n)).view(groups, ADAM_GROUP)
    most = x.abs().max(dim=1, keepdim=True).values
    # from here on upwards the largest magnitude is rounded up to the next power of two
    turn = 2 - 2.0 ** -(bits + 1)
    power = torch.floor(torch.log2(torch.where(most > 0, most, 1.0)))
    power = torch.where(most >= turn * torch.exp2(power), power + 1, power)
    codes = torch.arange(128 if bits == 3 else 256, dtype=torch.float64, device=DEV)
    value = torch.where(codes < 2 ** bits, codes * 2.0 ** (-14 - bits),
                        (1 + codes % 2 ** bits / 2 ** bits) * torch.exp2(torch.floor(codes / 2 ** bits) - 15))
    size, border = x.abs() * torch.exp2(-power), (value[1:] + value[:-1]) / 2
    at = torch.bucketize(size, border)
    # in the middle between two: the even code
    at += (size == border[at.clamp(max=border.numel() - 1)]) & (at % 2 == 1)
    if bits == 4:
        at = torch.where((at == 0) & (x > 0), 1, at)
    near = torch.sign(x) * value[at] * torch.exp2(power)
    return torch.where((most == 0) | (power < -126), 0.0, near).view(-1)[:n]


def _exact_adamw(case, s):
    steps, out = s["steps"].clone(), []
    steps[:, 0] += 1
    b1, b2 = ADAM["betas"]
    for t, count in zip(s["tensors"], steps[:, 0].tolist()):
        shape = t["p"].shape
        g = t["g"].double().flatten()
        p = (t["p"] if t["master"] is None else t["master"]).double().flatten()
        if case["bits"] == 8:
            m, r = _exact_values(t["m"], t["scale"][0], 3), _exact_values(t["v"], t["scale"][1], 4)
            v, old_m = r.square(), m
        else:
            m, v = t["m"].double().flatten(), t["v"].double().flatten()
        m, v = torch.lerp(g, m, b1), torch.lerp(g.square(), v, b2)
        unbiased_m, unbiased_v = m / (1 - b1 ** count), v / (1 - b2 ** count)
        p = p - ADAM["lr"] * (ADAM["weight_decay"] * p + unbiased_m / (unbiased_v.sqrt() + ADAM["eps"]))
        if case["bits"] == 8:
            # which code is nearest goes by the moment in 32 bits, each operation rounded: borders are hit often where gradients have
            # few bits themselves
            g, old = t["g"].float().flatten(), r.float()
            m = torch.add(old_m.float().mul(b1), g.mul(1 - b1)).double()
            v = torch.add(old.mul(old).mul(b2), g.mul(1 - b2).mul(g))
            m, v = _nearest(m, 3), _nearest(v.sqrt().double(), 4)
        out.append((p.view(shape), None if t["master"] is None else p.view(shape), m.view(shape), v.view(shape)))
    return steps, out


def exact(case, seed):
    s = prepare(case, seed)
    return {"route": _exact_route, "ring": _exact_ring, "adamw": _exact_adamw}[case["kind"]](case, s)
