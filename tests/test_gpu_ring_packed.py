"""A ring table in 8 bits: admission and lookup against the same calls on an fp32 table and ``pack_rows`` / ``unpack_rows``, the cache
around it, and a training run with everything that is held in 8 bits."""
import copy

import numpy as np
import pytest
import torch

import hiscache
import hiscache_backend as be

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def ring(gen, N, cap, F, group, filled=0.7):
    """A ring of nodes in its slots, in fp32 and in 8 bits, with maps of their own."""
    n = int(cap * filled)
    node = torch.randperm(N, generator=gen, device=DEV)[:n]
    slot = torch.randperm(cap, generator=gen, device=DEV)[:n]
    full2slot = torch.full((N,), -1, dtype=torch.int64, device=DEV)
    slot2full = torch.full((cap,), -1, dtype=torch.int64, device=DEV)
    full2slot[node], slot2full[slot] = slot, node
    maps = dict(full2slot=full2slot, slot2full=slot2full, header=torch.tensor([cap - 1 - cap // 5], device=DEV),
                checkin=torch.randint(0, 20, (cap,), generator=gen, device=DEV))
    rows = torch.randn(cap, F, generator=gen, device=DEV)
    kept = be.pack_rows(rows, group)
    return be.unpack_rows(kept), kept, maps, {k: v.clone() for k, v in maps.items()}


def same(a, b):
    return all(torch.equal(a[k], b[k]) for k in a)


def admit(table, maps, emb, score, slot, ids, thres, it, **how):
    return be.grad_check(None, emb, slot, ids, thres, table, maps["full2slot"], maps["slot2full"], maps["header"], it,
                         checkin=maps["checkin"], score=score, **how)


SHAPES = [(1, 1, 40, 32), (5, 7, 40, 64), (64, 31, 300, 32), (63, 47, 300, 128), (65, 64, 90, 64), (700, 128, 800, 128),
          (1000, 172, 2000, 32), (3000, 256, 5000, 64), (300, 602, 400, 64), (130, 1024, 200, 128), (90, 2000, 100, 64),
          (500, 64, 5, 64), (400, 100, 63, 32), (4000, 36, 900, 32), (70_000, 40, 100_000, 64), (140_001, 16, 30_000, 32)]


@pytest.mark.parametrize("M,F,cap,group", SHAPES)
def test_admission_and_lookup(M, F, cap, group):
    gen = torch.Generator(device=DEV).manual_seed(M + F)
    N = 3 * max(M, cap)
    plain, kept, maps, maps8 = ring(gen, N, cap, F, group)
    for turn in range(3):
        ids = torch.randperm(N, generator=gen, device=DEV)[:M]
        slot = maps["full2slot"][ids].contiguous()
        emb = torch.randn(M, F, generator=gen, device=DEV) * torch.exp(torch.randn(M, 1, generator=gen, device=DEV))
        score = torch.rand(M, generator=gen, device=DEV)
        thres = torch.tensor([(0.3, 1.0, 0.0)[turn]], device=DEV)
        used = torch.rand(M, generator=gen, device=DEV) < 0.8
        age = torch.randint(0, 30, (M,), generator=gen, device=DEV, dtype=torch.int32)
        how = dict(used=used, age=age, age_limit=20, want_slots=True) if turn == 1 else dict(want_slots=True)
        if turn == 2:
            thres = torch.tensor([0.5], device=DEV)
            it = torch.tensor([7 + turn], device=DEV)        # the iteration's number on the device
        else:
            it = 7 + turn
        beside = kept.codes.clone(), kept.scale.clone()
        got, want = admit(kept, maps8, emb, score, slot, ids, thres, it, **how), admit(plain, maps, emb, score, slot, ids, thres, it, **how)
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and same(maps, maps8)
        # the slots that were written hold their last row's codes, the others what they held
        at, row = got[2][got[0]], torch.nonzero(got[0]).view(-1)
        at, row = at[-cap:], row[-cap:]
        packed = be.pack_rows(emb, group)
        beside[0][at], beside[1][at] = packed.codes[row], packed.scale[row]
        assert torch.equal(kept.codes, beside[0]) and torch.equal(kept.scale, beside[1])
        find = torch.cat([ids, torch.randint(0, N, (50,), generator=gen, device=DEV), torch.tensor([-1, N, 5, 5], device=DEV)])
        for now, limit in ((9, 1 << 62), (12, 4)):
            slots, rows = be.ring_lookup(maps8["full2slot"], find, kept, checkin=maps8["checkin"], now=now, age_limit=limit)
            want_slots, _ = be.ring_lookup(maps["full2slot"], find, plain, checkin=maps["checkin"], now=now, age_limit=limit)
            assert torch.equal(slots, want_slots)
            whole = be.unpack_rows(kept)
            assert torch.equal(rows, torch.where((slots >= 0).unsqueeze(1), whole[slots.clamp(min=0)], 0.0))
            assert be.ring_lookup(maps8["full2slot"], find, kept, now=now, want_rows=False)[1] is None
        n_valid, now = torch.tensor([min(3, M)], device=DEV), torch.tensor([12], device=DEV)
        slots, rows = be.ring_lookup(maps8["full2slot"], ids, kept, checkin=maps8["checkin"], now=now, age_limit=4, n_valid=n_valid)
        assert torch.equal(slots[:3], be.ring_lookup(maps8["full2slot"], ids[:3], kept, checkin=maps8["checkin"], now=12, age_limit=4)[0])
        assert bool((slots[3:] == -1).all()) and bool((rows[3:] == 0).all())
        # (the fp32 table goes on with what the other holds)
        plain = be.unpack_rows(kept)


def test_scores_from_gradients():
    gen = torch.Generator(device=DEV).manual_seed(1)
    plain, kept, maps, maps8 = ring(gen, 4000, 900, 256, 64)
    ids = torch.randperm(4000, generator=gen, device=DEV)[:1500]
    slot = maps["full2slot"][ids].contiguous()
    emb, grad = torch.randn(1500, 256, generator=gen, device=DEV), torch.randn(1500, 256, generator=gen, device=DEV)
    thres = torch.tensor([16.0], device=DEV)
    a = be.grad_check(grad, emb, slot, ids, thres, kept, maps8["full2slot"], maps8["slot2full"], maps8["header"], 3)
    b = be.grad_check(grad, emb, slot, ids, thres, plain, maps["full2slot"], maps["slot2full"], maps["header"], 3)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and 0 < int(a[0].sum()) < 1500 and same(maps, maps8)


def test_rows_that_are_no_numbers_or_very_small_or_zeros():
    gen = torch.Generator(device=DEV).manual_seed(2)
    for F in (96, 100):
        emb = torch.randn(6, F, generator=gen, device=DEV)
        emb[0, 40], emb[1, 70], emb[2] = float("nan"), float("inf"), 0.0
        emb[3] *= 2.0 ** -126
        emb[4] = torch.finfo(torch.float32).max
        kept = be.pack_rows(torch.ones(10, F, device=DEV), 32)
        maps = dict(full2slot=torch.full((6,), -1, device=DEV), slot2full=torch.full((10,), -1, device=DEV),
                    header=torch.tensor([8], device=DEV), checkin=torch.full((10,), -1, device=DEV))
        ids = torch.arange(6, device=DEV)
        admit(kept, maps, emb, torch.zeros(6, device=DEV), torch.full((6,), -1, device=DEV), ids, torch.ones(1, device=DEV), 1)
        slots, rows = be.ring_lookup(maps["full2slot"], ids, kept)
        assert slots.tolist() == [8, 9, 0, 1, 2, 3]
        want = be.unpack_rows(be.pack_rows(emb, 32))
        assert torch.equal(torch.isnan(rows), torch.isnan(want)) and torch.equal(torch.nan_to_num(rows), torch.nan_to_num(want))
        assert bool(torch.isnan(rows[0, 32:64]).all()) and bool((rows[2:4] == 0).all()) and bool(torch.isfinite(rows[4]).all())


def test_large_offsets():
    """A table of more than 2^32 codes: rows at its end are written and found."""
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GiB of free device memory")
    F, cap = 1024, (1 << 32) // 1024 + 2000
    kept = be.PackedRows(torch.zeros(cap, F, dtype=torch.int8, device=DEV), torch.zeros(cap, F // 128, device=DEV), 128, torch.float32)
    maps = dict(full2slot=torch.full((cap,), -1, device=DEV), slot2full=torch.full((cap,), -1, device=DEV),
                header=torch.tensor([cap - 100], device=DEV), checkin=torch.full((cap,), -1, device=DEV))
    gen = torch.Generator(device=DEV).manual_seed(3)
    emb, ids = torch.randn(200, F, generator=gen, device=DEV), torch.arange(cap - 200, cap, device=DEV)
    admit(kept, maps, emb, torch.zeros(200, device=DEV), torch.full((200,), -1, device=DEV), ids, torch.ones(1, device=DEV), 1)
    slots, rows = be.ring_lookup(maps["full2slot"], ids, kept)
    assert slots.tolist() == list(range(cap - 100, cap)) + list(range(100))
    assert torch.equal(rows, be.unpack_rows(be.pack_rows(emb, 128)))
    assert int((kept.scale != 0).any(1).sum()) == 200


def test_views_and_other_streams():
    gen = torch.Generator(device=DEV).manual_seed(4)
    for F in (64, 172):
        plain, kept, maps, maps8 = ring(gen, 2000, 500, F, 64)
        # codes and rows off every alignment
        flat = torch.zeros(500 * F + 3, dtype=torch.int8, device=DEV)
        codes = flat[3:].view(500, F)
        codes.copy_(kept.codes)
        table = be.PackedRows(codes, kept.scale, 64, torch.float32)
        ids = torch.randperm(2000, generator=gen, device=DEV)[:300]
        emb = torch.randn(300 * F + 1, generator=gen, device=DEV)[1:].view(300, F)
        slot = maps["full2slot"][ids].contiguous()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            admit(table, maps8, emb, torch.zeros(300, device=DEV), slot, ids, torch.ones(1, device=DEV), 4)
            slots, rows = be.ring_lookup(maps8["full2slot"], ids, table)
        side.synchronize()
        admit(kept, maps, emb, torch.zeros(300, device=DEV), slot, ids, torch.ones(1, device=DEV), 4)
        assert torch.equal(codes, kept.codes) and same(maps, maps8) and bool((flat[:3] == 0).all())
        # (a node whose slot another has taken over is found no more)
        assert torch.equal(rows, torch.where((slots >= 0).unsqueeze(1), be.unpack_rows(kept)[slots.clamp(min=0)], 0.0))


def test_refusals():
    gen = torch.Generator(device=DEV).manual_seed(5)
    plain, kept, maps, _ = ring(gen, 100, 50, 64, 64)
    emb, ids = torch.zeros(4, 64, device=DEV), torch.arange(4, device=DEV)
    args = emb, torch.zeros(4, device=DEV), torch.full((4,), -1, device=DEV), ids, torch.ones(1, device=DEV), 1
    halves = be.gated_pack(torch.randn(50, 128, generator=gen, device=DEV))[1]
    for bad in (halves, be.PackedRows(kept.codes[:, :32].contiguous(), kept.scale, 64, torch.float32),
                be.PackedRows(kept.codes, kept.scale[:40], 64, torch.float32), be.PackedRows(kept.codes, kept.scale, 48, torch.float32)):
        with pytest.raises(ValueError):
            admit(bad, maps, *args)
    with pytest.raises((RuntimeError, ValueError)):
        admit(be.PackedRows(kept.codes.cpu(), kept.scale.cpu(), 64, torch.float32), maps, *args)
    with pytest.raises(ValueError):
        admit(kept, maps, *args, static_scratch=True)
    with pytest.raises(ValueError):
        admit(kept, dict(maps, checkin=maps["checkin"][:10]), *args)
    with pytest.raises(ValueError):
        admit(kept, dict(maps, slot2full=maps["slot2full"][:10]), *args)
    with pytest.raises(ValueError):
        be.ring_lookup(maps["full2slot"], ids, kept, checkin=maps["checkin"][:10])
    with pytest.raises(ValueError):
        be.ring_lookup(maps["full2slot"], ids, kept, n_valid=torch.tensor([1], device=DEV))
    # (halves of whole groups are rows of twice the width, and nothing tells them from such)
    assert be.ring_lookup(maps["full2slot"], ids, halves)[1].shape == (4, 128)
    with pytest.raises(ValueError):
        hiscache.RingHistoryCache(None, 100, 8, 64, 50, 2, table_dtype=torch.int8, group=48, device=DEV)


# ----------------------------------------------------------------------------- the cache
def cache_of(dtype, cap=400, group=64):
    return hiscache.RingHistoryCache(None, 1000, 16, 64, cap, 2, table_dtype=dtype, device=DEV, group=group)


def test_a_cache_s_checkpoint_and_warm_start():
    gen = torch.Generator(device=DEV).manual_seed(6)
    a, b = cache_of(torch.int8), cache_of(torch.int8)
    nodes, rows = torch.randperm(1000, generator=gen, device=DEV)[:300], torch.randn(300, 64, generator=gen, device=DEV)
    a.preload(nodes, rows.half())
    want = be.unpack_rows(be.pack_rows(rows.half().float(), 64))
    slots, got = be.ring_lookup(a.full2slot, nodes, a.table)
    assert slots.tolist() == list(range(300)) and torch.equal(got, want)
    state = copy.deepcopy(a.state_dict())
    b.load_state_dict(state)
    assert torch.equal(b.table.codes, a.table.codes) and torch.equal(b.table.scale, a.table.scale) and b.header == a.header == 300
    for other in (cache_of(torch.float16), cache_of(torch.int8, 500), cache_of(torch.int8, group=32)):
        with pytest.raises(ValueError):
            other.load_state_dict(state)
    with pytest.raises(ValueError):
        b.load_state_dict(cache_of(torch.float16).state_dict())
    fresh = cache_of(torch.int8)
    fresh.preload(nodes)                                     # marked as cached; the rows are zeros
    assert bool((be.ring_lookup(fresh.full2slot, nodes, fresh.table)[1] == 0).all())


# ----------------------------------------------------------------------------- together
class Net(torch.nn.Module):
    """A history model and a layer of experts, evenly loaded by a bias, on what it gives out."""

    def __init__(self, config, table):
        super().__init__()
        C = config.dl.dataset.num_classes
        self.base = hiscache.get_model(config, table)
        self.experts = hiscache.ExpertMLP(C, 32, 8, 2, score="sigmoid", num_group=4, top_group=2, scale=1.5, balance=True)

    @property
    def convs(self):
        return self.base.convs

    def forward(self, batch):
        h = self.base(batch)
        out = (h + self.experts(h)).log_softmax(1)
        if self.training:
            self.experts.balance_step(1e-3)
        return out


@pytest.mark.parametrize("recorded", (False, True))
def test_a_run_with_all_of_them(tmp_path, recorded):
    """Embeddings in a ring of 8 bits, AdamW with moments in 8 bits, balanced experts; enqueued step by step, and recorded and replayed."""
    from test_gpu_trainer import dataset
    rng = np.random.default_rng(9)
    Fin, H, C, L = 32, 64, 4, 3
    dataset(tmp_path, rng, Fin=Fin, C=C)
    cfg = hiscache.make_config(Fin, C, H, L, method="grad", rate=0.6, staleness_thres=5, device=DEV, path=str(tmp_path))

    def run(state=None, epochs=2):
        torch.manual_seed(7)
        t = hiscache.HistoryTrainer(cfg, fanout=[4, 3, 2], batch_size=200, lr=1e-2, num_epochs=epochs, eval_begin=0, ring_rows=3000,
                                    ring_dtype=torch.int8, state_bits=8, recorded=recorded, model_factory=Net)
        if state is not None:
            t.load_state_dict(state)
        t.train()
        return t

    a, b = run(), run()
    assert isinstance(a.optimizer, hiscache.AdamW) and a.table.table.codes.dtype == torch.int8 and a.table.header > 0
    assert int((a.table.table.scale != 0).any(1).sum()) > 500              # rows were admitted
    assert any("scale" in s for s in a.optimizer.state.values())
    if recorded:
        assert a._step.replays > 10
    assert bool((a.model.experts.balance_bias != 0).any())
    for p, q in zip(a.model.parameters(), b.model.parameters()):
        assert torch.equal(p, q) and bool(torch.isfinite(p).all())          # the same numbers every time
    assert torch.equal(a.table.table.codes, b.table.table.codes)
    resumed = run(copy.deepcopy(a.state_dict()), epochs=1)
    assert resumed.glb_iter == 3 * a.glb_iter // 2 and all(bool(torch.isfinite(p).all()) for p in resumed.model.parameters())
