"""Lookups in a ring table of 8 bits of more ids than one launch takes."""
import pytest
import torch

import hiscache_backend as be

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("F,group", ((4, 32), (3, 32)))
def test_more_ids_than_a_launch_takes(F, group):
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GiB of free device memory")
    n, nodes, capacity = (1 << 28) + 1003, 50_000, 20_000
    gen = torch.Generator(device=DEV).manual_seed(1)
    table = be.PackedRows(torch.randint(-127, 128, (capacity, F), generator=gen, device=DEV, dtype=torch.int8),
                          torch.rand(capacity, 1, generator=gen, device=DEV), group, torch.float32)
    full2slot = torch.full((nodes,), -1, dtype=torch.int64, device=DEV)
    full2slot[torch.randperm(nodes, generator=gen, device=DEV)[:capacity]] = torch.arange(capacity, device=DEV)
    ids = torch.randint(-3, nodes + 3, (n,), generator=gen, device=DEV)
    slot, rows = be.ring_lookup(full2slot, ids, table)
    edge = (((1 << 32) - 1) // 256) * 16                     # the first id of the second launch
    whole = table.codes.float() * table.scale
    for part in (slice(0, 5000), slice(edge - 5000, edge + 5000), slice(n - 5000, n)):
        i = ids[part]
        want = torch.where((i >= 0) & (i < nodes), full2slot[i.clamp(0, nodes - 1)], -1)
        assert torch.equal(slot[part], want)
        assert torch.equal(rows[part], torch.where((want >= 0).unsqueeze(1), whole[want.clamp(min=0)], 0.0))
    del rows
    valid, now = torch.tensor([edge + 7], device=DEV), torch.tensor([5], device=DEV)
    only = be.ring_lookup(full2slot, ids, table, now=now, n_valid=valid, want_rows=False)[0]
    assert torch.equal(only[:edge + 7], slot[:edge + 7]) and bool((only[edge + 7:] == -1).all())
