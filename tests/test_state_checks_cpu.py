"""What a call looks at of the tensors behind its handles: those that they hold now, not those that an earlier call saw."""
import pytest
import torch

import hiscache_backend as be


class OnDevice:
    """A tensor of the host that says it lies on a GPU."""
    is_cuda = True
    index = 0

    def __init__(self, t):
        self.t = t

    def __getattr__(self, name):
        return getattr(self.t, name)

    def get_device(self):
        return self.index


def state(shape, bits=32, master=False):
    made = be.adamw_state(torch.zeros(shape, dtype=torch.bfloat16 if master else torch.float32), bits, master)
    parts = [getattr(made, k) for k in ("exp_avg", "exp_avg_sq", "step", "scale", "master")]
    return be.AdamWState(*[None if t is None else OnDevice(t) for t in parts])


CHANGES = {
    "smaller": lambda t: t[:1].clone(), "narrower": lambda t: t.to(torch.int16), "of another type": lambda t: t.to(torch.int32),
    "expanded": lambda t: t.new_zeros(1).expand(t.shape), "in steps": lambda t: t.new_zeros(*t.shape[:-1], 2 * t.shape[-1])[..., ::2],
    "reshaped": lambda t: t.new_zeros(t.numel() + 1),
}


@pytest.mark.parametrize("part", ("exp_avg", "exp_avg_sq", "step", "scale", "master"))
@pytest.mark.parametrize("change", sorted(CHANGES))
def test_a_state_that_changed_behind_its_object_is_looked_at_again(part, change):
    shape = torch.Size([256])
    s = state(shape, 8, True)
    at = be._check_adamw_state(s, shape, 0)
    assert be._check_adamw_state(s, shape, 0) == at and at[0] == s.exp_avg.data_ptr()
    t = getattr(s, part)
    t.t.data = CHANGES[change](t.t)
    with pytest.raises(ValueError):
        be._check_adamw_state(s, shape, 0)


def test_a_state_elsewhere_or_without_memory():
    shape = torch.Size([64])
    s = state(shape)
    at = be._check_adamw_state(s, shape, 0)
    new = torch.ones(64)
    s.exp_avg.t.data = new                                   # the same kind at another place: its address is taken
    assert be._check_adamw_state(s, shape, 0) == (new.data_ptr(), *at[1:])
    s.exp_avg.t.data, s.exp_avg.index = torch.ones(64), -1   # (a device's address is no host's)
    with pytest.raises(ValueError):
        be._check_adamw_state(s, shape, 0)
    s = state(shape)
    be._check_adamw_state(s, shape, 0)
    s.exp_avg_sq.t.untyped_storage().resize_(0)
    with pytest.raises(ValueError):
        be._check_adamw_state(s, shape, 0)
    s = state(shape)
    be._check_adamw_state(s, shape, 0)
    s.exp_avg.t.resize_(32)
    with pytest.raises(ValueError):
        be._check_adamw_state(s, shape, 0)
    with pytest.raises(ValueError):
        be._check_adamw_state(state(shape), shape, 1)


@pytest.mark.parametrize("part", ("codes", "scale"))
@pytest.mark.parametrize("change", sorted(CHANGES))
def test_packed_rows_that_changed_behind_their_object_are_looked_at_again(part, change):
    kept = be.PackedRows(torch.zeros(6, 64, dtype=torch.int8), torch.zeros(6, 2), 32, torch.float32)
    assert be._check_kept(kept, 1) == be._check_kept(kept, 1) == (6, 64)
    t = getattr(kept, part)
    t.data = CHANGES[change](t)
    with pytest.raises(ValueError):
        be._check_kept(kept, 1)
    kept = be.PackedRows(torch.zeros(6, 64, dtype=torch.int8), torch.zeros(6, 2), 32, torch.float32)
    be._check_kept(kept, 1)
    getattr(kept, part).untyped_storage().resize_(0)
    with pytest.raises(ValueError):
        be._check_kept(kept, 1)


@pytest.mark.parametrize("part", ("slot", "offset"))
@pytest.mark.parametrize("change", sorted(CHANGES))
def test_an_order_that_changed_behind_its_object_is_looked_at_again(part, change):
    def make():
        return be.ExpertOrder(torch.zeros(12, dtype=torch.int32), torch.zeros(12, dtype=torch.int32), torch.zeros(5, dtype=torch.int64),
                              6, 2, 4)
    order = make()
    assert be._places(order)[2:] == be._places(order)[2:] == (6, 2, 4)
    t = getattr(order, part)
    t.data = t.to(torch.int16) if change == "of another type" else CHANGES[change](t)
    with pytest.raises(ValueError):
        be._places(order)
    order = make()
    be._places(order)
    getattr(order, part).untyped_storage().resize_(0)
    with pytest.raises(ValueError):
        be._places(order)


@pytest.mark.parametrize("part", (0, 1))
def test_an_order_that_changed_between_forward_and_backward_is_noticed(part):
    class Node:
        pass
    node, places = Node(), (torch.zeros(12, dtype=torch.int32), torch.zeros(5, dtype=torch.int64), 6, 2, 4)
    be._keep_places(node, places)
    assert be._kept_places(node) == places
    places[part].data = places[part][:1].clone()
    with pytest.raises(RuntimeError, match="modified"):
        be._kept_places(node)


def test_parts_of_states_that_two_parameters_would_share():
    a, b = (0x1000, 0x2000, 0x3000, 0, 0, 8), (0x4000, 0x5000, 0x6000, 0x7000, 0x8000, 8)
    be._written_once([0x9000, 0xA000], [a, b])
    be._written_once([0, 0], [(0, 0, 0x3000, 0, 0, 0), (0, 0, 0x6000, 0, 0, 0)])           # empty tensors lie nowhere
    for i in range(5):
        shared = list(b)
        shared[i] = 0x3000
        with pytest.raises(ValueError, match="one parameter"):
            be._written_once([0x9000, 0xA000], [a, tuple(shared)])
    with pytest.raises(ValueError, match="one parameter"):
        be._written_once([0x9000], [(0x1000, 0x1000, 0x3000, 0, 0, 8)])
    with pytest.raises(ValueError, match="part of a state"):
        be._written_once([0x9000, 0x8000], [a, b])


def test_a_ring_table_on_the_host_is_refused_every_time():
    table = be.PackedRows(torch.zeros(6, 64, dtype=torch.int8), torch.zeros(6, 1), 64, torch.float32)
    for _ in range(3):
        with pytest.raises(RuntimeError, match="no CPU path"):
            be._packed_table(table)
    be._check_kept(table, 1)                                 # (rows that another call has looked at)
    device = be.PackedRows(OnDevice(table.codes), OnDevice(table.scale), 64, torch.float32)
    assert be._packed_table(device) == be._packed_table(device) == (6, 64)
    device.codes.t.data = torch.zeros(7, 64, dtype=torch.int8)
    with pytest.raises(ValueError):
        be._packed_table(device)
