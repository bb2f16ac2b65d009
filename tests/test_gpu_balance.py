"""The bias that loads experts evenly, moved by the loads of the last pass: an eager one, or a recorded one that is replayed."""
import copy
import gc
import weakref

import numpy as np
import pytest
import torch

import hiscache
from hiscache.history_trainer import _balance

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def loads(layer, x):
    expert, _ = layer.route(x)
    return torch.bincount(expert.view(-1), minlength=layer.num_expert).float()


def moved(load, rate):
    return rate * torch.sign(load.mean() - load)


def test_loads_of_the_pass_that_was_replayed_last():
    """Two recordings of one layer, as for batches of two shapes: each replay is what the next step outside goes by."""
    torch.manual_seed(0)
    layer = hiscache.ExpertMLP(32, 32, 8, 2, score="sigmoid", balance=True, device=DEV).train()
    inputs = [torch.randn(n, 32, device=DEV) for n in (200, 77)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for x in inputs:
            layer(x).sum().backward()
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in inputs]
    for graph, x in zip(graphs, inputs):
        layer.zero_grad(set_to_none=True)
        with torch.cuda.graph(graph):
            layer(x).sum().backward()
    for i in (0, 1, 0, 0, 1, 0):
        graphs[i].replay()
        load, bias = loads(layer, inputs[i]), layer.balance_bias.clone()
        assert float(load.sum()) == 2 * inputs[i].shape[0]
        layer.balance_step(0.01)
        assert torch.equal(layer.balance_bias, bias + moved(load, 0.01))
        inputs[i].copy_(torch.randn_like(inputs[i]))
    # an eager pass comes next, an evaluation and a choice from outside do not count
    x = torch.randn(50, 32, device=DEV)
    layer(x).sum().backward()
    load = loads(layer, x)
    layer.eval()(inputs[0])
    layer.train()(inputs[1], expert=torch.zeros(77, dtype=torch.int64, device=DEV))
    bias = layer.balance_bias.clone()
    layer.balance_step(0.5)
    assert torch.equal(layer.balance_bias, bias + moved(load, 0.5))


def test_the_loads_go_where_the_layer_goes():
    torch.manual_seed(0)
    layer = hiscache.ExpertMLP(32, 32, 8, 2, balance=True, device=DEV).train()
    x = torch.randn(50, 32, device=DEV)
    layer(x)
    load = loads(layer, x)
    assert sorted(k for k in layer.state_dict() if "w_" not in k) == ["balance_bias", "router"]
    for other in (copy.deepcopy(layer), copy.deepcopy(layer).half(), copy.deepcopy(layer).cpu()):
        other.balance_step(0.25)
        assert other.balance_bias.dtype == torch.float32 and torch.equal(other.balance_bias.to(DEV), moved(load, 0.25))
    # a layer that is built without memory and then given some starts from zeros
    late = hiscache.ExpertMLP(32, 32, 8, 2, balance=True, device="meta").to_empty(device=DEV)
    late.reset_parameters()
    late.balance_step()
    assert not bool(late.balance_bias.any())
    late.train()(x)
    late.balance_step(1.0)
    assert bool(late.balance_bias.any())


def test_two_passes_before_one_backward():
    """The loads are a copy: a second pass leaves what the first one's backward pass goes by."""
    torch.manual_seed(0)
    layer = hiscache.ExpertMLP(32, 32, 8, 2, score="sigmoid", balance=True, device=DEV).train()
    x, y = torch.randn(60, 32, device=DEV), torch.randn(33, 32, device=DEV)
    layer(x).square().sum().backward()
    layer(y).square().sum().backward()
    want = [p.grad.clone() for p in layer.parameters()]
    layer.zero_grad(set_to_none=True)
    (layer(x).square().sum() + layer(y).square().sum()).backward()
    for p, g in zip(layer.parameters(), want):
        assert torch.allclose(p.grad, g, rtol=1e-5, atol=1e-6 * float(g.abs().max()))


class Net(torch.nn.Module):
    def __init__(self, config, table):
        super().__init__()
        C = config.dl.dataset.num_classes
        self.base = hiscache.get_model(config, table)
        self.experts = hiscache.ExpertMLP(C, 32, 8, 2, score="sigmoid", balance=True)
        self.fixed = hiscache.ExpertMLP(C, 32, 8, 2)

    @property
    def convs(self):
        return self.base.convs

    def forward(self, batch):
        h = self.base(batch)
        return (h + self.experts(h) + self.fixed(h)).log_softmax(1)


@pytest.mark.parametrize("recorded", (False, True))
def test_the_trainer_balances(tmp_path, recorded):
    """After every step, replayed ones too: each moves an expert's bias by the rate, or not where its load is the mean."""
    from test_gpu_trainer import dataset
    L = 3
    dataset(tmp_path, np.random.default_rng(9), Fin=32, C=4)
    cfg = hiscache.make_config(32, 4, 64, L, method="grad", rate=0.6, staleness_thres=5, device=DEV, path=str(tmp_path))

    def run(rate, epochs=2):
        torch.manual_seed(7)
        t = hiscache.HistoryTrainer(cfg, fanout=[4, 3, 2], batch_size=200, lr=1e-2, num_epochs=epochs, eval_begin=9, ring_rows=3000,
                                    recorded=recorded, model_factory=Net, balance_rate=rate)
        t.train()
        return t

    t = run(2.0 ** -10)
    moves = t.model.experts.balance_bias * 2 ** 10
    assert bool((moves == moves.round()).all()) and 0 < float(moves.abs().max()) <= t.glb_iter
    if recorded:
        assert t._step.replays > 10
    # a few rows beside the mean or not: what one step would do is seen from the last loads
    load = (t.model.experts._offset[1:] - t.model.experts._offset[:-1]).float()
    before = t.model.experts.balance_bias.clone()
    _balance(t.model, 2.0 ** -10)
    assert torch.equal(t.model.experts.balance_bias, before + moved(load, 2.0 ** -10))
    assert not bool(run(None, 1).model.experts.balance_bias.any())
    # a trainer that nobody holds is gone with its memory, without the collector's help
    gc.collect()
    gc.disable()
    try:
        gone = weakref.ref(t)
        del t
        assert gone() is None
    finally:
        gc.enable()
