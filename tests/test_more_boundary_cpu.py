"""The argument checks of routing by scores, the ring table in 8 bits and the AdamW step, where no kernel is launched."""
import ctypes

import numpy as np
import pytest
import torch

OK, EINVAL, EDTYPE, EWORKSPACE, EUNSUPPORTED = 0, 1, 2, 4, 5


@pytest.fixture(scope="module")
def lib():
    import hiscache_backend as be
    return be.load_library()


@pytest.fixture(scope="module")
def p():
    buf = np.zeros(1 << 10, np.int64)
    p = ctypes.c_void_p(buf.ctypes.data)
    p.keep = buf
    return p


def test_route_scores(lib, p):
    def call(logits=p, dtype=0, n=4, E=8, k=2, score=1, bias=p, G=4, top=2, normalize=1, scale=1.0, expert=p, weight=p, picked=p):
        return lib.hc_route_scores(logits, dtype, n, E, k, score, bias, G, top, normalize, scale, expert, weight, picked, None)
    for bad in (dict(n=-1), dict(E=0), dict(k=0), dict(k=9), dict(score=2), dict(score=-1), dict(G=0), dict(G=3), dict(top=0),
                dict(top=5), dict(k=5), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
                dict(logits=None), dict(expert=None), dict(weight=None)):
        assert call(**bad) == EINVAL, bad
    assert call(dtype=7) == EDTYPE and call(n=0, dtype=7) == EDTYPE
    assert call(E=1028, G=4) == EUNSUPPORTED and call(E=64, k=33, G=1, top=1) == EUNSUPPORTED
    assert call(E=130, G=65, top=65) == EUNSUPPORTED and call(n=1 << 40) == EUNSUPPORTED
    assert call(n=0, logits=None, expert=None, weight=None) == OK

    def grad(logits=p, dtype=0, n=4, E=8, k=2, score=1, normalize=1, scale=1.0, expert=p, picked=p, g=p, out=p):
        return lib.hc_route_scores_grad(logits, dtype, n, E, k, score, normalize, scale, expert, picked, g, out, None)
    for bad in (dict(n=-1), dict(k=9), dict(score=3), dict(scale=0.0), dict(picked=None), dict(score=0, normalize=0, logits=None),
                dict(expert=None), dict(g=None), dict(out=None)):
        assert grad(**bad) == EINVAL, bad
    assert grad(dtype=3) == EDTYPE and grad(E=1025) == EUNSUPPORTED and grad(n=1 << 40) == EUNSUPPORTED
    assert grad(n=0, expert=None, picked=None, g=None, out=None) == OK


def test_ring_in_8_bits(lib, p):
    def admit(score=p, emb=p, slot=p, ids=p, thres=p, mask=p, codes=p, scale=p, group=64, cap=8, f2s=p, s2f=p, header=p, M=4, F=64,
              ws=p, nbytes=8192, kind=0, cmp=0):
        return lib.hc_grad_check_packed(None, score, emb, slot, None, None, ids, thres, 0, kind, cmp, mask, None, None, codes, scale,
                                        group, cap, f2s, s2f, None, header, 0, None, M, F, ws, nbytes, None)
    for bad in (dict(M=-1), dict(F=0), dict(cap=0), dict(score=None), dict(emb=None), dict(slot=None), dict(ids=None),
                dict(thres=None), dict(mask=None), dict(codes=None), dict(scale=None), dict(f2s=None), dict(s2f=None),
                dict(header=None), dict(kind=5), dict(cmp=5)):
        assert admit(**bad) == EINVAL, bad
    assert admit(group=48) == EUNSUPPORTED and admit(F=1 << 30) == EUNSUPPORTED
    assert admit(ws=None) == EWORKSPACE and admit(nbytes=8) == EWORKSPACE
    assert admit(M=0, score=None, emb=None, scale=None) == OK

    def find(f2s=p, n_full=8, ids=p, codes=p, scale=p, group=64, cap=8, F=64, slots=p, rows=p, n=4):
        return lib.hc_ring_lookup_packed(f2s, n_full, ids, None, 0, None, None, 1, codes, scale, group, cap, F, slots, rows, n, None)
    for bad in (dict(n=-1), dict(n_full=-1), dict(cap=-1), dict(F=0), dict(f2s=None), dict(ids=None), dict(slots=None),
                dict(codes=None), dict(scale=None)):
        assert find(**bad) == EINVAL, bad
    assert find(group=16) == EUNSUPPORTED and find(F=1 << 30) == EUNSUPPORTED and find(n=1 << 50) == EUNSUPPORTED
    assert find(n=0, f2s=None, ids=None, slots=None) == OK


def test_adamw(lib, p):
    array = (ctypes.c_void_p * 2)(p.value, p.value)
    null = (ctypes.c_void_p * 2)(p.value, None)
    numel = lambda *n: (ctypes.c_int64 * 2)(*n)  # noqa: E731

    def step(count=2, param=array, grad=array, dtype=0, m=array, v=array, scale=None, master=None, steps=array, n=numel(4, 4), bits=32,
             lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, decay=0.0):
        return lib.hc_adamw_step(count, param, grad, dtype, m, v, scale, master, steps, n, bits, lr, None, b1, b2, eps, decay, None)
    for bad in (dict(count=-1), dict(bits=16), dict(b1=1.0), dict(b1=-0.1), dict(b2=1.0), dict(b2=float("nan")), dict(eps=-1.0),
                dict(param=None), dict(grad=null), dict(m=null), dict(v=None), dict(steps=null), dict(n=None), dict(n=numel(4, -1)),
                dict(bits=8), dict(scale=array), dict(bits=8, scale=null), dict(master=array), dict(dtype=1, master=null)):
        assert step(**bad) == EINVAL, bad
    assert step(dtype=5) == EDTYPE and step(n=numel(4, 1 << 62)) == EUNSUPPORTED
    assert step(count=0, param=None, n=None) == OK

    def read(count=2, m=array, v=array, scale=array, n=numel(4, 4), a=array, r=array, dtype=0):
        return lib.hc_adamw_moments(count, m, v, scale, n, a, r, dtype, None)
    for bad in (dict(count=-1), dict(m=None), dict(v=null), dict(scale=null), dict(a=null), dict(r=None), dict(n=numel(-1, 4))):
        assert read(**bad) == EINVAL, bad
    assert read(dtype=5) == EDTYPE and read(n=numel(4, 1 << 62)) == EUNSUPPORTED and read(count=0, m=None) == OK


def test_python_calls_refuse_the_host():
    import hiscache
    import hiscache_backend as be
    logits, bias = torch.zeros(3, 8), torch.zeros(8)
    with pytest.raises(RuntimeError, match="no CPU path"):
        be.route_rows(logits, 2, score="sigmoid", bias=bias)
    w = torch.zeros(4)
    with pytest.raises(RuntimeError, match="no CPU path"):
        be.adamw_step([w], [w.clone()], [be.adamw_state(w)])
    with pytest.raises(ValueError):
        be.adamw_step([w], [], [be.adamw_state(w)])
    with pytest.raises(ValueError):
        be.adamw_moments([be.adamw_state(w)])
    with pytest.raises(ValueError):
        be.adamw_state(w, 16)
    with pytest.raises(ValueError):
        be.adamw_state(w, 32, True)
    kept = be.PackedRows(torch.zeros(6, 64, dtype=torch.int8), torch.zeros(6, 1), 64, torch.float32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        be._packed_table(kept)
    with pytest.raises(ValueError):
        be._packed_table(be.PackedRows(torch.zeros(6, 64, dtype=torch.int8), torch.zeros(6, 2), 64, torch.float32))
    layer = hiscache.ExpertMLP(8, 16, 4, 2, balance=True, score="sigmoid")
    assert layer.balance_bias.dtype == torch.float32 and layer.half().balance_bias.dtype == torch.float32
    assert hiscache.ExpertMLP(8, 16, 4, 2).balance_bias is None
    layer.balance_step()                                     # nothing has been routed
    assert bool((layer.balance_bias == 0).all())


def test_states_fit_their_tensors():
    import hiscache_backend as be
    s = be.adamw_state(torch.zeros(5, 60, dtype=torch.bfloat16), 8, True)
    assert s.exp_avg.dtype == s.exp_avg_sq.dtype == s.scale.dtype == torch.uint8 and s.scale.shape == (2, 3)
    assert s.exp_avg.shape == (5, 60) and s.master.dtype == torch.float32 and s.step.tolist() == [0, 0]
    s = be.adamw_state(torch.zeros(0), 8)
    assert s.scale.shape == (2, 0)
    with pytest.raises(ValueError):
        be._check_adamw_state(s, torch.Size([1]), -1)


def test_the_example_s_options(tmp_path):
    import importlib.util
    import os
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "history-cache_amd", "example")
    spec = importlib.util.spec_from_file_location("hiscache_example_main", os.path.join(here, "main.py"))
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    config = ex.load_config(os.path.join(here, "config.yaml"), ["trainer.ring_dtype=int8", "trainer.state_bits=8"])
    options = ex.trainer_options(config)
    assert options["ring_dtype"] is torch.int8 and options["state_bits"] == 8
    with pytest.raises(ValueError):
        ex.trainer_options(ex.load_config(os.path.join(here, "config.yaml"), ["trainer.ring_dtype=int4"]))
