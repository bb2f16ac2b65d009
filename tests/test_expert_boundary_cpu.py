"""The argument checks of the expert layer's entry points and of the Python calls in front of them (no kernel is launched here)."""
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


def test_route(lib, p):
    assert lib.hc_route_rows(p, 0, -1, 8, 2, 1, p, p, None) == EINVAL
    assert lib.hc_route_rows(p, 0, 4, 0, 1, 1, p, p, None) == EINVAL
    assert lib.hc_route_rows(p, 0, 4, 8, 9, 1, p, p, None) == EINVAL
    assert lib.hc_route_rows(p, 0, 4, 8, 0, 1, p, p, None) == EINVAL
    assert lib.hc_route_rows(p, 0, 4, 1025, 2, 1, p, p, None) == EUNSUPPORTED
    assert lib.hc_route_rows(p, 0, 4, 64, 33, 1, p, p, None) == EUNSUPPORTED
    assert lib.hc_route_rows(p, 7, 4, 8, 2, 1, p, p, None) == EDTYPE
    assert lib.hc_route_rows(None, 0, 4, 8, 2, 1, p, p, None) == EINVAL
    assert lib.hc_route_rows(p, 0, 1 << 40, 8, 2, 1, p, p, None) == EUNSUPPORTED
    assert lib.hc_route_rows(None, 0, 0, 8, 2, 1, None, None, None) == OK
    assert lib.hc_route_rows(None, 9, 0, 8, 2, 1, None, None, None) == EDTYPE
    assert lib.hc_route_rows_grad(None, 0, 4, 8, 2, 0, p, p, p, p, None) == EINVAL          # logits are needed unless normalised
    assert lib.hc_route_rows_grad(p, 0, 4, 8, 2, 1, p, p, None, p, None) == EINVAL
    assert lib.hc_route_rows_grad(p, 3, 4, 8, 2, 1, p, p, p, p, None) == EDTYPE
    assert lib.hc_route_rows_grad(None, 0, 0, 8, 2, 1, None, None, None, None, None) == OK


def test_order(lib, p):
    assert lib.hc_expert_order(p, -1, 4, p, p, p, None, 0, None) == EINVAL
    assert lib.hc_expert_order(p, 8, 0, p, p, p, None, 0, None) == EINVAL
    assert lib.hc_expert_order(None, 8, 4, p, p, p, None, 0, None) == EINVAL
    assert lib.hc_expert_order(p, 8, 4, p, p, None, None, 0, None) == EINVAL
    assert lib.hc_expert_order(p, 8, 1025, p, p, p, None, 0, None) == EUNSUPPORTED
    assert lib.hc_expert_order(p, 1 << 31, 4, p, p, p, None, 0, None) == EUNSUPPORTED
    assert lib.hc_expert_order_workspace_bytes(8192, 1024) == 0 and lib.hc_expert_order_workspace_bytes(-1, 4) == 0
    need = lib.hc_expert_order_workspace_bytes(1_000_000, 64)
    assert need >= 65 * 4 * (1_000_000 // 1024) and lib.hc_expert_order_workspace_bytes((1 << 31) - 1, 1024) < 32 << 20
    assert lib.hc_expert_order(p, 1_000_000, 64, p, p, p, None, 0, None) == EWORKSPACE
    assert lib.hc_expert_order(p, 1_000_000, 64, p, p, p, p, need - 1, None) == EWORKSPACE


def test_rows(lib, p):
    for call in (lambda **k: lib.hc_rows_to_experts(k["x"], k["dt"], k["n"], k["k"], k["E"], k["D"], p, k["off"], p, None),
                 lambda **k: lib.hc_rows_from_experts_grad(p, k["x"], k["dt"], k["n"], k["k"], k["E"], k["D"], p, k["off"], p, p, p, None)):
        good = dict(x=p, dt=0, n=4, k=2, E=3, D=8, off=p)
        for bad, code in ((dict(n=-1), EINVAL), (dict(k=0), EINVAL), (dict(E=0), EINVAL), (dict(D=0), EINVAL), (dict(x=None), EINVAL),
                          (dict(off=None), EINVAL), (dict(dt=5), EDTYPE), (dict(n=1 << 31), EUNSUPPORTED), (dict(E=2000), EUNSUPPORTED),
                          (dict(D=1 << 30), EUNSUPPORTED)):
            assert call(**{**good, **bad}) == code, bad
        assert call(**{**good, "n": 0, "x": None, "off": None}) == OK
    assert lib.hc_rows_from_experts(None, 0, 4, 2, 3, 8, p, None, p, None) == EINVAL
    assert lib.hc_rows_from_experts(p, 4, 4, 2, 3, 8, p, None, p, None) == EDTYPE
    assert lib.hc_rows_from_experts(None, 1, 0, 2, 3, 8, None, None, None, None) == OK


def test_products(lib, p):
    assert lib.hc_expert_linear(p, 0, p, 0, p, -1, 2, 4, 4, p, None) == EINVAL
    assert lib.hc_expert_linear(p, 0, p, 0, p, 4, 0, 4, 4, p, None) == EINVAL
    assert lib.hc_expert_linear(p, 0, p, 0, None, 4, 2, 4, 4, p, None) == EINVAL
    assert lib.hc_expert_linear(p, 3, p, 0, p, 4, 2, 4, 4, p, None) == EDTYPE
    assert lib.hc_expert_linear(p, 0, p, 0, p, 4, 1025, 4, 4, p, None) == EUNSUPPORTED
    assert lib.hc_expert_linear(p, 0, p, 0, p, 4, 2, (1 << 20) + 1, 4, p, None) == EUNSUPPORTED
    assert lib.hc_expert_linear(p, 0, p, 0, p, 4, 2, 1 << 20, 1 << 20, p, None) == EUNSUPPORTED
    assert lib.hc_expert_linear(p, 0, p, 0, p, (1 << 31) - 1, 2, 4, 4, p, None) == EUNSUPPORTED
    assert lib.hc_expert_linear(None, 0, None, 0, None, 0, 2, 4, 4, None, None) == OK
    need = lib.hc_expert_linear_grad_workspace_bytes(60_000, 5, 256, 256, 0)
    assert need > 0 and lib.hc_expert_linear_grad_workspace_bytes(100, 5, 256, 256, 0) == 0
    assert lib.hc_expert_linear_grad_workspace_bytes(60_000, 5, 256, 256, 9) == 0
    assert lib.hc_expert_linear_grad(p, p, 0, p, 60_000, 5, 256, 256, p, None, 0, None) == EWORKSPACE
    assert lib.hc_expert_linear_grad(p, p, 0, p, 60_000, 5, 256, 256, p, p, need - 1, None) == EWORKSPACE
    assert lib.hc_expert_linear_grad(p, None, 0, p, 4, 5, 4, 4, p, None, 0, None) == EINVAL
    assert lib.hc_expert_linear_grad(p, p, 8, p, 4, 5, 4, 4, p, None, 0, None) == EDTYPE


def test_the_parts_of_a_gradient_fit_the_workspace(lib):
    # experts of p > 1 parts hold fewer parts than twice the rows over a part's rows
    for S in (513, 4096, 100_000, 5_000_000):
        for N, K in ((64, 64), (300, 172), (2048, 1024)):
            for dtype in (0, 1, 2):
                need = lib.hc_expert_linear_grad_workspace_bytes(S, 16, N, K, dtype)
                least = 128 if dtype == 0 else 512                # rows of the shortest part that is not an expert's last
                assert need % (N * K * 4) == 0 and need // (N * K * 4) <= 2 * (S // least)


def test_packed(lib, p):
    assert lib.hc_pack_rows(p, 0, -1, 8, 64, p, p, None) == EINVAL
    assert lib.hc_pack_rows(p, 0, 4, 0, 64, p, p, None) == EINVAL
    assert lib.hc_pack_rows(p, 0, 4, 8, 48, p, p, None) == EUNSUPPORTED
    assert lib.hc_pack_rows(p, 0, 1 << 40, 64, 64, p, p, None) == EUNSUPPORTED
    assert lib.hc_pack_rows(p, 6, 4, 8, 64, p, p, None) == EDTYPE
    assert lib.hc_pack_rows(None, 0, 4, 8, 64, p, p, None) == EINVAL
    assert lib.hc_unpack_rows(p, None, 4, 8, 64, p, 0, None) == EINVAL
    assert lib.hc_gated_pack(p, 0, 4, 8, 64, p, p, None, None) == EINVAL
    assert lib.hc_gated_grad(p, p, p, 0, 4, 8, 64, None, p, None) == EINVAL
    assert lib.hc_pack_rows(None, 0, 0, 8, 64, None, None, None) == OK
    assert lib.hc_gated_grad(None, None, None, 2, 0, 8, 32, None, None, None) == OK


def test_the_module_checks_its_arguments_without_a_gpu():
    import hiscache
    import hiscache_backend as be
    layer = hiscache.ExpertMLP(8, 16, 4, 2)
    assert {k: tuple(v.shape) for k, v in layer.state_dict().items()} == {"router": (4, 8), "w_in": (4, 32, 8), "w_out": (4, 8, 16)}
    assert "num_expert=4" in repr(layer)
    for bad in (0, 5):
        with pytest.raises(ValueError):
            hiscache.ExpertMLP(8, 16, 4, bad)
    with pytest.raises(RuntimeError):                              # there is no path on the CPU
        layer(torch.zeros(3, 8))
    with pytest.raises(RuntimeError):
        be.pack_rows(torch.zeros(3, 8))
    # tensors on the CPU pass through the hooks as they are
    with hiscache.packed_activations(min_elements=1):
        x = torch.randn(5, 6, requires_grad=True)
        y = (x * x).sum()
    y.backward()
    assert torch.equal(x.grad, 2 * x)


def test_an_order_that_does_not_fit_its_rows_is_refused():
    import hiscache_backend as be
    slot, offset = torch.zeros(12, dtype=torch.int32), torch.zeros(5, dtype=torch.int64)
    be._check_order(be.ExpertOrder(slot, slot, offset, 6, 2, 4))
    wide = torch.zeros(12, 2, dtype=torch.int32)
    for bad in ((slot[:11], offset, 6, 2, 4), (slot, offset, 7, 2, 4), (slot, offset, 6, 3, 4), (slot, offset[:4], 6, 2, 4),
                (slot, offset, 6, 2, 5), (slot.long(), offset, 6, 2, 4), (slot, offset.int(), 6, 2, 4), (wide[:, 0], offset, 6, 2, 4)):
        with pytest.raises(ValueError):
            be._check_order(be.ExpertOrder(bad[0], slot, *bad[1:]))
    with pytest.raises(TypeError):
        be._check_order(slot)


def test_kept_rows_that_are_not_whole_are_refused():
    import hiscache_backend as be
    codes, scale = torch.zeros(6, 200, dtype=torch.int8), torch.zeros(6, 4)
    assert be._check_kept(be.PackedRows(codes, scale, 64, torch.float16), 1) == (6, 200)
    assert be._check_kept(be.PackedRows(codes, scale, 64, torch.float16), 2) == (6, 100)
    assert be._check_kept(be.PackedRows(codes[:0], scale[:0], 64, torch.float16), 1) == (0, 200)
    for halves in (1, 2):
        for bad in ((codes, scale[:5], 64), (codes, scale[:, :3], 64), (codes, scale, 32), (codes, scale, 48), (codes, scale.view(-1), 64),
                    (codes.view(-1), scale, 64), (codes.int(), scale, 64), (codes, scale.double(), 64),
                    (torch.zeros(12, 200, dtype=torch.int8)[::2], scale, 64), (codes, torch.zeros(6, 8)[:, ::2], 64),
                    (codes[:, :0], scale[:, :0], 64)):
            with pytest.raises(ValueError):
                be._check_kept(be.PackedRows(*bad, torch.float16), halves)
        with pytest.raises(ValueError):
            be._check_kept(be.PackedRows(codes, scale, 64, torch.float64), halves)
    with pytest.raises(ValueError):
        be._check_kept(be.PackedRows(torch.zeros(6, 129, dtype=torch.int8), scale, 64, torch.float16), 2)


@pytest.mark.parametrize("module", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("autocast", (False, True))
def test_the_router_s_logits_are_fp32(monkeypatch, module, autocast):
    import hiscache
    import hiscache_backend as be
    seen = []
    monkeypatch.setattr(be, "route_rows", lambda logits, top_k, normalize: seen.append(logits))
    layer = hiscache.ExpertMLP(32, 16, 4, 2).to(module)
    x = torch.randn(50, 32).to(module)
    with torch.autocast("cpu", dtype=torch.bfloat16, enabled=autocast):
        layer.route(x)
        layer.route(x, torch.ones(4, dtype=torch.bool))
    want = x.float() @ layer.router.float().t()
    for logits in seen:
        assert logits.dtype == torch.float32 and torch.allclose(logits, want, rtol=32 * 2.0 ** -24, atol=32 * 2.0 ** -23)


def test_arguments_that_would_be_ignored_are_refused():
    import hiscache
    layer, x, expert = hiscache.ExpertMLP(8, 16, 4, 2), torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="weight goes with expert"):
        layer(x, weight=torch.ones(3, 2))
    with pytest.raises(ValueError, match="weight goes with expert"):
        layer(x, expert, allowed=torch.ones(4, dtype=torch.bool))


@pytest.mark.parametrize("call", ("order", "grad"))
def test_calls_of_two_threads_on_one_stream_share_no_scratch_memory(monkeypatch, call):
    """Both calls are held inside the library at the same time, as a call without the interpreter's lock may be."""
    import threading
    import hiscache_backend as be
    meet, seen = threading.Barrier(2), []

    class Library:
        def __getattr__(self, name):
            def enqueue(*args):
                if name.endswith("_workspace_bytes"):
                    return 4096
                seen.append([a for a, b in zip(args, args[1:]) if b == 4096][0])
                meet.wait(timeout=30)
                return 0
            return enqueue

    monkeypatch.setattr(be, "load_library", Library)
    monkeypatch.setattr(be, "_dev", lambda t, *_: t)
    monkeypatch.setattr(be, "_together", lambda *_: None)
    monkeypatch.setattr(be, "_stream_for", lambda _: 0)
    monkeypatch.setattr(be, "_raw_stream", lambda *_: 0)
    monkeypatch.setattr(be, "_ws_cache", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    one = {"order": lambda: be.expert_order(torch.zeros(9000, dtype=torch.int64), 4),
           "grad": lambda: be.expert_linear_grad(torch.zeros(8, 4), torch.zeros(8, 4), torch.tensor([0, 8]))}[call]
    threads = [threading.Thread(target=one) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(seen) == 2 and seen[0] != seen[1]


def test_more_pairs_than_an_order_holds_are_refused(lib, p):
    for n, k in ((1, 1 << 31), (1 << 30, 2), (2, 1 << 30), (1 << 40, 1 << 40), (0, 1 << 31)):
        for call in (lambda: lib.hc_rows_to_experts(p, 0, n, k, 4, 8, p, p, p, None),
                     lambda: lib.hc_rows_from_experts(p, 0, n, k, 4, 8, p, p, p, None),
                     lambda: lib.hc_rows_from_experts_grad(p, p, 0, n, k, 4, 8, p, p, p, p, p, None)):
            assert call() == EUNSUPPORTED, (n, k)


def test_the_documented_limits_of_rows(lib, p):
    """The first size behind each limit is refused before anything is launched."""
    for E, lanes in ((64, 8), (65, 16), (129, 32), (257, 64), (1024, 64)):
        assert lib.hc_route_rows(p, 0, (1 << 32) // lanes, E, 1, 1, p, p, None) == EUNSUPPORTED
        assert lib.hc_route_rows_grad(p, 0, (1 << 32) // lanes, E, 1, 1, p, p, p, p, None) == EUNSUPPORTED
    n = (1 << 32) // 512                                           # rows of 4 096 bf16: 512 pieces
    assert lib.hc_rows_to_experts(p, 2, n, 2, 4, 4096, p, p, p, None) == EUNSUPPORTED
    assert lib.hc_rows_from_experts(p, 2, n, 2, 4, 4096, p, p, p, None) == EUNSUPPORTED
    assert lib.hc_rows_from_experts_grad(p, p, 2, (1 << 32) // 64, 2, 4, 4096, p, p, p, p, p, None) == EUNSUPPORTED
    for group in (32, 64, 128):
        n = (1 << 35) // (2 * group)                               # rows of one group and a column
        assert lib.hc_pack_rows(p, 0, n, group + 1, group, p, p, None) == EUNSUPPORTED
        assert lib.hc_unpack_rows(p, p, n, group + 1, group, p, 0, None) == EUNSUPPORTED
        assert lib.hc_gated_pack(p, 0, n, group + 1, group, p, p, p, None) == EUNSUPPORTED
        assert lib.hc_gated_grad(p, p, p, 0, n, group + 1, group, p, p, None) == EUNSUPPORTED
