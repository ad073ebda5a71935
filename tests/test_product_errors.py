"""A wait that ran out inside a product: recorded in mapped host memory, and not passed over in silence."""
import contextlib
import ctypes as C
from types import SimpleNamespace

import pytest
import torch

import gpu_mode_kernels_b200 as pkg
from gpu_mode_kernels_b200 import _lib, all2all
from gpu_mode_kernels_b200.all2all import A2AContext
from gpu_mode_kernels_b200.linear import check, failed, linear
from gpu_mode_kernels_b200.local_world import LocalWorld
from gpu_mode_kernels_b200.moe import expert_mlp, moe_layer, topk_gate

DEV = "cuda:0"
TIMEOUT = _lib.A2A_ERR_TIMEOUT


def test_devices_that_there_are_not_have_no_word():
    assert _lib.load().a2a_product_word(-1) is None and _lib.load().a2a_product_word(64) is None
    assert _lib.product_error(-1) == 0


def test_codes_become_errors():
    failed(0)
    with pytest.raises(_lib.A2AError, match="earlier product") as e:
        failed(TIMEOUT)
    assert e.value.code == TIMEOUT
    with pytest.raises(_lib.A2AError, match="capacity"):
        failed(_lib.A2A_ERR_CAPACITY)


def context(monkeypatch, own, products):
    """A context whose kernels recorded `own`, on a GPU whose products recorded `products`."""
    left = [products]

    def look():
        code, left[0] = left[0], 0
        if code:
            raise _lib.A2AError(code, "a wait inside a product")

    c = object.__new__(A2AContext)
    c._h, c.device_index = None, 0
    c.lib = SimpleNamespace(a2a_status_peek=lambda h: own)
    c.status = lambda: _lib.Status(code=own)
    c.clear_status = lambda: None
    c.close = lambda: None
    monkeypatch.setattr(_lib, "product_error", lambda device: left[0])
    monkeypatch.setattr(all2all, "check_products", look)
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    return c


def test_a_context_answers_for_the_products_that_its_experts_ran_on(monkeypatch):
    for look in (A2AContext.check, A2AContext.raise_and_clear_if_failed):
        c = context(monkeypatch, 0, TIMEOUT)
        assert c.peek() == 0  # somebody else's: this context has had no experts
        look(c)
        c._products = True
        assert c.peek() == TIMEOUT
        with pytest.raises(_lib.A2AError) as e:
            look(c)
        assert e.value.code == TIMEOUT and c.peek() == 0
        look(c)
        c = context(monkeypatch, _lib.A2A_ERR_ROUTING, TIMEOUT)
        c._products = True
        with pytest.raises(_lib.A2AError) as e:
            look(c)
        assert e.value.code == _lib.A2A_ERR_ROUTING == c.peek()


def record(code):
    word = _lib.load().a2a_product_word(torch.cuda.current_device())
    assert word is not None
    C.c_int32.from_address(word).value = code


@pytest.mark.gpu
def test_products_refuse_after_one_that_recorded_an_error(monkeypatch):
    g = torch.Generator(device=DEV).manual_seed(1)
    x, gate_up, down = (torch.randn(*s, device=DEV, generator=g).bfloat16() for s in ((5, 64), (8, 64, 64), (8, 64, 32)))
    idx, w = topk_gate(x.float()[:, :8].contiguous(), 2)
    rows, counts = torch.randn(8, 1, 4, 64, device=DEV, generator=g).bfloat16(), torch.full((1, 4, 8), 3, dtype=torch.int32, device=DEV)
    kept = torch.zeros_like(rows)
    calls = [lambda: linear(x, gate_up[0]), lambda: linear(x[:, :32], gate_up[0, :, :32]), lambda: moe_layer(x, idx, w, gate_up, down),
             lambda: expert_mlp(rows, counts, gate_up, down, out=kept)]
    want = [f().clone() for f in calls]
    kept.zero_()
    for host in (_lib.host(), _lib.Interpreted):
        monkeypatch.setattr(_lib, "_host", host)
        record(TIMEOUT)
        for f in calls:  # until somebody has looked
            with pytest.raises(_lib.A2AError, match="earlier product") as e:
                f()
            assert e.value.code == TIMEOUT
        assert _lib.product_error(0) == TIMEOUT
        topk_gate(x.float()[:, :8].contiguous(), 2)  # waits for nothing
        with pytest.raises(_lib.A2AError) as e:
            check()
        assert e.value.code == TIMEOUT and not bool(kept.any()) and _lib.product_error(0) == 0
        check()
        assert all(torch.equal(f(), y) for f, y in zip(calls, want))
        kept.zero_()


@pytest.mark.gpu
def test_a_group_whose_experts_recorded_an_error_says_so():
    cfg, rd, _, _ = pkg.generate_input(8, 2, 64, 6, seed=5, rank=0, world_size=1, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(2)
    experts = [tuple(torch.randn(*s, device=DEV, generator=g).bfloat16() for s in ((8, 64, 64), (8, 64, 32)))]
    group = LocalWorld(cfg, 1)
    try:
        want = group.forward_phases([rd], experts=experts)[0].clone()
        group.check()
        record(TIMEOUT)
        assert group.ctxs[0].peek() == TIMEOUT
        with pytest.raises(_lib.A2AError):
            group.check()
        assert group.ctxs[0].peek() == 0
        group.check()
        record(TIMEOUT)
        with pytest.raises(_lib.A2AError):
            group.ctxs[0].raise_and_clear_if_failed()
        assert torch.equal(group.forward_phases([rd], experts=experts)[0], want)
        group.check()
    finally:
        group.close()
