"""The gate, the experts' products and dense products against 64 bits, and what they refuse."""
import ctypes as C
import zlib

import pytest
import torch

import gpu_mode_kernels_b200 as pkg
from gpu_mode_kernels_b200 import _lib
from gpu_mode_kernels_b200.linear import DTYPES, check, linear
from gpu_mode_kernels_b200.moe import expert_mlp, moe_layer, route, topk_gate
from tests import product_oracle as O

DEV = "cuda:0"
CONFIG, CAPACITY = _lib.A2A_ERR_CONFIG, _lib.A2A_ERR_CAPACITY


def generator(*seed):
    return torch.Generator().manual_seed(zlib.crc32(repr(seed).encode()))


def normal(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g) * std).to(dtype)


def some_experts(g, E, hidden, inner, dtype):
    return normal(g, E, 2 * inner, hidden, std=hidden ** -0.5, dtype=dtype), normal(g, E, hidden, inner, std=inner ** -0.5, dtype=dtype)


def distinct(g, tokens, E, k):
    return torch.rand(tokens, E, generator=g).topk(k, dim=1).indices.to(torch.int32)


# ---- refusals at the C boundary, without a device ---------------------------------------------------
ONE = 1 << 20  # an address that is aligned and never read


def gate_args(**kw):
    a = dict(logits=ONE, stride=8, bias=0, indices=ONE, weights=ONE, tokens=2, experts=8, topk=2, dtype=0, score=0, renormalize=1, scale=1.0)
    return _lib.Gate(**{**a, **kw})


def linear_args(**kw):
    a = dict(x=ONE, weight=ONE, bias=0, residual=0, y=ONE, x_stride=64, weight_stride=64, residual_stride=0, y_stride=16, tokens=2, inputs=64,
             outputs=16, dtype=0, out_dtype=0, bias_dtype=0, activation=0)
    return _lib.Linear(**{**a, **kw})


def layer_args(**kw):
    a = dict(x=ONE, topk_idx=ONE, topk_weights=ONE, gate_up=ONE, down=ONE, residual=0, y=ONE, workspace=ONE, workspace_bytes=1 << 30, tokens=2,
             topk=2, experts=8, hidden_dim=64, inner=32, dtype=0)
    return _lib.Layer(**{**a, **kw})


def experts_args(**kw):
    a = dict(rows=ONE, counts=ONE, gate_up=ONE, down=ONE, out=ONE, workspace=ONE, workspace_bytes=1 << 30, local_experts=4, world=2, capacity=8,
             hidden_dim=64, inner=32, dtype=0)
    return _lib.Experts(**{**a, **kw})


@pytest.mark.parametrize("make,entry,kw", [
    *[(gate_args, "a2a_gate", kw) for kw in (
        dict(dtype=3), dict(experts=0), dict(experts=1025), dict(topk=0), dict(topk=9), dict(topk=33, experts=64), dict(score=2), dict(tokens=-1), dict(tokens=(1 << 30) + 1),
        dict(logits=0), dict(indices=0), dict(weights=0), dict(stride=-8))],
    *[(linear_args, "a2a_linear", kw) for kw in (
        dict(dtype=2), dict(dtype=1, out_dtype=0), dict(bias=ONE, bias_dtype=1), dict(activation=5), dict(activation=-1), dict(tokens=-1),
        dict(inputs=0), dict(inputs=60, x_stride=64), dict(outputs=0), dict(outputs=(1 << 24) + 1, y_stride=(1 << 24) + 1), dict(tokens=(1 << 30) + 1), dict(inputs=65544, x_stride=65544, weight_stride=65544),
        dict(x=0), dict(weight=0), dict(y=0), dict(x=ONE + 8), dict(weight=ONE + 2), dict(x_stride=56), dict(x_stride=68), dict(weight_stride=60),
        dict(y_stride=15), dict(residual=ONE, residual_stride=-1))],
    *[(layer_args, "a2a_layer", kw) for kw in (
        dict(dtype=2), dict(experts=0), dict(experts=1025), dict(hidden_dim=60), dict(inner=0), dict(inner=4), dict(tokens=-1), dict(tokens=257),
        dict(topk=0), dict(topk=33), dict(x=0), dict(topk_idx=0), dict(topk_weights=0), dict(gate_up=0), dict(down=0), dict(y=0), dict(workspace=0),
        dict(x=ONE + 8), dict(gate_up=ONE + 8), dict(down=ONE + 8), dict(workspace=ONE + 64))],
    *[(experts_args, "a2a_experts", kw) for kw in (
        dict(dtype=2), dict(local_experts=0), dict(local_experts=1025), dict(world=0), dict(world=9), dict(capacity=0), dict(capacity=65536),
        dict(hidden_dim=4), dict(inner=36), dict(rows=0), dict(counts=0), dict(gate_up=0), dict(down=0), dict(out=0), dict(workspace=0),
        dict(rows=ONE + 8), dict(workspace=ONE + 16))],
])
def test_bad_arguments_are_refused_before_a_device_is_touched(make, entry, kw):
    assert getattr(_lib.load(), entry)(C.byref(make(**kw)), None) == CONFIG


def test_small_workspaces_no_tokens_and_null():
    lib = _lib.load()
    for tokens in (8, 9, 256):
        need = lib.a2a_layer_workspace(tokens, 2, 64, 32)
        assert need >= tokens * 2 * 32 * 2
        assert lib.a2a_layer(C.byref(layer_args(tokens=tokens, workspace_bytes=need - 1)), None) == CAPACITY
    need = lib.a2a_experts_workspace(4, 2, 8, 32)
    assert need >= 4 * 2 * 8 * 32 * 2
    assert lib.a2a_experts(C.byref(experts_args(workspace_bytes=need - 1)), None) == CAPACITY
    assert lib.a2a_layer_workspace(-1, 2, 64, 32) == lib.a2a_experts_workspace(0, 2, 8, 32) == 0
    for make, entry in ((gate_args, "a2a_gate"), (linear_args, "a2a_linear"), (layer_args, "a2a_layer")):
        assert getattr(lib, entry)(C.byref(make(tokens=0)), None) == 0
        assert getattr(lib, entry)(None, None) == CONFIG
    assert lib.a2a_experts(None, None) == lib.a2a_product_status(None) == CONFIG


def test_host_tensors_are_refused():
    g = generator(1)
    x, w = normal(g, 4, 64, dtype=torch.bfloat16), normal(g, 16, 64, dtype=torch.bfloat16)
    gate_up, down = some_experts(g, 8, 64, 32, torch.bfloat16)
    for call in (lambda: linear(x, w), lambda: topk_gate(normal(g, 4, 8), 2), lambda: route(x, w, 2),
                 lambda: moe_layer(x, distinct(g, 4, 8, 2), torch.ones(4, 2), gate_up, down),
                 lambda: expert_mlp(torch.zeros(8, 1, 4, 64, dtype=torch.bfloat16), torch.zeros(1, 4, 8, dtype=torch.int32), gate_up, down)):
        with pytest.raises(_lib.A2AError):
            call()


# ---- the oracle's own arithmetic: two ways to the same numbers --------------------------------------------
def test_the_oracles_layer_is_the_sum_over_pairs():
    g = generator(2)
    gate_up, down = some_experts(g, 5, 16, 24, torch.float16)
    x, w = normal(g, 6, 16, dtype=torch.float16), torch.rand(6, 3, generator=g)
    idx = distinct(g, 6, 5, 3)
    idx[1] = torch.tensor([4, 4, 9])
    want = torch.zeros(6, 16, dtype=torch.float64)
    for t in range(6):
        for k in range(3):
            e = int(idx[t, k])
            if e < 5:
                h = gate_up[e].double() @ x[t].double()
                want[t] += float(w[t, k]) * (down[e].double() @ (h[:24] / (1 + torch.exp(-h[:24])) * h[24:]))
    got, bound = O.layer(x, idx, w, gate_up, down, None)
    torch.testing.assert_close(got, want, rtol=1e-12, atol=1e-12)
    assert bool((bound > 0).all())


# ---- gate ----------------------------------------------------------------------------------------------------
def check_gate(logits, k, **kw):
    args = dict(score="softmax", bias=None, renormalize=True, scale=1.0)
    args.update(kw)
    dev = logits.to(DEV) if not logits.is_cuda else logits
    idx, w = topk_gate(dev, k, **{**args, "bias": None if args["bias"] is None else args["bias"].to(DEV)})
    want_idx, want = O.gate(logits.cpu(), k, args["score"], args["bias"], args["renormalize"], args["scale"])
    assert idx.dtype == torch.int32 and torch.equal(idx.cpu(), want_idx)
    # expf and logistic 4 half steps of 2^-23 together, a sum of up to 1024 terms and one of k, two divisions, a product, rounding
    torch.testing.assert_close(w.cpu().double(), want, rtol=2.0 ** -18, atol=1e-38)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,experts,k", [(1, 64, 6), (1, 1, 1), (3, 2, 2), (5, 33, 16), (130, 64, 8), (7, 128, 4), (9, 256, 8), (64, 384, 8),
                                              (2, 513, 32), (3, 1024, 32), (5, 32, 32)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kw", [dict(), dict(renormalize=False), dict(score="sigmoid", scale=2.5), dict(score="sigmoid", bias=True),
                                dict(bias=True, renormalize=False)], ids=str)
def test_gate(tokens, experts, k, dtype, kw):
    g = generator(tokens, experts, k)
    logits = normal(g, tokens, experts, std=2.0).to(dtype)
    kw = dict(kw, bias=normal(g, experts, std=0.1)) if kw.get("bias") else kw
    check_gate(logits, k, **kw)


@pytest.mark.gpu
def test_gate_ties_strides_and_views():
    g = generator(3)
    check_gate(torch.zeros(4, 100), 7)
    check_gate(torch.tensor([[0.0, -0.0, 1.0, -0.0, 1.0, 0.0]]).repeat(3, 1), 5)
    wide = normal(g, 6, 200).to(DEV)
    check_gate(wide[:, 3:70], 4)
    check_gate(wide[::2, 100:], 4)
    check_gate(normal(g, 40, 9).to(DEV).t(), 3)
    check_gate(wide[:1].expand(5, 200), 3)
    assert topk_gate(wide[:0], 3)[0].shape == (0, 3)


@pytest.mark.gpu
def test_gate_rows_with_nothing_to_choose():
    inf = float("inf")
    logits = torch.full((5, 40), -inf)
    logits[1, 17] = 0.5           # one expert left, two asked for: the others are the first excluded ones
    logits[2, 30], logits[2, 3] = 2.0, 2.0
    logits[3] = torch.arange(40.0)
    logits[3, 12] = float("nan")  # ranks first; its row has no weights
    logits[4, 5] = torch.finfo(torch.float32).min
    idx, w = topk_gate(logits.to(DEV), 2)
    assert idx.tolist() == [[0, 1], [17, 0], [3, 30], [12, 39], [5, 0]]
    assert w[:3].tolist() == [[0.0, 0.0], [1.0, 0.0], [0.5, 0.5]] and w[4].tolist() == [1.0, 0.0] and bool(w[3].isnan().all())
    idx, w = topk_gate(logits.to(DEV), 2, score="sigmoid")
    assert w[0].tolist() == [0.0, 0.0] and w[1].tolist() == [1.0, 0.0]
    idx, w = topk_gate(logits.to(DEV), 2, bias=torch.zeros(40, device=DEV))
    assert idx[:3].tolist() == [[0, 1], [17, 0], [3, 30]] and w[:3].tolist() == [[0.0, 0.0], [1.0, 0.0], [0.5, 0.5]]
    assert sorted(set(idx[3].tolist())) == sorted(idx[3].tolist()) and 0 <= int(idx.min()) and int(idx.max()) < 40


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_gate_excluded_experts_stay_out_whatever_their_bias(score):
    logits, bias = torch.full((4, 70), -float("inf")), torch.zeros(70)
    logits[:, 40:45] = torch.arange(5.0)
    logits[1, 66] = -1e30         # small, but a number
    logits[2, 41:45] = -float("inf")  # one left, three asked for
    logits[3] = -float("inf")
    bias[:8], bias[66] = 5.0, 2.0
    idx, w = topk_gate(logits.to(DEV), 3, score=score, bias=bias.to(DEV), renormalize=False)
    assert idx.tolist() == [[44, 43, 42], [66, 44, 43], [40, 0, 1], [0, 1, 2]]
    s = torch.softmax(logits.double(), 1).nan_to_num() if score == "softmax" else torch.sigmoid(logits.double())
    torch.testing.assert_close(w.cpu().double(), s.gather(1, idx.cpu().long()), rtol=2.0 ** -18, atol=1e-38)


@pytest.mark.gpu
def test_gate_refusals():
    l = torch.zeros(4, 16, device=DEV)
    for call in (lambda: topk_gate(l.double(), 2), lambda: topk_gate(l[0], 2), lambda: topk_gate(l, 0), lambda: topk_gate(l, 17),
                 lambda: topk_gate(l, 2, score="tanh"), lambda: topk_gate(l, 2, bias=l[0, :8]), lambda: topk_gate(l, 2, bias=l[0].half()),
                 lambda: topk_gate(l, 2, bias=torch.zeros(16)), lambda: topk_gate(torch.zeros(2, 1025, device=DEV), 2),
                 lambda: topk_gate(torch.zeros(2, 64, device=DEV), 33), lambda: topk_gate(torch.zeros(2, 0, device=DEV), 1)):
        with pytest.raises(_lib.A2AError):
            call()


# ---- dense products --------------------------------------------------------------------------------------------
def check_linear(x, w, bias=None, activation="none", residual=None, out_dtype=None):
    args = [None if t is None else t.to(DEV) for t in (x, w, bias, residual)]
    y = linear(args[0], args[1], args[2], activation=activation, residual=args[3], out_dtype=out_dtype)
    flat = [None if t is None else t.cpu().reshape(-1, t.shape[-1]) for t in (x, residual)]
    value, bound = O.linear(flat[0], w.cpu(), None if bias is None else bias.cpu(), activation, flat[1], out_dtype or x.dtype)
    assert y.shape[:-1] == x.shape[:-1] and y.dtype == (out_dtype or x.dtype) and y.is_contiguous()
    O.assert_within(y.reshape(value.shape), value, bound, f"{tuple(x.shape)} {tuple(w.shape)} {activation}")
    return y


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 2, 7, 8, 9, 16, 17, 33, 100, 255, 256, 257, 300, 600])
@pytest.mark.parametrize("inputs,outputs", [(8, 1), (72, 15), (64, 128), (520, 333), (1000, 1025)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_linear_sizes(tokens, inputs, outputs, dtype):
    g = generator(tokens, inputs, outputs)
    x, w = normal(g, tokens, inputs, dtype=dtype), normal(g, outputs, inputs, std=inputs ** -0.5, dtype=dtype)
    check_linear(x, w)
    check_linear(x, w, out_dtype=torch.float32)
    check()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 5, 12, 40, 270])
@pytest.mark.parametrize("activation", ["none", "relu", "gelu", "silu", "swiglu"])
@pytest.mark.parametrize("bias,residual,out", [(None, False, None), ("same", True, None), ("fp32", True, torch.float32), ("same", False, None)])
def test_linear_epilogues(tokens, activation, bias, residual, out):
    g, dtype = generator(tokens, activation, residual), torch.bfloat16 if tokens % 2 else torch.float16
    outputs, inputs = 203, 328
    rows = outputs * (2 if activation == "swiglu" else 1)
    b = None if bias is None else normal(g, rows, dtype=dtype if bias == "same" else torch.float32)
    check_linear(normal(g, tokens, inputs, dtype=dtype), normal(g, rows, inputs, std=inputs ** -0.5, dtype=dtype), b, activation,
                 normal(g, tokens, outputs, dtype=out or dtype) if residual else None, out)
    check()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,inputs,outputs", [(2000, 512, 1100), (1100, 136, 2048), (513, 1024, 2050), (1030, 2048, 384), (90, 2880, 700)])
@pytest.mark.parametrize("activation,bias,residual,out", [("none", None, True, None), ("swiglu", "fp32", True, torch.float32), ("gelu", "same", False, None),
                                                          ("swiglu", None, False, None), ("silu", "same", True, torch.float32)])
def test_linear_many_rows(tokens, inputs, outputs, activation, bias, residual, out):
    """Single blocks, clusters that share a sum and pairs of blocks; whole and ragged tiles; stores of sixteen bytes and of single values."""
    g, dtype = generator(tokens, activation), torch.bfloat16 if outputs % 4 else torch.float16
    rows = outputs * (2 if activation == "swiglu" else 1)
    b = None if bias is None else normal(g, rows, dtype=dtype if bias == "same" else torch.float32)
    check_linear(normal(g, tokens, inputs, dtype=dtype), normal(g, rows, inputs, std=inputs ** -0.5, dtype=dtype), b, activation,
                 normal(g, tokens, outputs, dtype=out or dtype) if residual else None, out)
    check()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,inputs,outputs", [(1, 7168, 600), (16, 7168, 256), (64, 7168, 256), (40, 4096, 1000), (3, 20000, 40)])
def test_linear_long_sums(tokens, inputs, outputs):
    g = generator(tokens, inputs)
    x, w = normal(g, tokens, inputs, dtype=torch.bfloat16), normal(g, outputs, inputs, std=inputs ** -0.5, dtype=torch.bfloat16)
    check_linear(x, w, out_dtype=torch.float32)
    check_linear(x, w, residual=normal(g, tokens, outputs, dtype=torch.bfloat16))


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,inputs,outputs", [(600, 7168, 512), (1000, 4096, 2048), (20, 7168, 3000), (5, 7168, 256)])
def test_linear_sums_of_32_bits_do_not_drift(tokens, inputs, outputs):
    """The tensor core cuts its sums after every 16 products: up to 2^-23 of what is there, 2/3 of the end's on average. In parts of at most 896, 56 of them,
    that is 56 * 2/3 * 2^-23 in the 2-norm even if all go one way; 7168 at once were 8e-6 off."""
    g = generator(tokens, inputs, 32)
    x, w = normal(g, tokens, inputs, dtype=torch.bfloat16).to(DEV), normal(g, outputs, inputs, std=inputs ** -0.5, dtype=torch.bfloat16).to(DEV)
    want = x.double() @ w.double().t()
    assert float((linear(x, w, out_dtype=torch.float32).double() - want).norm() / want.norm()) < 56 * 2 / 3 * 2.0 ** -23


@pytest.mark.gpu
def test_linear_strides_shapes_and_views():
    g = generator(5)
    base = normal(g, 80, 400, dtype=torch.bfloat16).to(DEV)
    w = normal(g, 96, 640, std=0.1, dtype=torch.bfloat16).to(DEV)
    for rows in (6, 40):
        check_linear(base[:rows, 16:272], w[:, 64:320])             # rows further apart than they are long
        check_linear(base[:rows:2, 3:259], w[:, :256])              # a start that is off 16 bytes: copied
        check_linear(base.t()[:rows, :80], w[::2, :80])             # columns for rows: copied
        check_linear(base[:1, :256].expand(rows, 256), w[:, :256])  # one row many times
        shifted = torch.empty(rows * 256 + 3, dtype=torch.bfloat16, device=DEV)[3:].view(rows, 256).copy_(base[:rows, :256])
        check_linear(shifted, w[:, :256].contiguous())              # contiguous, but off 16 bytes: copied
        check_linear(base[:rows, :256], w[:, :256], residual=base[:rows, 100:196])
        check_linear(base[:rows, :256], w[:, :256], residual=base[:1, 100:196].expand(rows, 96))
        check_linear(base[:rows, :256], w[:, :256], residual=normal(g, 96, rows, dtype=torch.bfloat16).to(DEV).t())
    check_linear(base.view(4, 20, 400)[:, :, :64], w[:, :64])
    check_linear(base[0, :64], w[:, :64], residual=base[1, :96])
    check_linear(base[:1, :64], w[:1, :64])
    odd = normal(g, 3, 403, dtype=torch.bfloat16).to(DEV)
    check_linear(base[:5, :64], torch.as_strided(w, (1, 64), (7, 1)), odd[:, 0][:1])  # strides of a length of one say nothing
    assert linear(base[:0, :64], w[:, :64]).shape == (0, 96)
    assert linear(base.view(4, 20, 400)[:, :0, :64], w[:, :64]).shape == (4, 0, 96)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,inputs", [(5, 2048), (70, 72), (600, 136), (1500, 520)])
@pytest.mark.parametrize("outputs,stride", [(203, 208), (203, 211), (1000, 1016), (1001, 1008)])
@pytest.mark.parametrize("activation,onto,out", [("none", False, None), ("gelu", False, None), ("silu", True, None), ("swiglu", False, None), ("swiglu", True, torch.float32),
                                                 ("none", True, torch.float32)])
def test_linear_results_in_rows_further_apart(tokens, inputs, outputs, stride, activation, onto, out):
    """The C entry's strides: results beside what is not theirs, and onto the residual."""
    g, dtype = generator(tokens, outputs, stride, activation), torch.float16 if stride % 3 else torch.bfloat16
    rows = outputs * (2 if activation == "swiglu" else 1)
    x, w, b = normal(g, tokens, inputs, dtype=dtype), normal(g, rows, inputs, std=inputs ** -0.5, dtype=dtype), normal(g, rows, dtype=dtype)
    before = normal(g, tokens, stride, dtype=out or dtype)
    dev, y = [t.to(DEV) for t in (x, w, b)], before.to(DEV)
    at = y.data_ptr()
    args = _lib.Linear(*(t.data_ptr() for t in dev), at if onto else 0, at, inputs, inputs, stride if onto else 0, stride, tokens, inputs, outputs,
                       DTYPES[dtype], DTYPES[out or dtype], DTYPES[dtype], _lib.ACTIVATION[activation])
    assert _lib.load().a2a_linear(C.byref(args), _lib.current_stream()) == 0
    check()
    value, bound = O.linear(x, w, b, activation, before[:, :outputs] if onto else None, out or dtype)
    O.assert_within(y[:, :outputs], value, bound)
    assert torch.equal(y[:, outputs:].cpu(), before[:, outputs:])


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 30, 300])
def test_linear_many_outputs(tokens):
    """As many as a vocabulary has, past the sizes that a layer's matrices have."""
    g = generator(tokens, 70001)
    x, w = normal(g, tokens, 64, dtype=torch.bfloat16), normal(g, 70001, 64, std=0.125, dtype=torch.bfloat16)
    check_linear(x, w, out_dtype=torch.float32)
    check_linear(x, w, normal(g, 70001, dtype=torch.bfloat16), residual=normal(g, tokens, 70001, dtype=torch.bfloat16))


@pytest.mark.gpu
def test_linear_infinities_stay_in_their_rows_and_columns():
    g = generator(6)
    for tokens in (5, 12, 50):
        x, w = normal(g, tokens, 136, dtype=torch.float16), normal(g, 150, 136, std=0.1, dtype=torch.float16)
        want = linear(x.to(DEV), w.to(DEV)).cpu()
        x[2, 7], w[31, 9] = float("inf"), float("nan")
        got = linear(x.to(DEV), w.to(DEV)).cpu()
        rows, cols = [t for t in range(tokens) if t != 2], [f for f in range(150) if f != 31]
        assert torch.equal(got[rows][:, cols], want[rows][:, cols])
        assert not bool(got[2].isfinite().any()) and bool(got[:, 31].isnan().all())


@pytest.mark.gpu
def test_linear_refusals():
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16, device=DEV), torch.zeros(16, 64, dtype=torch.bfloat16, device=DEV)
    b, r = torch.zeros(16, device=DEV), torch.zeros(4, 16, dtype=torch.bfloat16, device=DEV)
    for call in (lambda: linear(x.float(), w.float()), lambda: linear(x, w.half()), lambda: linear(x, w[:, :56]), lambda: linear(x, w[0]),
                 lambda: linear(x, w, activation="tanh"), lambda: linear(x[:, :60], w[:, :60]), lambda: linear(x, w[:0]),
                 lambda: linear(x, w[:15], activation="swiglu"), lambda: linear(x, w, b.double()), lambda: linear(x, w, b[:8]),
                 lambda: linear(x, w, b.cpu()), lambda: linear(x, w, residual=r.float()), lambda: linear(x, w, residual=r[:2]),
                 lambda: linear(x, w, residual=r.cpu()), lambda: linear(x, w, out_dtype=torch.float16), lambda: linear(x, w.cpu()),
                 lambda: linear(x[:, 4:60], w[:, 4:60]), lambda: linear(x, w.t()[:, :16].t()[:, ::2])):
        with pytest.raises(_lib.A2AError):
            call()


# ---- a layer of a few tokens ----------------------------------------------------------------------------------------
def check_layer(x, idx, w, gate_up, down, residual=None):
    args = [None if t is None else t.to(DEV) for t in (x, idx, w, gate_up, down, residual)]
    y = moe_layer(*args[:5], residual=args[5])
    assert y.shape == x.shape and y.dtype == x.dtype
    O.assert_within(y, *O.layer(x, idx, w, gate_up, down, residual), f"{tuple(x.shape)} {tuple(idx.shape)}")
    check()
    return y


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 2, 5, 8, 9, 17, 64, 173, 256])
@pytest.mark.parametrize("E,k,hidden,inner", [(8, 2, 256, 136), (64, 6, 128, 64), (4, 4, 72, 200), (1, 1, 8, 8), (300, 8, 264, 24)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_layer(tokens, E, k, hidden, inner, dtype):
    g = generator(tokens, E, k)
    gate_up, down = some_experts(g, E, hidden, inner, dtype)
    x, idx = normal(g, tokens, hidden, dtype=dtype), distinct(g, tokens, E, k)
    w = torch.softmax(normal(g, tokens, k), 1)
    check_layer(x, idx, w, gate_up, down)
    check_layer(x, idx, w, gate_up, down, normal(g, tokens, hidden, dtype=dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 6, 8, 9, 30])
def test_layer_pads_repeats_and_weights_of_any_sign(tokens):
    """Indices outside the experts mark none, a token may have none at all, and the same expert twice counts twice."""
    g, E, k, hidden, inner = generator(tokens, 7), 16, 5, 136, 72
    gate_up, down = some_experts(g, E, hidden, inner, torch.bfloat16)
    x, w = normal(g, tokens, hidden, dtype=torch.bfloat16), normal(g, tokens, k)
    idx = torch.randint(-2, E + 2, (tokens, k), generator=g, dtype=torch.int32)
    idx[-1] = torch.tensor([-1, E, 1 << 30, -(1 << 31), -1], dtype=torch.int32)
    idx[0] = torch.tensor([3, 3, 7, 3, -1], dtype=torch.int32) if tokens > 1 else idx[0]
    residual = normal(g, tokens, hidden, dtype=torch.bfloat16)
    y = check_layer(x, idx, w, gate_up, down)
    assert not bool(y[-1].any())
    y = check_layer(x, idx, w, gate_up, down, residual)
    assert torch.equal(y[-1].cpu(), residual[-1])


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [8, 9, 256])
def test_layer_one_expert_for_all_and_most_choices(tokens):
    g = generator(tokens, 8)
    gate_up, down = some_experts(g, 40, 64, 40, torch.bfloat16)
    x = normal(g, tokens, 64, dtype=torch.bfloat16)
    check_layer(x, torch.full((tokens, 1), 39, dtype=torch.int32), torch.ones(tokens, 1), gate_up, down)
    check_layer(x, distinct(g, tokens, 40, 32), torch.rand(tokens, 32, generator=g), gate_up, down)
    check_layer(x, torch.full((tokens, 32), 5, dtype=torch.int32), torch.rand(tokens, 32, generator=g), gate_up, down)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [5, 20])
def test_layer_infinities_reach_only_their_tokens(tokens):
    """Weights of experts that nobody chose, and of experts that others chose, may hold anything."""
    g = generator(tokens, 9)
    gate_up, down = some_experts(g, 8, 64, 48, torch.bfloat16)
    x, w = normal(g, tokens, 64, dtype=torch.bfloat16), torch.rand(tokens, 2, generator=g)
    idx = distinct(g, tokens, 6, 2)
    idx[3] = torch.tensor([6, 1])
    want = moe_layer(*(t.to(DEV) for t in (x, idx, w, gate_up, down)))
    gate_up[7], down[7] = float("nan"), float("inf")
    gate_up[6] = float("nan")
    got = moe_layer(*(t.to(DEV) for t in (x, idx, w, gate_up, down)))
    others = [t for t in range(tokens) if t != 3]
    assert torch.equal(got[others], want[others]) and bool(got[3].isnan().all())


@pytest.mark.gpu
def test_layer_repeats_itself_bit_for_bit():
    g = generator(10)
    gate_up, down = (t.to(DEV) for t in some_experts(g, 32, 256, 128, torch.bfloat16))
    for tokens in (7, 120):
        x, idx = normal(g, tokens, 256, dtype=torch.bfloat16).to(DEV), distinct(g, tokens, 32, 8).to(DEV)
        w = torch.rand(tokens, 8, generator=g).to(DEV)
        first = moe_layer(x, idx, w, gate_up, down)
        for _ in range(20):
            assert torch.equal(moe_layer(x, idx, w, gate_up, down), first)


@pytest.mark.gpu
def test_layer_refusals():
    g = generator(11)
    gate_up, down = (t.to(DEV) for t in some_experts(g, 8, 64, 32, torch.bfloat16))
    x, idx, w = normal(g, 4, 64, dtype=torch.bfloat16).to(DEV), distinct(g, 4, 8, 2).to(DEV), torch.ones(4, 2, device=DEV)
    assert moe_layer(x[:0], idx[:0], w[:0], gate_up, down).shape == (0, 64)
    for args, kw in (((x.float(), idx, w, gate_up, down), {}), ((x.t(), idx, w, gate_up, down), {}), ((x, idx.long(), w, gate_up, down), {}),
                     ((x, idx[:2], w, gate_up, down), {}), ((x, idx, w.half(), gate_up, down), {}), ((x, idx, w[:, :1], gate_up, down), {}),
                     ((x, idx, w, gate_up.half(), down), {}), ((x, idx, w, gate_up[:4], down), {}), ((x, idx, w, down, gate_up), {}),
                     ((x, idx, w, gate_up, down.cpu()), {}), ((x, idx, w, gate_up, down), dict(residual=x[:2])),
                     ((x, idx, w, gate_up, down), dict(residual=x.float())), ((x, idx, w, gate_up[:, :, ::2], down[:, ::2]), {}),
                     ((x.repeat(65, 1), idx.repeat(65, 1), w.repeat(65, 1), gate_up, down), {}),
                     ((x, idx.repeat(1, 17), w.repeat(1, 17), gate_up, down), {}), ((x, idx[:, :0], w[:, :0], gate_up, down), {}),
                     ((x[:, :60].contiguous(), idx, w, gate_up[:, :, :60].contiguous(), down[:, :60].contiguous()), {})):
        with pytest.raises(_lib.A2AError):
            moe_layer(*args, **kw)


# ---- experts on dispatched rows -------------------------------------------------------------------------------------
def check_slabs(rows, n, gate_up, down, in_place=False):
    """n: valid rows [world, local]."""
    local, world, capacity, hidden = rows.shape
    counts = torch.full((world, 4, local), 1 << 20, dtype=torch.int32)  # entries 1 to 3 are not read
    counts[:, 0] = n
    given = rows.to(DEV)
    out = None if in_place else torch.full_like(given, 3.0)
    args = [t.to(DEV) for t in (counts, gate_up, down)]
    got = expert_mlp(given, *args, out=out)
    assert got is (given if in_place else out)
    if not in_place:
        assert torch.equal(given.cpu().view(torch.int16), rows.view(torch.int16))
    got = got.cpu()
    for l in range(local):
        for s in range(world):
            v = min(max(int(n[s, l]), 0), capacity)
            if v:
                value, bound = O.expert(rows[l, s, :v], gate_up[l], down[l], rows.dtype)
                O.assert_within(got[l, s, :v], value, O.rounded(value, bound, rows.dtype), f"slab {l}, {s}")
            behind = rows[l, s, v:] if in_place else torch.full_like(rows[l, s, v:], 3.0)
            assert torch.equal(got[l, s, v:].view(torch.int16), behind.view(torch.int16)), "rows behind the last one"
    check()


@pytest.mark.gpu
@pytest.mark.parametrize("local,world,capacity,hidden,inner", [(4, 2, 24, 128, 72), (1, 1, 1, 8, 8), (3, 8, 70, 136, 64), (32, 4, 9, 64, 40),
                                                               (2, 3, 400, 72, 136)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("in_place", [False, True])
def test_experts_on_slabs(local, world, capacity, hidden, inner, dtype, in_place):
    g = generator(local, world, capacity)
    gate_up, down = some_experts(g, local, hidden, inner, dtype)
    rows = normal(g, local, world, capacity, hidden, dtype=dtype)
    n = torch.randint(0, capacity + 1, (world, local), generator=g)
    n[0, 0], n[-1, -1] = capacity, 0 if world * local > 1 else capacity
    behind = torch.arange(capacity)[None, None] >= n.t()[..., None]
    rows[behind] = float("nan")  # what an earlier call left
    check_slabs(rows, n, gate_up, down, in_place)


@pytest.mark.gpu
@pytest.mark.parametrize("hidden,inner", [(1416, 8), (8, 2056)])
def test_more_tiles_than_a_block_has_room_for(hidden, inner):
    """1024 experts of a row each, of which a block gets 80 to 230 tiles: in its table, and behind the end of that."""
    g = generator(hidden, inner)
    gate_up, down = some_experts(g, 1024, hidden, inner, torch.bfloat16)
    x, w = normal(g, 32, hidden, dtype=torch.bfloat16), torch.softmax(normal(g, 32, 32), 1)
    check_layer(x, torch.randperm(1024, generator=g).view(32, 32).to(torch.int32), w, gate_up, down)
    check_slabs(normal(g, 1024, 1, 1, hidden, dtype=torch.bfloat16), torch.ones(1, 1024, dtype=torch.int64), gate_up, down)


@pytest.mark.gpu
@pytest.mark.parametrize("hidden", [64, 264, 1032])
def test_experts_results_off_sixteen_bytes(hidden):
    g = generator(hidden, 3)
    gate_up, down = some_experts(g, 3, hidden, 40, torch.float16)
    rows, n = normal(g, 3, 2, 70, hidden, dtype=torch.float16), torch.tensor([[70, 0, 33], [1, 64, 7]])
    space = torch.full((rows.numel() + 3,), 3.0, dtype=torch.float16, device=DEV)
    out = space[3:].view(rows.shape)
    counts = torch.zeros(2, 4, 3, dtype=torch.int32)
    counts[:, 0] = n
    expert_mlp(rows.to(DEV), counts.to(DEV), gate_up.to(DEV), down.to(DEV), out=out)
    check()
    for l in range(3):
        for s in range(2):
            v = int(n[s, l])
            if v:
                value, bound = O.expert(rows[l, s, :v], gate_up[l], down[l], rows.dtype)
                O.assert_within(out[l, s, :v], value, O.rounded(value, bound, rows.dtype))
            assert bool((out[l, s, v:] == 3.0).all())
    assert bool((space[:3] == 3.0).all())


@pytest.mark.gpu
def test_experts_without_rows_and_with_counts_out_of_range():
    g = generator(12)
    gate_up, down = some_experts(g, 5, 64, 40, torch.bfloat16)
    rows = normal(g, 5, 2, 6, 64, dtype=torch.bfloat16)
    check_slabs(rows, torch.zeros(2, 5, dtype=torch.int64), gate_up, down)
    n = torch.tensor([[-3, 7, 1 << 30, 0, 2], [6, -(1 << 31), 0, 6, 1]])
    check_slabs(rows, n, gate_up, down)
    check_slabs(rows, n, gate_up, down, in_place=True)


@pytest.mark.gpu
def test_experts_refusals():
    g = generator(13)
    gate_up, down = (t.to(DEV) for t in some_experts(g, 4, 64, 32, torch.bfloat16))
    rows, counts = torch.zeros(4, 2, 8, 64, dtype=torch.bfloat16, device=DEV), torch.zeros(2, 4, 4, dtype=torch.int32, device=DEV)
    space = torch.zeros(4 * 2 * 8 * 64 + 64, dtype=torch.bfloat16, device=DEV)
    inside, shifted = space[:4096].view(4, 2, 8, 64), space[64:].view(4, 2, 8, 64)
    for args in ((rows.float(), counts, gate_up, down), (rows[0], counts, gate_up, down), (rows.transpose(0, 1), counts, gate_up, down),
                 (rows, counts.long(), gate_up, down), (rows, counts[:1], gate_up, down), (rows, counts[:, 0], gate_up, down),
                 (rows, counts, gate_up[:2], down[:2]), (rows, counts, gate_up.half(), down.half()), (rows, counts, down, gate_up),
                 (rows, counts, gate_up, down, rows[:, :, :4]), (rows, counts, gate_up, down, rows.half()), (inside, counts, gate_up, down, shifted),
                 (rows, counts.cpu(), gate_up, down), (rows[:, :, :0], counts, gate_up, down)):
        with pytest.raises(_lib.A2AError):
            expert_mlp(*args)
