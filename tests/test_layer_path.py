"""The gate, the products and the all-to-all together, as a model's layer runs them; streams, graphs, other devices, calls back to back."""
import os
import subprocess
import sys
import threading

import pytest
import torch

import gpu_mode_kernels_b200 as pkg
from gpu_mode_kernels_b200 import _lib
from gpu_mode_kernels_b200.all2all import A2AContext
from gpu_mode_kernels_b200.linear import check, linear
from gpu_mode_kernels_b200.local_world import LocalWorld
from gpu_mode_kernels_b200.moe import expert_mlp, moe_layer, route, topk_gate
from tests import product_oracle as O

DEV = "cuda:0"


def bits(t):
    return t.contiguous().view(torch.int16 if t.element_size() == 2 else torch.int32)


def normal(g, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=g) * std).to(dtype)


class Weights:
    """A layer: router, experts and a shared expert, on the host and on the GPU."""

    def __init__(self, seed, E, hidden, inner, dtype=torch.bfloat16):
        g = torch.Generator().manual_seed(seed)
        self.router = normal(g, E, hidden, std=hidden ** -0.5, dtype=dtype)
        self.gate_up, self.down = normal(g, E, 2 * inner, hidden, std=hidden ** -0.5, dtype=dtype), normal(g, E, hidden, inner, std=inner ** -0.5, dtype=dtype)
        self.shared_up, self.shared_down = normal(g, 2 * inner, hidden, std=hidden ** -0.5, dtype=dtype), normal(g, hidden, inner, std=inner ** -0.5, dtype=dtype)

    def to(self, device):
        out = object.__new__(Weights)
        out.__dict__ = {k: v.to(device) for k, v in self.__dict__.items()}
        return out


def layer(w, x, k):
    """x + shared expert + routed experts, from the rows alone."""
    indices, weights = route(x, w.router, k, score="sigmoid", scale=1.5)
    shared = linear(linear(x, w.shared_up, activation="swiglu"), w.shared_down, residual=x)
    return moe_layer(x, indices, weights, w.gate_up, w.down, residual=shared), indices, weights


def test_without_the_compiled_part_calls_go_on_in_python():
    assert _lib.Interpreted.gate(None) is _lib.Interpreted.linear(None) is _lib.Interpreted.layer(None) is None


def test_experts_are_refused_where_the_phases_do_not_hand_over_rows(monkeypatch):
    for schedule, chunks in (("pipelined", 1), ("phased", 2)):
        c = object.__new__(A2AContext)
        c.schedule, c._chunked = schedule, chunks > 1
        with pytest.raises(_lib.A2AError) as e:
            A2AContext.experts(c, None, None)
        assert e.value.code == _lib.A2A_ERR_STATE


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 7, 65, 200])
def test_a_whole_layer(tokens):
    E, k, hidden, inner = 24, 4, 256, 104
    w = Weights(tokens, E, hidden, inner)
    x = normal(torch.Generator().manual_seed(tokens), tokens, hidden)
    y, indices, weights = layer(w.to(DEV), x.to(DEV), k)
    check()
    # the choice, by logits that the bound allows: each chosen logit is among the k largest, up to twice the bound
    logits, off = O.product(x, w.router)
    rank = logits.sort(dim=1, descending=True).values[:, k - 1:k]
    picked = logits.gather(1, indices.cpu().long())
    assert bool((picked + 2 * off.amax(1, keepdim=True) >= rank).all())
    # the rest from what was chosen; the inner values and the shared expert's output are rounded on the way
    h, dh = O.swiglu(*O.product(x, w.shared_up))
    dh = O.rounded(h, dh, x.dtype)
    s, ds = O.product(h, w.shared_down)
    s, ds = s + x.double(), ds * 1.01 + dh @ w.shared_down.double().abs().t()
    ds = O.rounded(s, ds + 2.0 ** -23 * (s.abs() + x.double().abs()), x.dtype)
    value, bound = O.layer(x, indices.cpu(), weights.cpu(), w.gate_up, w.down, s)
    O.assert_within(y, value, bound + ds * (1 + O.half_step(x.dtype)))


@pytest.mark.gpu
@pytest.mark.parametrize("world,payload,T,routing", [(1, "direct", 40, "uniform"), (2, "direct", 24, "zipf"), (2, "dedup", 31, "uniform"), (4, "direct", 9, "uniform"),
                                                     (8, "dedup", 40, "zipf")])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_experts_between_dispatch_and_combine(world, payload, T, routing, dtype):
    """Rows go to the ranks of their experts, through real experts there and back: the same as a layer on one GPU."""
    E, k, hidden, inner = 16, 3, 264, 72
    w = Weights(world, E, hidden, inner, dtype).to(DEV)
    datas = [pkg.generate_input(E, k, hidden, T, seed=71, rank=r, world_size=world, dtype=dtype, routing=routing, ragged=True) for r in range(world)]
    rds, L = [d[1].to(DEV) for d in datas], E // world
    group = LocalWorld(datas[0][0], world, payload=payload)
    try:
        for again in range(2):
            ys = group.forward_phases(rds, experts=[(w.gate_up[r * L:(r + 1) * L], w.down[r * L:(r + 1) * L]) for r in range(world)])
            torch.cuda.synchronize()
            group.check()
            for y, rd in zip(ys, rds):
                value, bound = O.layer(rd.x.cpu(), rd.indices.cpu(), rd.weights.cpu(), w.gate_up.cpu(), w.down.cpu(), None)
                # an expert's row is rounded once more on the way home: half a step of each row, weighted
                extra = torch.zeros_like(value)
                for j in range(k):
                    v, d = zip(*[O.expert(rd.x[t:t + 1].cpu(), w.gate_up[int(e)].cpu(), w.down[int(e)].cpu(), dtype) for t, e in enumerate(rd.indices[:, j])])
                    row = torch.cat(v)
                    extra += rd.weights[:, j:j + 1].cpu().double() * O.rounded(row, torch.cat(d), dtype).sub(torch.cat(d))
                O.assert_within(y, value, bound + extra * (1 + O.half_step(dtype)))
                O.assert_within(moe_layer(rd.x, rd.indices, rd.weights, w.gate_up, w.down), value, bound)
        with pytest.raises(_lib.A2AError):
            group.forward_phases(rds, experts=[(w.gate_up, w.down)] * (world + 1))
    finally:
        group.close()
    check()


@pytest.mark.gpu
def test_experts_on_rows_that_came_as_fp8():
    """Rows of -1, 0 and 1 are themselves after eight bits with a scale for 128 values, so the layer is the one of 16-bit rows."""
    world, E, k, hidden, inner, T = 2, 8, 2, 256, 64, 17
    w = Weights(3, E, hidden, inner).to(DEV)
    datas = [pkg.generate_input(E, k, hidden, T, seed=72, rank=r, world_size=world) for r in range(world)]
    rds = [d[1].to(DEV) for d in datas]
    for rd in rds:
        rd.x = rd.x.sign()
    L, outs = E // world, []
    for payload in ("fp8", "direct"):
        group = LocalWorld(datas[0][0], world, payload=payload)
        try:
            outs.append(group.forward_phases(rds, experts=[(w.gate_up[r * L:(r + 1) * L], w.down[r * L:(r + 1) * L]) for r in range(world)]))
            torch.cuda.synchronize()
            group.check()
        finally:
            group.close()
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip(*outs))


@pytest.mark.gpu
def test_weights_written_just_before_the_call():
    """The second product has its first weights on their way before the first one is through: what the stream did before counts."""
    w = Weights(21, 16, 128, 64).to(DEV)
    g = torch.Generator().manual_seed(22)
    downs = [normal(g, 16, 128, 64).to(DEV) for _ in range(3)]
    down = downs[0].clone()
    for tokens in (1, 7, 90):
        x = normal(g, tokens, 128).to(DEV)
        idx, weights = route(x, w.router, 3)
        want = [moe_layer(x, idx, weights, w.gate_up, d) for d in downs]
        rows = normal(g, 16, 1, 40, 128).to(DEV)
        counts = torch.full((1, 4, 16), 33, dtype=torch.int32, device=DEV)
        slabs = [expert_mlp(rows, counts, w.gate_up, d, out=torch.zeros_like(rows)) for d in downs]
        torch.cuda.synchronize()
        got, on_slabs = [], []
        for i in range(30):
            down.copy_(downs[i % 3])
            got.append(moe_layer(x, idx, weights, w.gate_up, down))
            down.copy_(downs[(i + 1) % 3])
            on_slabs.append(expert_mlp(rows, counts, w.gate_up, down, out=torch.zeros_like(rows)))
        assert all(torch.equal(y, want[i % 3]) for i, y in enumerate(got))
        assert all(torch.equal(y, slabs[(i + 1) % 3]) for i, y in enumerate(on_slabs))


@pytest.mark.gpu
def test_a_first_call_may_be_a_captured_one():
    """Nothing of a call's set-up, which the first one of a process makes, is forbidden in a capture."""
    code = """
import torch
from gpu_mode_kernels_b200.linear import linear
from gpu_mode_kernels_b200.moe import moe_layer, topk_gate, expert_mlp
x, up, down = (torch.randn(*s, device="cuda").bfloat16() for s in ((80, 64), (8, 64, 64), (8, 64, 32)))
idx, w = torch.zeros(80, 2, dtype=torch.int32, device="cuda"), torch.ones(80, 2, device="cuda")
rows, counts = torch.randn(8, 1, 16, 64, device="cuda").bfloat16(), torch.full((1, 4, 8), 9, dtype=torch.int32, device="cuda")
s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
torch.cuda.synchronize()
def calls():
    return [linear(x, up[0]), linear(x.repeat(30, 1), up[0]), linear(x[:2], up[0]), *topk_gate(x.float()[:, :8].contiguous(), 2, bias=w[:4].flatten()),
            moe_layer(x, idx, w, up, down), moe_layer(x[:3], idx[:3], w[:3], up, down), expert_mlp(rows, counts, up, down, out=torch.zeros_like(rows))]
with torch.cuda.graph(g, stream=s):
    got = calls()
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, calls()))
print("alike")
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), capture_output=True, text=True, timeout=240)
    assert done.returncode == 0 and "alike" in done.stdout, done.stderr[-2000:]


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [3, 70])
def test_captured_calls_replay_on_new_inputs(tokens):
    w = Weights(5, 16, 128, 64).to(DEV)
    g = torch.Generator().manual_seed(6)
    xs = [normal(g, tokens, 128).to(DEV) for _ in range(4)]
    want = [layer(w, x, 3)[0] for x in xs]
    x = xs[0].clone()
    graphs, outs, side = [], [], torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):  # two graphs, which share the pool of their temporaries with nobody
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs.append(layer(w, x, 3)[0])
            graphs.append(graph)
    torch.cuda.current_stream().wait_stream(side)
    for i in (1, 2, 3, 1):
        x.copy_(xs[i])
        for graph, out in zip(graphs, outs):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(bits(out), bits(want[i]))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(10):  # both at once
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(bits(out), bits(want[1])) for out in outs)
    check()


@pytest.mark.gpu
def test_calls_on_several_streams_and_threads_at_once():
    w = Weights(7, 16, 128, 64).to(DEV)
    g = torch.Generator().manual_seed(8)
    xs = [normal(g, 4 + 30 * i, 128).to(DEV) for i in range(4)]
    want = [bits(layer(w, x, 3)[0]) for x in xs]
    torch.cuda.synchronize()
    wrong, streams = [], [torch.cuda.Stream() for _ in xs]

    def work(i):
        with torch.cuda.stream(streams[i]):
            got = [layer(w, xs[i], 3)[0] for _ in range(30)]
            streams[i].synchronize()
            wrong.extend(i for y in got if not torch.equal(bits(y), want[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(xs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    check()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [2, 9, 100])
def test_calls_on_each_others_outputs(tokens):
    """A launch may be resident while the one before it still writes what it reads; weights too are the output of a call just before."""
    w = Weights(9, 16, 128, 64).to(DEV)
    g = torch.Generator().manual_seed(10)
    first = normal(g, tokens, 128).to(DEV)

    def run(wait):
        x, weights = first, Weights(9, 16, 128, 64).to(DEV)
        for i in range(40):
            x, _, _ = layer(weights, x, 3)
            x = linear(x, weights.router.repeat(8, 1), activation="silu")
            if i % 5 == 2:  # another program's kernels, which change rows and weights
                x.mul_(0.5)
                weights.down.copy_(weights.down.flip(0))
                weights.gate_up.neg_()
            if wait:
                torch.cuda.synchronize()
        return bits(x)

    assert torch.equal(run(False), run(True))
    check()


@pytest.mark.gpu
def test_the_same_bits_without_the_compiled_part(monkeypatch):
    w = Weights(11, 16, 128, 64).to(DEV)
    g = torch.Generator().manual_seed(12)
    x, bias = normal(g, 19, 128).to(DEV), torch.randn(16, generator=g).to(DEV)

    def everything():
        y, idx, weights = layer(w, x, 3)
        other = topk_gate(linear(x, w.router, out_dtype=torch.float32), 2, bias=bias, renormalize=False)
        return [y, idx, weights, *other, linear(x, w.router, bias.to(x.dtype), activation="gelu"), linear(x[:1], w.router, bias, out_dtype=torch.float32)]

    assert _lib.host() is not _lib.Interpreted
    want = everything()
    monkeypatch.setattr(_lib, "_host", _lib.Interpreted)
    assert all(torch.equal(bits(a), bits(b)) and a.dtype == b.dtype for a, b in zip(everything(), want))


@pytest.mark.gpu
def test_parameters_profilers_and_scales():
    """Parameters are plain tensors here; a profiler sees the outputs; whole numbers are taken for a scale."""
    w = Weights(13, 16, 128, 64).to(DEV)
    x = normal(torch.Generator().manual_seed(14), 5, 128).to(DEV)
    want = linear(x, w.router)
    assert torch.equal(linear(x, torch.nn.Parameter(w.router)), want)
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]):
        assert torch.equal(linear(x, w.router), want)
    a, b = topk_gate(want, 2, scale=2), topk_gate(want, 2, scale=2.0)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.gpu
def test_another_device_than_the_current_one():
    if torch.cuda.device_count() < 2:
        pytest.skip("one device")
    w = Weights(15, 16, 128, 64).to("cuda:1")
    x = normal(torch.Generator().manual_seed(16), 5, 128).to("cuda:1")
    with torch.cuda.device(1):
        want = layer(w, x, 3)[0]
    torch.cuda.synchronize(1)
    with torch.cuda.device(0):
        assert torch.equal(layer(w, x, 3)[0], want)


@pytest.mark.gpu
def test_far_offsets():
    """Rows and weights whose bytes lie beyond 32 bits: experts of 5 GB, the last of them chosen; slabs of 4.5 GB."""
    g = torch.Generator(device=DEV).manual_seed(17)
    E, hidden, inner = 1024, 1024, 816
    gate_up = torch.empty(E, 2 * inner, hidden, dtype=torch.bfloat16, device=DEV).normal_(0, hidden ** -0.5, generator=g)
    down = torch.empty(E, hidden, inner, dtype=torch.bfloat16, device=DEV).normal_(0, inner ** -0.5, generator=g)
    assert gate_up.numel() * 2 > 1 << 31
    for tokens in (3, 70):
        x = torch.randn(tokens, hidden, device=DEV, generator=g).bfloat16()
        idx = torch.tensor([[1023, 1021]], dtype=torch.int32, device=DEV).repeat(tokens, 1)
        few = idx - 1020
        got, want = (moe_layer(x, i, torch.ones(tokens, 2, device=DEV), u, d) for i, u, d in ((idx, gate_up, down), (few, gate_up[1020:], down[1020:])))
        assert torch.equal(got, want)
    del gate_up, down
    local, capacity = 5, 56000
    rows = torch.empty(local, 8, capacity, hidden, dtype=torch.bfloat16, device=DEV)
    rows[4, 7] = torch.randn(capacity, hidden, device=DEV, generator=g).bfloat16()
    assert rows.numel() > 1 << 31
    counts = torch.zeros(8, 4, local, dtype=torch.int32, device=DEV)
    counts[7, 0, 4] = 37
    gate_up = torch.empty(local, 16, hidden, dtype=torch.bfloat16, device=DEV).normal_(0, hidden ** -0.5, generator=g)
    down = torch.empty(local, hidden, 8, dtype=torch.bfloat16, device=DEV).normal_(0, 8 ** -0.5, generator=g)
    before = rows[4, 7].clone()
    expert_mlp(rows, counts, gate_up, down)
    alone = before[:40].view(1, 1, 40, hidden).clone()
    expert_mlp(alone, torch.full((1, 4, 1), 37, dtype=torch.int32, device=DEV), gate_up[4:], down[4:])
    assert torch.equal(rows[4, 7, :37], alone[0, 0, :37]) and torch.equal(rows[4, 7, 37:], before[37:])
    check()
