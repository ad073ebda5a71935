"""Calls that a program may make of the layer and its experts, and that are easily got wrong: padded batches, several at once, replayed ones."""
import pytest
import torch

from gpu_mode_kernels_b200.linear import check
from gpu_mode_kernels_b200.moe import expert_mlp, moe_layer
from tests import product_oracle as O

DEV = "cuda:0"


def normal(g, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=g) * std).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [65, 130, 256])
@pytest.mark.parametrize("E,k", [(16, 5), (300, 32)])
def test_pads_and_repeats_among_many_tokens(tokens, E, k):
    """More tokens than go without a sort: pairs without an expert leave no row between the others."""
    g = torch.Generator().manual_seed(tokens * E)
    hidden, inner = 136, 72
    gate_up, down = normal(g, E, 2 * inner, hidden, std=hidden ** -0.5), normal(g, E, hidden, inner, std=inner ** -0.5)
    x, w, residual = normal(g, tokens, hidden), torch.randn(tokens, k, generator=g), normal(g, tokens, hidden)
    idx = torch.randint(-3, E + 3, (tokens, k), generator=g, dtype=torch.int32)
    idx[0], idx[-1], idx[7] = -1, E, 3
    idx[20:40] = torch.tensor([-(1 << 31), 1 << 30], dtype=torch.int32).repeat(16)[:k]
    y = moe_layer(*(t.to(DEV) for t in (x, idx, w, gate_up, down)), residual=residual.to(DEV))
    O.assert_within(y, *O.layer(x, idx, w, gate_up, down, residual))
    assert torch.equal(y[-1].cpu(), residual[-1]) and torch.equal(y[20:40].cpu(), residual[20:40])
    y = moe_layer(*(t.to(DEV) for t in (x, torch.full_like(idx, -1), w, gate_up, down)))
    assert not bool(y.any())
    check()


@pytest.mark.gpu
def test_experts_of_few_rows_at_once_and_replayed():
    """Slabs of 1 to 16 rows on two streams at the same time, as calls and as graphs, on counts that change from replay to replay."""
    g = torch.Generator(device=DEV).manual_seed(1)
    E, world, capacity, hidden, inner = 96, 2, 16, 1032, 328
    up = torch.empty(E, 2 * inner, hidden, dtype=torch.bfloat16, device=DEV).normal_(0, hidden ** -0.5, generator=g)
    down = torch.empty(E, hidden, inner, dtype=torch.bfloat16, device=DEV).normal_(0, inner ** -0.5, generator=g)
    rows = [torch.empty(E, world, capacity, hidden, dtype=torch.bfloat16, device=DEV).normal_(0, 1, generator=g) for _ in range(2)]
    given = [torch.randint(0, 9, (world, 4, E), dtype=torch.int32, device=DEV, generator=g) for _ in range(3)]
    counts, streams = [c.clone() for c in given[:2]], [torch.cuda.Stream() for _ in range(2)]
    want = [[expert_mlp(r, c, up, down, out=torch.zeros_like(r)) for c in given] for r in rows]
    out = [torch.zeros_like(r) for r in rows]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                expert_mlp(rows[i], counts[i], up, down, out=out[i])
    torch.cuda.synchronize()
    assert all(torch.equal(out[i], want[i][i]) for i in range(2))
    graphs = []
    for i, s in enumerate(streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out[i].zero_()
            expert_mlp(rows[i], counts[i], up, down, out=out[i])
        graphs.append(graph)
    for c in (2, 0, 1):
        for i in range(2):
            counts[i].copy_(given[c])
        torch.cuda.synchronize()
        for _ in range(5):
            for s, graph in zip(streams, graphs):
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out[i], want[i][c]) for i in range(2))
    check()
