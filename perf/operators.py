"""The calls that a program makes of the mixture-of-experts layer around the all-to-all: the gate that chooses the
experts, the experts' own products, and the dense products beside them.

Four operators, each in a plain form (torch operations in 32 bits, in 64 where a choice hangs on them) and as the
framework's call:

``gate``     ``moe.topk_gate``: the k experts of every token and their weights, from the router's logits.
``layer``    ``moe.moe_layer``: a whole layer for a few tokens on one GPU, from (x, indices, weights) to the output.
``experts``  ``moe.expert_mlp``: the products of the experts on the rows that a dispatch has left in their buffers.
``linear``   ``linear.linear``: a dense product with bias, activation and residual in its epilogue.

Sizes are those of ``cases.py``'s expert layouts with an inner size of the experts added to each, one token to a prefill
batch of 2048, ragged token counts and outputs.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}

# (experts, top-k, hidden, inner size of an expert); the first three as they occur in cases.py
LAYOUTS = [(8, 2, 6144, 4096), (8, 2, 2048, 4096), (64, 6, 2048, 1024), (128, 4, 2880, 1440), (128, 8, 4096, 1280),
           (256, 8, 7168, 1024)]


def _gate(name, tokens, experts, topk, dtype="fp32", score="softmax", bias=False, renormalize=True, scale=1.0):
    case = dict(op="gate", tokens=tokens, experts=experts, topk=topk, dtype=dtype, score=score, bias=bias,
                renormalize=renormalize, scale=scale)
    return dict(case, name=name) if name else case


def _layer(name, layout, tokens, dtype="bf16", routing="uniform", residual=False):
    experts, topk, hidden, inner = layout
    case = dict(op="layer", experts=experts, topk=topk, hidden=hidden, inner=inner, tokens=tokens, dtype=dtype,
                routing=routing, residual=residual)
    return dict(case, name=name) if name else case


def _experts(name, layout, world, max_tokens, tokens, dtype="bf16", routing="uniform"):
    experts, topk, hidden, inner = layout
    case = dict(op="experts", experts=experts, topk=topk, hidden=hidden, inner=inner, world=world, max_tokens=max_tokens,
                tokens=tokens, dtype=dtype, routing=routing)
    return dict(case, name=name) if name else case


def _linear(name, tokens, inputs, outputs, dtype="bf16", out="same", activation="none", bias=False, residual=False):
    case = dict(op="linear", tokens=tokens, inputs=inputs, outputs=outputs, dtype=dtype, out=out, activation=activation,
                bias=bias, residual=residual)
    return dict(case, name=name) if name else case


def listed():
    return [
        # the router of one token being decoded: nothing but latency
        _gate("gate_one_token", 1, 64, 6, dtype="fp16"),
        # the router of a prefill batch: sigmoid scores, a correction of the choice for each expert, scaled weights
        _gate("gate_prefill", 2048, 256, 8, score="sigmoid", bias=True, scale=2.5),
        # one token being decoded through small experts
        _layer("layer_one_token", (64, 6, 2048, 1024), 1, dtype="fp16"),
        # a handful of sequences through the layout of the headline workload; almost every pair has an expert of its own
        _layer("layer_few_tokens", (256, 8, 7168, 1024), 7, residual=True),
        # a decode batch that touches every expert, a few tokens each
        _layer("layer_decode_batch", (128, 8, 4096, 1280), 64),
        # the largest batch for one GPU, ragged, few large experts
        _layer("layer_large_experts", (8, 2, 6144, 4096), 173, dtype="fp16"),
        # one rank's experts after a dispatch of four ranks with ragged batches
        _experts("experts4_ragged", (128, 8, 4096, 1280), 4, 128, 117),
        # one rank's experts after a dispatch of eight ranks, skewed popularity: full slabs beside empty ones
        _experts("experts8_skewed", (64, 6, 2048, 1024), 8, 256, 256, routing="zipf"),
        # the router's logits of a decode batch: few outputs, a long sum, 32-bit result
        _linear("linear_router_logits", 16, 7168, 256, out="fp32"),
        # an output projection of one decoded token with its residual
        _linear("linear_one_token", 1, 4096, 7168, residual=True),
        # a ragged batch with odd sizes, bias and GELU
        _linear("linear_ragged", 93, 2880, 2879, dtype="fp16", activation="gelu", bias=True),
        # a shared expert's gate and up projection in prefill
        _linear("linear_shared_expert_prefill", 2048, 7168, 2048, activation="swiglu"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["gate", "gate", "layer", "layer", "layer", "experts", "experts", "linear", "linear", "linear"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "gate":
        experts, topk = rng.choice([(8, 2), (64, 6), (128, 4), (128, 8), (256, 8), (rng.randint(33, 384), rng.randint(1, 16))])
        return _gate(None, _log_int(rng, 1, 2048), experts, topk, dtype=rng.choice(["fp32", "bf16", "fp16"]),
                     score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.4, renormalize=rng.random() < 0.7,
                     scale=rng.choice([1.0, 2.5]))
    if op == "linear":
        while True:
            tokens = _log_int(rng, 1, 2048)
            inputs = rng.choice([2048, 2880, 4096, 6144, 7168, 8 * rng.randint(64, 896)])
            outputs = rng.choice([256, 1024, 2048, 2880, 4096, 7168, rng.randint(129, 7168)])
            activation = rng.choice(["none", "none", "relu", "gelu", "silu", "swiglu"])
            if tokens * inputs * outputs * (2 if activation == "swiglu" else 1) <= 2048 * 7168 * 4096:
                return _linear(None, tokens, inputs, outputs, dtype=dtype, out="fp32" if rng.random() < 0.25 else "same",
                               activation=activation, bias=rng.random() < 0.4, residual=rng.random() < 0.4)
    while True:
        experts, topk, hidden, inner = rng.choice(LAYOUTS)
        if rng.random() < 0.3:
            inner = 8 * rng.randint(64, inner // 8)
        layout, skew = (experts, topk, hidden, inner), "zipf" if experts >= 64 and rng.random() < 0.25 else "uniform"
        if op == "layer":
            case = _layer(None, layout, _log_int(rng, 1, 256), dtype=dtype, routing=skew, residual=rng.random() < 0.3)
        else:
            world, max_tokens = rng.choice([1, 2, 4, 8]), _log_int(rng, 1, 256)
            case = _experts(None, layout, world, max_tokens, rng.randint((max_tokens + 1) // 2, max_tokens), dtype=dtype,
                            routing=skew)
        cost = work(case)
        if cost["bytes"] <= 4.1e9 and cost["flops"] <= 1.2e11:
            return case


def _generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def _normal(gen, *shape, std=1.0, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device="cuda").normal_(0, std, generator=gen)


def _choose(gen, tokens, experts, topk, routing):
    """Distinct experts for every token: the largest of independent keys (Gumbel keys where popularity is skewed)."""
    keys = torch.rand(tokens, experts, generator=gen, device="cuda")
    if routing == "zipf":
        popularity = -1.2 * torch.log(torch.arange(1, experts + 1, device="cuda", dtype=torch.float32))
        keys = popularity - torch.log(-torch.log(keys.clamp(1e-7, 1 - 1e-6)))
    return keys.topk(topk, dim=1).indices.to(torch.int32).contiguous()


def _local_experts(case):
    """A rank's experts; the first rank's, which skewed routing likes best."""
    return case["experts"] // case["world"]


def prepare(case, seed):
    gen, op, dtype = _generator(seed), case["op"], DTYPES[case["dtype"]]
    if op == "gate":
        logits = _normal(gen, case["tokens"], case["experts"]).to(dtype)
        bias = _normal(gen, case["experts"], std=0.05) if case["bias"] else None
        return case, (logits, bias)
    if op == "linear":
        n, k = case["outputs"], case["inputs"]
        rows = 2 * n if case["activation"] == "swiglu" else n
        out = dtype if case["out"] == "same" else DTYPES[case["out"]]
        x, weight = _normal(gen, case["tokens"], k, dtype=dtype), _normal(gen, rows, k, std=k ** -0.5, dtype=dtype)
        bias = _normal(gen, rows, std=0.5, dtype=dtype) if case["bias"] else None
        residual = _normal(gen, case["tokens"], n, dtype=out) if case["residual"] else None
        return case, (x, weight, bias, residual, out)
    hidden, inner = case["hidden"], case["inner"]
    held = case["experts"] if op == "layer" else _local_experts(case)
    gate_up = _normal(gen, held, 2 * inner, hidden, std=hidden ** -0.5, dtype=dtype)
    down = _normal(gen, held, hidden, inner, std=inner ** -0.5, dtype=dtype)
    if op == "layer":
        tokens = case["tokens"]
        x = _normal(gen, tokens, hidden, dtype=dtype)
        indices = _choose(gen, tokens, case["experts"], case["topk"], case["routing"])
        weights = torch.softmax(_normal(gen, tokens, case["topk"]), dim=-1)
        residual = _normal(gen, tokens, hidden, dtype=dtype) if case["residual"] else None
        return case, (x, indices, weights, gate_up, down, residual)
    # what a dispatch leaves: rows [local experts, source rank, capacity, hidden], valid rows of each slab in counts
    # [source rank, 4, local experts] (entry 0 with one chunk); behind them whatever an earlier call left there
    world, capacity = case["world"], case["max_tokens"]
    rows = _normal(gen, held, world, capacity, hidden, dtype=dtype)
    counts = torch.zeros(world, 4, held, dtype=torch.int32, device="cuda")
    chosen = _choose(gen, world * case["tokens"], case["experts"], case["topk"], case["routing"]).view(world, -1)
    counts[:, 0] = (chosen[:, :, None] == torch.arange(held, device="cuda")).sum(1)
    return case, (rows, counts, gate_up, down, torch.zeros_like(rows))


def _silu(x):
    return x / (1 + torch.exp(-x))


def _act(y, activation):
    if activation == "relu":
        return y.clamp_min(0)
    if activation == "gelu":
        return 0.5 * y * (1 + torch.erf(y * 0.5 ** 0.5))
    if activation == "silu":
        return _silu(y)
    if activation == "swiglu":
        gate, up = y.chunk(2, dim=-1)
        return _silu(gate) * up
    return y


def _plain_gate(case, logits, bias):
    # in 64 bits: which of two near scores is the larger decides an expert
    l = logits.double()
    if case["score"] == "softmax":
        e = torch.exp(l - l.max(dim=1, keepdim=True).values)
        scores = e / e.sum(dim=1, keepdim=True)
    else:
        scores = 1 / (1 + torch.exp(-l))
    order = (l if bias is None else scores + bias.double()).sort(dim=1, descending=True, stable=True).indices
    indices = order[:, :case["topk"]]
    weights = scores.gather(1, indices)
    if case["renormalize"]:
        weights = weights / weights.sum(dim=1, keepdim=True)
    return indices.to(torch.int32), (weights * case["scale"]).float()


def _plain_layer(x, indices, weights, gate_up, down, residual):
    tokens, topk = indices.shape
    experts = gate_up.shape[0]
    if tokens * topk <= experts:
        # the chosen experts' weights, pair by pair
        pairs = indices.reshape(-1).long()
        xs = x.float().repeat_interleave(topk, dim=0)[:, :, None]
        h = _act(torch.bmm(gate_up[pairs].float(), xs)[:, :, 0], "swiglu")
        rows = torch.bmm(down[pairs].float(), h[:, :, None])[:, :, 0].view(tokens, topk, -1)
        y = (rows * weights[:, :, None]).sum(1)
    else:
        # every token through every expert, weighted with zero where the expert was not chosen
        share = (weights[:, :, None] * (indices[:, :, None] == torch.arange(experts, device=x.device))).sum(1)
        h = _act(torch.matmul(x.float(), gate_up.float().transpose(1, 2)), "swiglu")
        y = torch.bmm(h * share.t()[:, :, None], down.float().transpose(1, 2)).sum(0)
    return (y if residual is None else y + residual.float()).to(x.dtype)


def _plain_experts(rows, counts, gate_up, down, out):
    held, world, capacity, hidden = rows.shape
    x = rows.view(held, world * capacity, hidden).float()
    h = _act(torch.bmm(x, gate_up.float().transpose(1, 2)), "swiglu")
    y = torch.bmm(h, down.float().transpose(1, 2)).view_as(rows).to(rows.dtype)
    valid = torch.arange(capacity, device=rows.device) < counts[:, 0].t()[:, :, None]
    out.copy_(torch.where(valid[..., None], y, out))
    return out


def _plain_linear(case, x, weight, bias, residual, out):
    y = x.float() @ weight.float().t()
    if bias is not None:
        y = y + bias.float()
    y = _act(y, case["activation"])
    return (y if residual is None else y + residual.float()).to(out)


def run(state):
    case, what = state
    op = case["op"]
    if own:
        from gpu_mode_kernels_b200.linear import linear
        from gpu_mode_kernels_b200.moe import expert_mlp, moe_layer, topk_gate
        if op == "gate":
            logits, bias = what
            return topk_gate(logits, case["topk"], score=case["score"], bias=bias, renormalize=case["renormalize"],
                             scale=case["scale"])
        if op == "layer":
            x, indices, weights, gate_up, down, residual = what
            return moe_layer(x, indices, weights, gate_up, down, residual=residual)
        if op == "experts":
            rows, counts, gate_up, down, out = what
            return expert_mlp(rows, counts, gate_up, down, out=out)
        x, weight, bias, residual, out = what
        return linear(x, weight, bias, activation=case["activation"], residual=residual, out_dtype=out)
    if op == "gate":
        return _plain_gate(case, *what)
    if op == "layer":
        return _plain_layer(*what)
    if op == "experts":
        return _plain_experts(*what)
    return _plain_linear(case, *what)


def exact(case, seed):
    _, what = prepare(case, seed)
    op = case["op"]
    if op == "gate":
        logits, bias = what
        l = logits.double()
        scores = torch.softmax(l, dim=1) if case["score"] == "softmax" else torch.sigmoid(l)
        indices = torch.argsort(l if bias is None else scores + bias.double(), dim=1, descending=True, stable=True)
        weights = torch.gather(scores, 1, indices[:, :case["topk"]])
        if case["renormalize"]:
            weights = weights / weights.sum(1, keepdim=True)
        return None, weights * case["scale"]
    if op == "linear":
        x, weight, bias, residual, _ = what
        y = torch.nn.functional.linear(x.double(), weight.double(), None if bias is None else bias.double())
        if case["activation"] == "swiglu":
            y = torch.nn.functional.silu(y[:, :case["outputs"]]) * y[:, case["outputs"]:]
        elif case["activation"] != "none":
            y = getattr(torch.nn.functional, case["activation"])(y)
        return y if residual is None else y + residual.double()

    def expert(rows, e, gate_up, down):
        gate, up = (rows.double() @ gate_up[e].double().t()).split(case["inner"], dim=1)
        return (torch.nn.functional.silu(gate) * up) @ down[e].double().t()

    if op == "layer":
        x, indices, weights, gate_up, down, residual = what
        y = torch.zeros(x.shape, dtype=torch.float64, device=x.device) if residual is None else residual.double()
        for e in range(case["experts"]):
            token, k = (indices == e).nonzero(as_tuple=True)
            if token.numel():
                y.index_add_(0, token, expert(x[token], e, gate_up, down) * weights[token, k, None].double())
        return y
    rows, counts, gate_up, down, out = what
    y = out.double()
    for e in range(rows.shape[0]):
        for s in range(case["world"]):
            n = int(counts[s, 0, e])
            if n:
                y[e, s, :n] = expert(rows[e, s, :n], e, gate_up, down)
    return y


def _used(case, tokens, held):
    """Experts that get a row, on average: each token takes topk of them; skewed routing counts as uniform."""
    return held * (1 - (1 - case["topk"] / case["experts"]) ** tokens)


def work(case):
    op = case["op"]
    if op == "gate":
        size = case["tokens"] * case["experts"]
        return {"bytes": size * DTYPES[case["dtype"]].itemsize + case["tokens"] * case["topk"] * 8, "flops": 4 * size}
    if op == "linear":
        m, n, k = case["tokens"], case["outputs"], case["inputs"]
        rows = 2 * n if case["activation"] == "swiglu" else n
        size = 2 if case["out"] == "same" else 4
        return {"bytes": 2 * (m * k + rows * k + (rows if case["bias"] else 0)) + m * n * size * (2 if case["residual"] else 1),
                "flops": 2 * m * rows * k}
    hidden, inner, topk = case["hidden"], case["inner"], case["topk"]
    if op == "layer":
        tokens = case["tokens"]
        rows, used = tokens * topk, _used(case, tokens, case["experts"])
        moved = 2 * tokens * hidden * (3 if case["residual"] else 2) + 8 * rows
    else:
        tokens, held = case["tokens"] * case["world"], _local_experts(case)
        rows, used = tokens * topk / case["world"], _used(case, tokens, held)
        moved = 2 * 2 * rows * hidden + 4 * held * case["world"]
    return {"bytes": round(moved + used * 3 * inner * hidden * 2), "flops": round(6 * rows * inner * hidden)}
