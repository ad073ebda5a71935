"""Weights of scores that are next to nothing: renormalized ones are the ratio of the scores, however small these are."""
import pytest
import torch

from gpu_mode_kernels_b200.moe import topk_gate
from tests import product_oracle as O

DEV = "cuda:0"
INF = float("inf")


def ratios(logits, indices, score):
    """Renormalized weights in 64 bits, from the logarithms of the scores."""
    l = logits.double()
    logs = torch.log_softmax(l, 1) if score == "softmax" else torch.nn.functional.logsigmoid(l)
    return torch.softmax(logs.gather(1, indices.long()), 1).nan_to_num()


def check_gate(logits, k, score, bias=None, scale=1.0, atol=0.0):
    indices, weights = topk_gate(logits.to(DEV), k, score=score, bias=None if bias is None else bias.to(DEV), scale=scale)
    order, _ = O.gate(logits, logits.shape[1], score, bias, True, 1.0)
    # an expert of -inf is behind all others, also behind those whose score is 0 in 64 bits
    out = logits.gather(1, order.long()) == -INF
    want = order.gather(1, out.sort(dim=1, stable=True).indices)[:, :k]
    assert torch.equal(indices.cpu(), want)
    # 64 bits until the end: one rounding to fp32, half a step of 2^-23, and half its smallest value; the logarithms here are off by |logit| 2^-52
    torch.testing.assert_close(weights.cpu().double(), ratios(logits, want, score) * scale, rtol=2.0 ** -23, atol=max(atol, 2.0 ** -149) * scale)
    return weights.cpu()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("level", [-75.0, -90.0, -104.0, -200.0, -600.0, -1000.0, -30000.0])
@pytest.mark.parametrize("experts,k", [(8, 3), (64, 6), (300, 32)])
def test_sigmoids_of_low_logits(dtype, level, experts, k):
    g = torch.Generator().manual_seed(int(-level))
    logits = (level + 2 * torch.randn(9, experts, generator=g)).to(dtype)
    check_gate(logits, k, "sigmoid")
    check_gate(logits, k, "sigmoid", torch.zeros(experts), scale=2.5)


@pytest.mark.gpu
def test_equal_logits_share_equally_and_both_forms_agree():
    for level in (-89.0, -90.0, -120.0, -800.0, -1e30, torch.finfo(torch.float32).min):
        logits = torch.full((3, 40), level)
        for bias in (None, torch.zeros(40)):
            assert check_gate(logits, 4, "sigmoid", bias).tolist() == [[0.25] * 4] * 3


@pytest.mark.gpu
def test_one_high_score_beside_low_ones():
    """Scores below fp32's range weigh nothing next to a sum that is above 2^-64: they are off by less than 2^-126 / 2^-64."""
    for top in (-30.0, -44.0, -45.0, -50.0, -88.0, 3.0):
        logits = torch.full((2, 20), -100.0) - torch.arange(20.0)
        logits[:, 7] = top
        check_gate(logits, 3, "sigmoid", atol=2.0 ** -62)
        check_gate(logits, 3, "sigmoid", torch.zeros(20))


@pytest.mark.gpu
def test_nothing_and_next_to_nothing():
    logits = torch.full((3, 33), -INF)
    logits[1, 30], logits[1, 4] = -100.0, -101.0
    logits[2, 9] = -5000.0
    for bias in (None, torch.zeros(33)):
        w = check_gate(logits, 3, "sigmoid", bias)
        assert w[0].tolist() == [0.0] * 3 and w[1, 2] == 0.0 and w[2].tolist() == [1.0, 0.0, 0.0]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("level", [-100.0, -700.0, -900.0, -5000.0])
def test_softmax_of_experts_that_the_bias_alone_has_chosen(dtype, level):
    g = torch.Generator().manual_seed(int(-level))
    logits = level + 2 * torch.randn(5, 70, generator=g)
    logits[:, 3] = 0.0
    bias = torch.full((70,), 10.0)
    bias[3] = 0.0
    check_gate(logits.to(dtype), 6, "softmax", bias)


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_scores_themselves_stay_as_they_are(score):
    """Without renormalize a weight is the score, rounded to fp32: 0 below its range."""
    logits = torch.full((2, 12), -200.0)
    logits[1] = torch.arange(12.0) - 60
    s = torch.softmax(logits.double(), 1) if score == "softmax" else torch.sigmoid(logits.double())
    for bias in (None, torch.zeros(12)):
        idx, w = topk_gate(logits.to(DEV), 4, score=score, renormalize=False, bias=None if bias is None else bias.to(DEV))
        torch.testing.assert_close(w.cpu().double(), s.gather(1, idx.cpu().long()), rtol=2.0 ** -18, atol=1e-38)
