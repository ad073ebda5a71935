"""A logit of -inf excludes an expert as long as others are there, also where a bias of -inf keeps those back."""
import pytest
import torch

from gpu_mode_kernels_b200.moe import topk_gate

DEV = "cuda:0"
INF = float("inf")


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_excluded_experts_come_behind_those_that_a_bias_keeps_back(score, dtype):
    logits, bias = torch.zeros(3, 70, dtype=dtype), torch.full((70,), -INF)
    logits[:, :40] = -INF
    bias[50], bias[3] = 0.0, 5.0
    logits[1, 50] = -INF
    logits[2] = -INF
    idx, w = topk_gate(logits.to(DEV), 4, score=score, bias=bias.to(DEV))
    # the one with a bias, then those that are left, in order; where none are left, the excluded ones, in order
    assert idx.tolist() == [[50, 40, 41, 42], [40, 41, 42, 43], [0, 1, 2, 3]]
    assert w.tolist() == [[0.25] * 4] * 2 + [[0.0] * 4]
