"""Results of 32 bits: how much of a sum stays in tensor memory, whose additions are cut, and what that leaves of an error."""
import ctypes as C
import os
import re
import subprocess

import pytest
import torch

from gpu_mode_kernels_b200.linear import check, linear

DEV = "cuda:0"
CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gpu-mode-kernels_b200", "csrc")


def test_a_sum_in_tensor_memory_is_of_512_at_most(tmp_path):
    """For every size of a stage's blocks: a tile of one feature and 16 columns to one of 128 rows and 128 columns, sums of any length."""
    (tmp_path / "sums.cpp").write_text('#include "product_shares.h"\n'
                                       'extern "C" int stage(int blocks, int bytes, int of, int most) { return stage_blocks(blocks, bytes, of, most); }\n'
                                       'extern "C" int sum(int per_stage, int most) { return sum_blocks(per_stage, most); }\n')
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-I", CSRC, "-o", str(tmp_path / "sums.so"), str(tmp_path / "sums.cpp")], check=True)
    lib = C.CDLL(str(tmp_path / "sums.so"))
    tiles = open(os.path.join(CSRC, "product_tiles.cuh")).read()
    most = int(re.search(r"kSumBlocks = (\d+)", tiles).group(1))
    assert "sum_blocks(per_stage, kSumBlocks)" in tiles and "k32 ? kSumBlocks : blocks_all" in tiles and 64 * most == 512
    for weights in range(1024, 16 * 1024 + 1, 1024):
        for columns in range(16, 129, 16):
            for blocks in (1, 2, 7, 8, 9, 14, 15, 112, 1024):
                per_stage = lib.stage(blocks, weights + 128 * columns, 48 * 1024, most)
                assert 1 <= per_stage <= min(blocks, most)
                assert per_stage <= lib.sum(per_stage, most) <= most and lib.sum(per_stage, most) % per_stage == 0


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,inputs,outputs", [(16, 7168, 256), (1, 7168, 600), (3, 20000, 40), (2, 65536, 8), (1, 65536, 300), (600, 7168, 512), (70, 12000, 9)])
@pytest.mark.parametrize("activation", ["none", "swiglu"])
def test_sums_of_32_bits_do_not_drift_with_few_outputs_and_long_sums(tokens, inputs, outputs, activation):
    """A sum is cut after every 16 products, each time by up to 2^-23 of what is there, 2/3 of the end's on average. In parts of 512, 32 of them, that is 32 * 2/3 * 2^-23
    of each part; parts of signs that do not hang together have, by squares, the whole's norm, and up to 128 additions of theirs round by 2^-24 of what is there:
    by squares again sqrt(128) * 2/3 * 2^-24, half a part's. SwiGLU takes each factor's error at the other's size."""
    g = torch.Generator(device=DEV).manual_seed(tokens * inputs + outputs)
    off = (32 + 16) * 2 / 3 * 2.0 ** -23
    x = torch.randn(tokens, inputs, device=DEV, generator=g).bfloat16()
    w = (torch.randn(outputs * (2 if activation == "swiglu" else 1), inputs, device=DEV, generator=g) * inputs ** -0.5).bfloat16()
    want = x.double() @ w.double().t()
    if activation == "swiglu":
        gate, up = want.chunk(2, -1)
        s = torch.sigmoid(gate)
        want = gate * s * up
        # slope of silu times the gate's value, and silu; expf and the division are 2^-21 of the value
        allowed = off * ((s * (1 + gate * (1 - s)) * gate * up).norm() + want.norm()) + 2.0 ** -21 * want.norm()
    else:
        allowed = off * want.norm()
    assert float((linear(x, w, activation=activation, out_dtype=torch.float32).double() - want).norm()) < float(allowed)
    check()
