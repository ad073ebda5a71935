"""Pairs of blocks in the products over experts: what each copies, roles that nothing may leave behind, experts of few rows with long sums."""
import ctypes as C
import os
import random
import subprocess

import pytest
import torch

from gpu_mode_kernels_b200.linear import check
from gpu_mode_kernels_b200.moe import expert_mlp
from tests import product_oracle as O
from tests.pair_model import Pair

DEV = "cuda:0"
CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gpu-mode-kernels_b200", "csrc")
SIDES = (0, 1)
ROLES = [("products", 0)] + [(role, side) for role in ("weights", "rows", "lists", "epilogue") for side in SIDES]


@pytest.fixture(scope="module")
def shares(tmp_path_factory):
    """(columns of a tile, block) -> (columns it copies, first of them, rows of its boxes), by the kernel's own functions."""
    where = tmp_path_factory.mktemp("shares")
    source, library = where / "shares.cpp", where / "shares.so"
    source.write_text('#include "product_shares.h"\n'
                      'extern "C" int columns(int n, int product, int of, int* from) { return copied_columns(n, product, 2, of, from); }\n'
                      'extern "C" int rows(int n) { return boxed_rows(n); }\n')
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-I", CSRC, "-o", str(library), str(source)], check=True)
    lib = C.CDLL(str(library))

    def of(columns, side):
        first = C.c_int()
        n = lib.columns(columns, (columns + 31) // 32 * 32, side, C.byref(first))
        return n, first.value, lib.rows(n)

    return of


def test_both_blocks_of_a_pair_copy_rows_of_every_tile(shares):
    for columns in range(1, 257):
        share = (columns + 31) // 32 * 16
        end = 0
        for side in SIDES:
            n, first, rows = shares(columns, side)
            assert n % 8 == 0 and 8 <= n <= share and first == side * share and n <= rows < n + 64
            end = max(end, min(first + n, (columns + 7) // 8 * 8))
        assert end >= columns


@pytest.mark.parametrize("up", [True, False], ids=["first product", "second product"])
@pytest.mark.parametrize("stages,steps", [(1, 1), (2, 3), (3, 6), (4, 17), (12, 1)])
def test_no_role_is_left_behind(shares, up, stages, steps):
    """Tiles of all widths, among them ones whose columns are all the first block's."""
    rng = random.Random(f"{up} {stages} {steps}")
    for slow in [()] + [(role,) for role in ROLES] + [(("rows", 1), ("lists", 1))]:
        for _ in range(3):
            widths = [rng.choice([1, 3, 8, 16, 17, 24, 40, 100, 256]) for _ in range(30)]
            tiles = [tuple(shares(n, side)[2] for side in SIDES) for n in widths]
            assert Pair(tiles, stages, steps, up).run(rng, slow) == [], (widths, slow)


@pytest.mark.parametrize("up", [True, False], ids=["first product", "second product"])
def test_a_role_whose_bytes_nobody_waits_for_is_left_behind(up):
    """The model shows the fault that the second block's share of nothing had."""
    left = Pair([(8, 0)] * 60, 3, 6, up).run(random.Random(1), [("rows", 1)])
    assert ("rows", 1) in left and (("products", 0) in left) == up


def generator(*seed):
    return torch.Generator(device=DEV).manual_seed(hash(seed) & 0xffffffff)


def check_slabs(counts, base, hidden, inner, experts, g, dtype=torch.bfloat16):
    """`experts` experts, of which `base` differ, on slabs of counts.max() rows; expert e is the (e % base)-th of them."""
    capacity, world = int(counts.max()), counts.shape[0]
    up = torch.empty(base, 2 * inner, hidden, dtype=dtype, device=DEV).normal_(0, hidden ** -0.5, generator=g)
    down = torch.empty(base, hidden, inner, dtype=dtype, device=DEV).normal_(0, inner ** -0.5, generator=g)
    rows = torch.empty(experts, world, capacity, hidden, dtype=dtype, device=DEV).normal_(0, 1, generator=g)
    given = torch.zeros(world, 4, experts, dtype=torch.int32, device=DEV)
    given[:, 0] = counts.to(DEV)
    valid = torch.arange(capacity, device=DEV) < given[:, 0].t()[..., None]
    rows[~valid] = float("nan")
    many = experts // base
    weights = up.repeat(many, 1, 1), down.repeat(many, 1, 1)
    out = torch.full_like(rows, 3.0)
    assert expert_mlp(rows, given, *weights, out=out) is out
    check()
    assert bool((out[~valid] == 3.0).all())
    for e in range(base):
        mine = torch.zeros_like(valid)
        mine[e::base] = valid[e::base]
        value, bound = O.expert(rows[mine], up[e], down[e], dtype)
        O.assert_within(out[mine], value.cpu(), O.rounded(value, bound, dtype).cpu(), f"experts {e} of {base}")
    return rows, given, weights, out


@pytest.mark.gpu
@pytest.mark.parametrize("hidden,inner", [(1032, 648), (520, 1288)])
@pytest.mark.parametrize("most", [1, 16, 17, 40])
def test_experts_of_few_rows_with_long_sums_and_more_tiles_than_a_table_holds(hidden, inner, most):
    """1024 experts of up to `most` rows: 40 to 150 tiles a pair, of sums that take the ring several times round, with columns of one block alone and of
    both in turn."""
    g = generator(hidden, inner, most)
    counts = torch.randint(1, most + 1, (1, 1024), generator=torch.Generator().manual_seed(most))
    check_slabs(counts, 16, hidden, inner, 1024, g)


@pytest.mark.gpu
@pytest.mark.parametrize("world", [1, 3, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_experts_of_few_rows_beside_experts_of_many(world, dtype):
    """Slabs of nothing, of a few rows and of hundreds: tiles of 256 columns whose last ones are narrow. The same bits every time."""
    g, h = generator(world), torch.Generator().manual_seed(world)
    counts = torch.randint(0, 17, (world, 64), generator=h)
    counts[torch.rand(world, 64, generator=h) < 0.15] = 290
    counts[:, 5], counts[-1, 9] = 0, 300
    rows, given, weights, out = check_slabs(counts, 8, 776, 328, 64, g, dtype)
    for _ in range(10):
        assert torch.equal(expert_mlp(rows, given, *weights, out=torch.full_like(out, 3.0)).view(torch.int16), out.view(torch.int16))
    check()


@pytest.mark.gpu
def test_experts_of_a_decode_batch():
    """A few rows for each of a layer's experts, the least one a source and the most sixteen."""
    for most in (1, 16):
        counts = torch.randint(1, most + 1, (4, 32), generator=torch.Generator().manual_seed(most))
        check_slabs(counts, 32, 4096, 1280, 32, generator(most, 3))
