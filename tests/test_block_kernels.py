"""Which kernel each product of the bf16 gated MLP runs, as the library itself says (host
only): the sizes of test_gpu_block_kernels.py reach all of them, so a plan that leaves a
kernel without a test fails here."""
import pytest

import test_gpu_block_kernels as sizes
from momijo_amd import _lib

GATE, DOWN, DGATE, DX, DW = range(5)
TILES = {"256x256", "128x128", "128x64", "64x64, 3 stages", "64x64, 5 stages"}
SLICED = {t + ", K slices" for t in TILES}
KERNELS = {GATE: TILES | {"16 rows", "32 rows"}, DOWN: TILES | SLICED | {"16 rows", "32 rows", "4 rows, 16 waves"},
           DGATE: TILES, DX: TILES | SLICED, DW: TILES}


def kernel(m, k, i, h, product):
    return _lib.load().mj_gated_mlp_kernel(m, k, i, h, product).decode()


def depth(m, k, i, h, product):
    """The length of a product's sums."""
    return (k, i, h, i, m)[product]


@pytest.mark.parametrize("product", sorted(KERNELS))
def test_sizes_reach_every_kernel(product):
    assert {kernel(*s, product) for s in sizes.SHAPES} == KERNELS[product]


@pytest.mark.parametrize("product", sorted(KERNELS))
def test_sizes_reach_every_tile_with_and_without_a_last_part_stage(product):
    """The 64-deep stages of a sum: whole ones (their own loop on the two large tiles) and a
    last one in part."""
    took = {(kernel(*s, product), depth(*s, product) % 64 == 0) for s in sizes.SHAPES
            if depth(*s, product) >= 512}
    for tile in TILES - ({"64x64, 3 stages"} if product == DX else set()):
        assert {(tile, True), (tile, False)} <= took, tile


def test_kernel_of_no_product_and_of_refused_sizes():
    assert kernel(0, 8, 8, 8, GATE) == kernel(4, 8, 0, 8, DW) == ""
    assert kernel(4, 12, 8, 8, GATE) == kernel(4, 8, 8, 8, 5) == kernel(4, 8, 8, 8, -1) == ""
    assert kernel(1 << 31, 8, 8, 8, GATE) == kernel((1 << 31) - 1000, 8, 8, 8, GATE) == ""
