"""Host check that the sizes of the GPU tests reach every kernel that the plans of the experts'
block and of the 8-bit products can choose, and what those names are for empty products."""
import pytest

import test_gpu_experts as experts
import test_gpu_experts_kernels as kernels
import test_gpu_fp8 as fp8
from momijo_amd import _lib

TILES = {"256x256", "128x128", "64x64, 3 stages", "64x64, 5 stages", "128x64"}


@pytest.mark.parametrize("product", range(5))
def test_every_kernel_of_the_experts_block(product):
    name = _lib.load().mj_experts_mlp_kernel
    sizes = [(T * k, E, K, I, H) for T, k, E, K, I, H, *_ in experts._MLP + kernels.EXPERTS]
    assert {name(*s, product).decode() for s in sizes} == TILES | ({"16 rows"} if product < 2 else set())


@pytest.mark.parametrize("product", range(4))
def test_rounds_of_the_experts_block(product):
    """The sizes leave nothing, up to half a round and more than that over their whole rounds."""
    rests = set()
    for counts, K, I, H in kernels.ROUNDS:
        name = _lib.load().mj_experts_mlp_kernel(sum(counts), len(counts) - 1, K, I, H, product)
        assert name == b"256x256"
        width, cols = ((I, 128), (H, 256), (I, 256), (K, 256))[product]
        groups = counts if product % 2 else counts[:-1]  # y and dx have the dropped rows too
        rests.add(sum(-(-c // 256) for c in groups) * -(-width // cols) % 256)
    assert any(0 < r <= 128 for r in rests) and any(r > 128 for r in rests)
    assert product % 2 == 0 or {0, 128} <= rests


def test_every_kernel_of_the_8_bit_products():
    name = _lib.load().mj_gemm_f8_kernel
    tiles = {"256x256", "192x256", "128x128", "64x64"}
    assert {name(*s, 0, 0).decode() for s in fp8._LINEAR + kernels.LINEAR} == \
        tiles | {t + ", K slices" for t in tiles} | {"16 rows, quantizing", "16 rows", "32 rows", "64 rows"}
    sizes = [s[:6] for s in fp8._EXPERTS] + kernels.F8_EXPERTS
    assert {name(T * k, I, K, E, 1).decode() for T, k, E, K, I, H in sizes} == tiles | {"16 rows", "32 rows"}
    assert {name(T * k, H, I, E, 0).decode() for T, k, E, K, I, H in sizes} == tiles | {"16 rows", "32 rows"}


def test_names_of_nothing():
    mlp, f8 = _lib.load().mj_experts_mlp_kernel, _lib.load().mj_gemm_f8_kernel
    for s in ((0, 4, 8, 8, 8, 0), (8, 0, 8, 8, 8, 0), (8, 4, 12, 8, 8, 0), (8, 4, 8, 0, 8, 0), (8, 4, 8, 8, 8, 5)):
        assert mlp(*s) == b""
    for s in ((0, 8, 16, 0, 0), (8, 0, 16, 0, 0), (8, 8, 24, 0, 0), (8, 8, 16, 0, 1), (8, 8, 16, 1025, 0)):
        assert f8(*s) == b""
