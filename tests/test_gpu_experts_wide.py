"""Few rows an expert through layers so wide that the few-row kernels need more than 2^32 threads: 2^18 column
tiles for each of 33 and more segments of rows."""
import pytest

import test_gpu_experts as experts
import test_gpu_fp8 as fp8
from momijo_amd import _lib

pytestmark = pytest.mark.gpu

WIDE = 1 << 22                     # (the first width that is refused)
# tokens, experts, K, I, H
BF16 = [(33, 33, 8, WIDE - 8, 8), (33, 33, 8, 8, WIDE - 8)]
F8 = [(33, 33, 16, WIDE - 16, 16), (33, 33, 16, 16, WIDE - 3), (500, 60, 16, WIDE - 16, 16),
      (500, 60, 16, 16, WIDE - 3)]


@pytest.mark.parametrize("T,E,K,I,H", BF16)
def test_experts(dev, T, E, K, I, H):
    for product in (0, 1):
        assert _lib.load().mj_experts_mlp_kernel(T, E, K, I, H, product) == b"16 rows"
    experts.test_experts(dev, T, 1, E, K, I, H, "even")


@pytest.mark.parametrize("T,E,K,I,H", F8)
def test_f8_experts(dev, T, E, K, I, H):
    name = b"16 rows" if T <= 8 * E else b"32 rows"
    assert _lib.load().mj_gemm_f8_kernel(T, I, K, E, 1) == name == _lib.load().mj_gemm_f8_kernel(T, H, I, E, 0)
    fp8.test_experts(dev, T, 1, E, K, I, H, "even")
