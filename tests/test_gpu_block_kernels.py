"""Every kernel that the bf16 gated MLP chooses from, in every product that it takes, on sums
of whole 64-deep stages and of others, short and long (which kernels these sizes run is
asserted in test_block_kernels.py; bounds as in test_gpu_block.py)."""
import pytest
import torch

import _block as plain
import momijo_amd as mj
from test_gpu_block import ACTS, _close, _mlp_inputs

pytestmark = pytest.mark.gpu

# tokens, K, I, H
SHAPES = [(1, 8, 8, 8), (3, 64, 9000, 72), (4, 520, 8192, 264), (64, 8, 64, 64), (1028, 64, 8, 8),
          (1, 1024, 512, 3456), (17, 24, 480, 1096), (1, 4352, 1088, 8), (1, 5760, 896, 56),
          (448, 8, 2528, 8), (484, 4416, 8, 4824), (1472, 8, 1536, 8), (18, 1536, 1024, 64),
          (2013, 8, 1584, 8), (1580, 1968, 8, 2368), (898, 4128, 8, 4224), (17, 192, 1048, 5184),
          (2434, 3584, 8, 5120), (3083, 8, 2440, 16), (2304, 8, 5496, 8), (3430, 592, 64, 640),
          (192, 64, 5584, 248), (3321, 8, 4776, 16), (915, 3440, 64, 3456), (2368, 128, 1000, 64),
          (320, 8, 4992, 512), (132, 5864, 832, 256), (141, 5784, 928, 32), (2312, 8, 4608, 192),
          (1024, 8, 1024, 2368), (2701, 128, 2112, 256), (1106, 1280, 1024, 64),
          (1408, 320, 2432, 384), (4144, 2408, 128, 1832), (896, 320, 2336, 1280),
          (2983, 256, 1088, 1320), (512, 4096, 1128, 2112), (2318, 1376, 448, 4520),
          (1088, 1920, 1080, 5056), (1425, 1480, 1728, 1768), (2880, 1592, 1104, 1088),
          (2328, 88, 3584, 1792), (2624, 3080, 1024, 512), (2595, 3328, 1360, 3480),
          (3107, 1344, 2048, 3264), (3264, 1568, 3896, 1456)]


@pytest.mark.parametrize("act", sorted(ACTS))
@pytest.mark.parametrize("m,k,i,h", SHAPES)
def test_gated_mlp_kernels(dev, m, k, i, h, act):
    x, wg, wu, wd, dy = _mlp_inputs(m, k, i, h, torch.bfloat16)
    ref = plain.mlp(x, wg, wu, wd, dy, act, 2.0 ** -8, 2.0 ** -18)
    y0 = mj.gated_mlp(x, wg, wu, wd, ACTS[act])
    y, saved = mj.gated_mlp_train(x, wg, wu, wd, ACTS[act])
    grads = mj.gated_mlp_backward(dy, saved)
    assert torch.equal(y0, y)
    for key, got in zip(("y", "dx", "dgate", "dup", "ddown"), (y,) + tuple(grads)):
        _close(got, ref[key][0], ref[key][1] + 1e-30, key)
