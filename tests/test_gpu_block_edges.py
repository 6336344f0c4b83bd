"""The feed-forward block's operators where an operand, a width or a mask is out of the
ordinary (bounds as in test_gpu_block.py)."""
import pytest
import torch

import momijo_amd as mj
from test_gpu_block import DT, _gen, _normal

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ gated MLP
def _mlp_operands(m, k, i, h, dt):
    g = _gen("edges", m, k, i, h)
    return [_normal(g, shape, dt) for shape in ((m, k), (i, k), (i, k), (h, i), (m, h))]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("m,i,n", [(200, 6912, 2560), (64, 4096, 64), (3, 72, 40), (40, 1000, 1001)])
def test_gated_mlp_zero_width(dev, m, i, n, dtype):
    """No input features give y = 0, no output features gradients of 0, where y and dx
    are summed in K slices as well as where they are not."""
    dt = DT[dtype]
    x, wg, wu, wd, dy = _mlp_operands(m, 0, i, n, dt)
    y, saved = mj.gated_mlp_train(x, wg, wu, wd)
    dx, dgate, dup, ddown = mj.gated_mlp_backward(dy, saved)
    assert y.shape == (m, n) and dx.shape == (m, 0) and dgate.shape == dup.shape == (i, 0)
    assert not bool(y.any()) and not bool(mj.gated_mlp(x, wg, wu, wd).any()) and not bool(ddown.any())
    x, wg, wu, wd, dy = _mlp_operands(m, n, i, 0, dt)
    y, saved = mj.gated_mlp_train(x, wg, wu, wd)
    dx, dgate, dup, ddown = mj.gated_mlp_backward(dy, saved)
    assert y.shape == (m, 0) and dx.shape == (m, n) and ddown.shape == (0, i)
    assert not bool(dx.any()) and not bool(dgate.any()) and not bool(dup.any())
