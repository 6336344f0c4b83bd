"""The feed-forward block's operators on arrays whose byte offsets pass 32 bits, the
last rows against the 64-bit plain forms (bounds as in test_gpu_block.py)."""
import numpy as np
import pytest
import torch

import _block as plain
import momijo_amd as mj
from test_gpu_block import DT, _close, _gen, _normal

pytestmark = pytest.mark.gpu

LAST = 40


@pytest.fixture(autouse=True)
def release():
    """What a test held goes back before the next one allocates."""
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype,m", [("bf16", 200_007), ("f32", 100_003)])
def test_gated_mlp_many_rows(dev, dtype, m):
    """Hidden arrays of 4.4 GB.  Only the last rows have a gradient, so the weights'
    gradients are theirs too."""
    k, i, h, dt = 24, 11008, 16, DT[dtype]
    g = _gen("rows", dtype)
    x, dy = _normal(g, (m, k), dt), torch.zeros((m, h), dtype=dt, device=dev)
    dy[-LAST:] = _normal(g, (LAST, h), dt)
    wg, wu = _normal(g, (i, k), dt, k ** -0.5), _normal(g, (i, k), dt, k ** -0.5)
    wd = _normal(g, (h, i), dt, i ** -0.5)
    assert m * i * dt.itemsize > 1 << 32
    y, saved = mj.gated_mlp_train(x, wg, wu, wd)
    dx, *dw = mj.gated_mlp_backward(dy, saved)
    unit, e32 = (2.0 ** -8, 2.0 ** -18) if dtype == "bf16" else (2.0 ** -24, 2.0 ** -20)
    ref = plain.mlp(x[-LAST:], wg, wu, wd, dy[-LAST:], "silu", unit, e32)
    got = dict(y=y[-LAST:], dx=dx[-LAST:], dgate=dw[0], dup=dw[1], ddown=dw[2])
    for key, value in got.items():
        _close(value, ref[key][0], ref[key][1] + 1e-30, key)
    assert not bool(dx[:-LAST].any())


@pytest.mark.parametrize("m", [2, 20])
def test_gated_mlp_large_weights(dev, m):
    """Gate and up of 4.3 GB each, for few rows."""
    k, i, h = 2056, (1 << 20) + 8, 8
    g = _gen("weights")
    x = _normal(g, (m, k), torch.bfloat16)
    wg, wu = (torch.zeros((i, k), dtype=torch.bfloat16, device=dev) for _ in range(2))
    wg[-LAST:], wu[-LAST:] = (_normal(g, (LAST, k), torch.bfloat16, k ** -0.5) for _ in range(2))
    wd = _normal(g, (h, i), torch.bfloat16)
    assert wg.numel() * 2 > 1 << 32
    y = mj.gated_mlp(x, wg, wu, wd)
    dy = torch.zeros((m, h), dtype=torch.bfloat16, device=dev)
    ref = plain.mlp(x, wg[-LAST:], wu[-LAST:], wd[:, -LAST:], dy, "silu", 2.0 ** -8, 2.0 ** -18)["y"]
    _close(y, ref[0], ref[1] + 1e-30, "y")


@pytest.mark.parametrize("dtype,rows", [("bf16", (1 << 20) + 5), ("f32", (1 << 19) + 5)])
def test_residual_norm_many_rows(dev, dtype, rows):
    dim, dt = 2056, DT[dtype]
    g = _gen("norm rows", dtype)
    assert rows * dim * dt.itemsize > 1 << 32
    full = {}
    for name in ("x", "branch", "dy", "dn"):
        full[name] = torch.zeros((rows, dim), dtype=dt, device=dev)
        full[name][-LAST:] = _normal(g, (LAST, dim), dt)
    w = _normal(g, (dim,), torch.float32, 0.2, 1.0)
    y, n, saved = mj.residual_norm_train(full["x"], full["branch"], post_weight=w, next_weight=w, eps=1e-3)
    grads = mj.residual_norm_backward(full["dy"], full["dn"], saved)
    o = dict(dict.fromkeys(("gate", "scale", "post_bias", "next_bias")), post_weight=w, next_weight=w,
             **{k: v[-LAST:] for k, v in full.items()})
    ref, size = plain.residual_norm(o, "rms", 1e-3, 0.0, 0, 0)
    got = dict(y=y[-LAST:], n=n[-LAST:], d_x=grads["x"][-LAST:], d_branch=grads["branch"][-LAST:],
               d_post_weight=grads["post_weight"], d_next_weight=grads["next_weight"])
    unit = 2.0 ** -8 if dt == torch.bfloat16 else 2.0 ** -24
    for name, have in got.items():
        want = ref[name]
        err = 2.0 ** -19 * (want.abs() + want.abs().max(-1, keepdim=True).values + 1e-3)
        if name in size:
            err = 2.0 ** -18 * (size[name] + size[name].max(-1, keepdim=True).values)
        u = unit if have.dtype == torch.bfloat16 else 2.0 ** -24
        _close(have, want, u * want.abs() * 1.01 + err, name)
    for t in (y, n, grads["x"], grads["branch"]):
        assert not bool(t[:-LAST].any())


def test_dropout_many_elements(dev):
    """Element numbers past 2^32: the last block's mask is its own."""
    n = (1 << 32) + 8 * 1000 + 3
    x = torch.ones(n, dtype=torch.bfloat16, device=dev)
    mj.dropout(x, 0.25, 11, 5, out=x)
    first = n // 8 - 100
    w = plain.philox4x32(np.arange(first, n // 8 + 1), 5, 11).view(np.uint16).reshape(-1)
    keep = torch.from_numpy(w[:n - 8 * first] >= plain.threshold(0.25)).to(dev)
    scale = torch.tensor(plain.keep_scale(0.25), device=dev).to(torch.bfloat16)
    want = torch.where(keep, scale, torch.zeros_like(scale))
    assert torch.equal(x[8 * first:], want)


def test_residual_norm_dropout_many_elements(dev):
    """The norm's mask past 2^32 elements is the one dropout draws (without norms and
    with x = 0, y is the dropped branch)."""
    dim = 4104
    rows = (1 << 32) // dim + 9
    x = torch.zeros((rows, dim), dtype=torch.bfloat16, device=dev)
    b = torch.ones((rows, dim), dtype=torch.bfloat16, device=dev)
    y, _ = mj.residual_norm(x, b, p=0.25, seed=11, counter=5)
    mj.dropout(b, 0.25, 11, 5, out=b)
    assert torch.equal(y[-LAST:], b[-LAST:])
    assert rows * dim > 1 << 32 and bool(y[-LAST:].any())
