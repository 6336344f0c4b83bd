"""The feed-forward block's operators where an operand, a width or a mask is out of the
ordinary (bounds as in test_gpu_block.py)."""
import pytest
import torch

import _block as plain
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


# ------------------------------------------------------------------ residual norm
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,dim", [(34, 264), (21, 1001), (9, 4100), (5, 8200)])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("bias", [False, True])
def test_residual_norm_dropped_places(dev, rows, dim, post, bias, dtype):
    """What a dropped place holds (the gate's value; without a post norm the branch's
    too: infinite, NaN) is in no output and no gradient: the bits are those of other
    values there."""
    dt, p, seed, counter = DT[dtype], 0.5, 21, 4
    g = _gen("dropped", rows, dim)
    vec = lambda: _normal(g, (dim,), torch.float32, 0.2, 1.0)  # noqa: E731
    keep = torch.from_numpy(plain.keep(rows * dim, p, seed, counter)).reshape(rows, dim).to(dev)
    x, branch, dy, dn = (_normal(g, (rows, dim), dt) for _ in range(4))
    gate = _normal(g, (rows, dim), dt, 0.3, 0.5)   # a gate row for every row
    kw = dict(scale=vec(), next_weight=vec(), p=p, seed=seed, counter=counter)
    if post:
        kw["post_weight"] = vec()
    if bias:
        kw["next_bias"] = vec()

    def step(b, q):
        y, n, saved = mj.residual_norm_train(x, b, gate=q, **kw)
        return [y, n] + list(mj.residual_norm_backward(dy, dn, saved).values())

    want = step(branch, gate)
    bad = torch.tensor([float("inf"), float("nan"), -float("inf")], device=dev, dtype=dt)
    bad = bad.repeat(rows * dim // 3 + 1)[:rows * dim].reshape(rows, dim)
    b = branch if post else torch.where(keep, branch, bad)
    for q in (gate, torch.where(keep, gate, bad)):
        assert all(torch.equal(a, c) for a, c in zip(step(b, q), want))


@pytest.mark.parametrize("dim,bias", [(264, True), (1001, False), (8200, True)])
def test_residual_norm_all_dropped(dev, dim, bias):
    """p = 1: the branch is in nothing, whatever it and the gate hold."""
    rows = 12
    g = _gen("all", dim)
    x, dy, dn = (_normal(g, (rows, dim), torch.bfloat16) for _ in range(3))
    w = _normal(g, (dim,), torch.float32, 0.2, 1.0)
    kw = dict(next_weight=w, next_bias=w if bias else None)
    nan = torch.full_like(x, float("nan"))
    y, n, saved = mj.residual_norm_train(x, nan, gate=nan[:2], p=1.0, seed=1, **kw)
    grads = mj.residual_norm_backward(dy, dn, saved)
    y0, n0, saved = mj.residual_norm_train(x, torch.zeros_like(x), gate=torch.ones_like(x[:2]), **kw)
    want = mj.residual_norm_backward(dy, dn, saved)
    assert torch.equal(y, x) and torch.equal(y0, x) and torch.equal(n, n0)
    assert not bool(grads["branch"].any()) and not bool(grads["gate"].any())
    for name in ("x", "next_weight") + (("next_bias",) if bias else ()):
        assert torch.equal(grads[name], want[name]), name


def test_residual_norm_arguments_without_work(dev):
    """Where y is x and no norm follows, wrong arguments are refused as elsewhere, and right
    ones give x and its gradient."""
    x, w = torch.randn((6, 32), device=dev), torch.ones(32, device=dev)
    for bad in (dict(p=0.5), dict(gate=torch.ones((2, 32), device=dev)), dict(post_weight=w),
                dict(next_bias=w), dict(post_bias=w), dict(eps=-1.0), dict(p=float("nan"))):
        with pytest.raises(mj.MomijoHipError):
            mj.residual_norm(x, **bad)
        with pytest.raises(mj.MomijoHipError):
            mj.residual_norm_train(x, **bad)
    with pytest.raises(mj.MomijoHipError):
        mj.residual_norm(torch.zeros((1, 16392), device=dev))
    y, n, saved = mj.residual_norm_train(x)
    assert y is x and n is None
    dy = torch.randn_like(x)
    assert torch.equal(mj.residual_norm_backward(dy, None, saved)["x"], dy)
    assert mj.residual_norm(x[:0])[0].shape == (0, 32)


def test_residual_norm_gate_without_rows(dev):
    """A gate of no rows is a gate that does not divide the rows; with no rows it fits."""
    x = torch.zeros((6, 32), dtype=torch.bfloat16, device=dev)
    with pytest.raises(ValueError):
        mj.residual_norm(x, x, gate=x[:0])
    with pytest.raises(ValueError):
        mj.residual_norm_train(x, x, gate=x[:0])
    y, _, saved = mj.residual_norm_train(x[:0], x[:0], gate=x[:0])
    grads = mj.residual_norm_backward(y, None, saved)
    assert y.shape == grads["gate"].shape == (0, 32)


# ------------------------------------------------------------------ dropout
def test_dropout_class_with_a_device_seed(dev):
    """A captured forward and backward draw from the seed tensor: every replay the mask of the
    counter that it holds then, as the eager call with that counter."""
    x, dy = (_normal(_gen("class", i), (5000,), torch.bfloat16) for i in range(2))
    state = torch.tensor([77, 0], dtype=torch.int64, device=dev)
    layer = mj.Dropout(0.3, state)
    y, c = layer.forward(x)
    assert c == 0 and torch.equal(y, mj.dropout(x, 0.3, 77, 0))
    torch.cuda.synchronize()
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        g.capture_begin()
        y, c = layer.forward(x)
        dx = layer.backward(dy, c)
        g.capture_end()
    assert c == 1
    for step in (0, 1, 9, 2 ** 40):
        state[1] = step
        y.zero_(), dx.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, mj.dropout(x, 0.3, 77, step + c))
        assert torch.equal(dx, mj.dropout(dy, 0.3, 77, step + c))
    with pytest.raises(ValueError):
        mj.Dropout(0.3, state.float()).forward(x)
