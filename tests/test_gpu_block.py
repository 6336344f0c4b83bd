"""The feed-forward block's operators on the GPU against their 64-bit plain forms:
the gated MLP, the residual norm and dropout, forward and backward.

Bounds, derived per element:
  * bf16 holds 8 significant bits, so a rounding is off by up to 2^-8 relative; the gated MLP rounds h, dg and du (errors that pass through the next
    product with the other operand's magnitudes) and its outputs;
  * an fp32 sum is off by at most about 2^-20 of the sum of its terms' magnitudes
    at these lengths (pairs of 32-long MFMA sums in sequence, wave trees);
  * dropout selects and multiplies once: equal bits to the 32-bit product.
"""
import zlib

import numpy as np
import pytest
import torch

import _block as plain
import momijo_amd as mj

pytestmark = pytest.mark.gpu

ACTS = {"none": mj.EPI_NONE, "relu": mj.EPI_RELU, "gelu": mj.EPI_GELU_TANH, "silu": mj.EPI_SILU}
DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def _normal(gen, shape, dt, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=gen, device="cuda") * std + mean).to(dt)


def _gen(*key):
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(repr(key).encode()))


def _close(got, want, bound, name):
    got = got.to(want.device, torch.float64)
    assert got.shape == want.shape, (name, got.shape, want.shape)
    bad = ~((got - want).abs() <= bound)
    assert not bool(bad.any()), (
        f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {float((got - want).abs().max()):.3e}, "
        f"first at {torch.nonzero(bad)[0].tolist()}")


# ------------------------------------------------------------------ gated MLP
# tokens, K, I, H: one token, decode sizes, widths below and across a tile, tokens
# across 16 / 64 / 128 / 256 rows, odd widths (padded in bf16); the last two fill the
# chip with 256 x 256 tiles in every product, with and without K edges
_MLP = [(1, 64, 64, 64), (1, 1024, 2816, 1024), (2, 8, 8, 8), (3, 1, 1, 1), (5, 33, 47, 29),
        (16, 256, 704, 256), (17, 520, 264, 136), (48, 512, 1376, 512), (65, 96, 200, 328),
        (129, 264, 520, 72), (200, 1001, 999, 77), (257, 128, 1000, 640), (300, 640, 1728, 640),
        (700, 520, 1400, 520), (4001, 2600, 5000, 2568), (4096, 2560, 5120, 2560)]


def _mlp_inputs(m, k, i, h, dt):
    g = _gen(m, k, i, h)
    return (_normal(g, (m, k), dt), _normal(g, (i, k), dt, k ** -0.5), _normal(g, (i, k), dt, k ** -0.5),
            _normal(g, (h, i), dt, i ** -0.5), _normal(g, (m, h), dt))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("m,k,i,h", _MLP)
def test_gated_mlp(dev, m, k, i, h, dtype):
    name = ["silu", "gelu", "relu", "none"][(m + k) % 4]
    dt = DT[dtype]
    x, wg, wu, wd, dy = _mlp_inputs(m, k, i, h, dt)
    unit, e32 = (2.0 ** -8, 2.0 ** -18) if dtype == "bf16" else (2.0 ** -24, 2.0 ** -20)
    ref = plain.mlp(x, wg, wu, wd, dy, name, unit, e32)
    y0 = mj.gated_mlp(x, wg, wu, wd, ACTS[name])
    y, saved = mj.gated_mlp_train(x, wg, wu, wd, ACTS[name])
    grads = mj.gated_mlp_backward(dy, saved)
    torch.cuda.synchronize()
    assert y.dtype == dt and all(t.dtype == dt for t in grads)
    for key, got in zip(("y", "y", "dx", "dgate", "dup", "ddown"), (y0, y) + tuple(grads)):
        _close(got, ref[key][0], ref[key][1] + 1e-30, key)


@pytest.mark.parametrize("m,k,i,h", [(200, 2560, 6912, 2560), (1000, 1040, 2808, 1040), (48, 1536, 4160, 1536),
                                     (130, 2000, 4232, 1800)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_gated_mlp_k_slices(dev, m, k, i, h, dtype):
    """Few outputs and long sums: y and dx in slices of K, of unequal lengths too."""
    dt = DT[dtype]
    x, wg, wu, wd, dy = _mlp_inputs(m, k, i, h, dt)
    unit, e32 = (2.0 ** -8, 2.0 ** -18) if dtype == "bf16" else (2.0 ** -24, 2.0 ** -20)
    ref = plain.mlp(x, wg, wu, wd, dy, "silu", unit, e32)
    y, saved = mj.gated_mlp_train(x, wg, wu, wd)
    for key, got in zip(("y", "dx", "dgate", "dup", "ddown"),
                        (y,) + tuple(mj.gated_mlp_backward(dy, saved))):
        _close(got, ref[key][0], ref[key][1] + 1e-30, key)


@pytest.mark.parametrize("name", sorted(ACTS))
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_gated_mlp_activations(dev, name, dtype):
    m, k, i, h = 40, 72, 136, 48
    dt = DT[dtype]
    x, wg, wu, wd, dy = _mlp_inputs(m, k, i, h, dt)
    x = x * 4      # g well into the saturated parts
    unit, e32 = (2.0 ** -8, 2.0 ** -18) if dtype == "bf16" else (2.0 ** -24, 2.0 ** -20)
    ref = plain.mlp(x, wg, wu, wd, dy, name, unit, e32)
    y, saved = mj.gated_mlp_train(x, wg, wu, wd, ACTS[name])
    for key, got in zip(("y", "dx", "dgate", "dup", "ddown"),
                        (y,) + tuple(mj.gated_mlp_backward(dy, saved))):
        _close(got, ref[key][0], ref[key][1] + 1e-30, key)


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_gated_mlp_saturated_gate(dev, act):
    """Gates far out give the limits, not NaN: act(-big) = 0 with gradient 0,
    act(big) = big with gradient 1."""
    for big in (1e4, 1e15):
        one = torch.ones((1, 8), dtype=torch.bfloat16, device=dev)
        for sign in (1.0, -1.0):
            wg = torch.zeros((8, 8), dtype=torch.bfloat16, device=dev)
            wg[:, 0] = sign * big
            wu = torch.eye(8, dtype=torch.bfloat16, device=dev)
            y, saved = mj.gated_mlp_train(one, wg, wu, wu, ACTS[act])
            grads = mj.gated_mlp_backward(torch.ones_like(y), saved)
            assert all(bool(torch.isfinite(t).all()) for t in (y,) + tuple(grads))
            want = float(wg[0, 0]) if sign > 0 else 0.0
            assert bool((y.float() == want).all())


def test_gated_mlp_gradient_against_differences(dev):
    """Directional derivatives of the Float32 block: central differences of step e
    err by e^2 of the third derivative (order 1 here) and 2^-23 |L| / e."""
    m, k, i, h = 9, 40, 56, 24
    g = _gen("diff")
    x, wg, wu, wd, dy = _mlp_inputs(m, k, i, h, torch.float32)
    ops = [x, wg, wu, wd]
    _, saved = mj.gated_mlp_train(*ops, mj.EPI_SILU)
    grads = mj.gated_mlp_backward(dy, saved)
    for n in range(4):
        d = torch.randn(ops[n].shape, generator=g, device=dev)
        d = d / d.norm()
        e = 0.02
        ends = []
        for s in (e, -e):
            moved = [t + s * d if j == n else t for j, t in enumerate(ops)]
            ends.append(float((mj.gated_mlp(*moved, mj.EPI_SILU).double() * dy.double()).sum()))
        slope = (ends[0] - ends[1]) / (2 * e)
        want = float((grads[n].double() * d.double()).sum())
        assert abs(slope - want) <= 2e-2 * float(grads[n].double().norm()) + 1e-3, n


def test_gated_mlp_shapes_and_strides(dev):
    """Leading dimensions, non-contiguous and misaligned operands, no rows."""
    k, i, h = 64, 72, 40
    x, wg, wu, wd, dy = _mlp_inputs(12, k, i, h, torch.bfloat16)
    y, saved = mj.gated_mlp_train(x, wg, wu, wd)
    grads = mj.gated_mlp_backward(dy, saved)
    y3, saved3 = mj.gated_mlp_train(x.reshape(3, 4, k), wg, wu, wd)
    assert y3.shape == (3, 4, h) and torch.equal(y3.reshape(12, h), y)
    g3 = mj.gated_mlp_backward(dy.reshape(3, 4, h), saved3)
    assert g3[0].shape == (3, 4, k) and all(torch.equal(a.reshape(b.shape), b) for a, b in zip(g3, grads))
    wide = torch.empty((12, 2 * k), dtype=torch.bfloat16, device=dev)
    wide[:, ::2] = x
    wt = wg.t().contiguous().t()
    off = torch.empty(h * i + 1, dtype=torch.bfloat16, device=dev)
    off[1:] = wd.reshape(-1)
    y4, saved4 = mj.gated_mlp_train(wide[:, ::2], wt, wu, off[1:].reshape(h, i))
    assert torch.equal(y4, y)
    dyt = dy.t().contiguous().t()
    assert all(torch.equal(a, b) for a, b in zip(mj.gated_mlp_backward(dyt, saved4), grads))
    y0, saved0 = mj.gated_mlp_train(x[:0], wg, wu, wd)
    g0 = mj.gated_mlp_backward(dy[:0], saved0)
    assert y0.shape == (0, h) and g0[0].shape == (0, k)
    assert all(not bool(t.any()) for t in g0[1:])


def test_gated_mlp_repeats(dev):
    """The same inputs give the same bits."""
    x, wg, wu, wd, dy = _mlp_inputs(40, 2048, 1024, 64, torch.bfloat16)
    first = None
    for _ in range(3):
        y, saved = mj.gated_mlp_train(x, wg, wu, wd)
        now = (y,) + tuple(mj.gated_mlp_backward(dy, saved))
        first = first or now
        assert all(torch.equal(a, b) for a, b in zip(first, now))


def test_gated_mlp_refusals(dev):
    x, wg, wu, wd, dy = _mlp_inputs(4, 16, 24, 8, torch.bfloat16)
    with pytest.raises(TypeError):
        mj.gated_mlp(x.half(), wg, wu, wd)
    with pytest.raises(TypeError):
        mj.gated_mlp(x, wg.float(), wu, wd)
    with pytest.raises(ValueError):
        mj.gated_mlp(x, wg, wu[:8], wd)
    with pytest.raises(ValueError):
        mj.gated_mlp(x[:, :8], wg, wu, wd)
    with pytest.raises(ValueError):
        mj.gated_mlp(x, wg, wu, wd[:, :16])
    with pytest.raises(ValueError):
        mj.gated_mlp(x.cpu(), wg, wu, wd)
    with pytest.raises(mj.MomijoHipError):
        mj.gated_mlp(x, wg, wu, wd, mj.EPI_SILU_APPROX)
    with pytest.raises(mj.MomijoHipError):
        mj.gated_mlp(x, wg, wu, wd, 99)
    _, saved = mj.gated_mlp_train(x, wg, wu, wd)
    with pytest.raises(ValueError):
        mj.gated_mlp_backward(dy[:3], saved)
    with pytest.raises(ValueError):
        mj.GatedMLP(wg, wu[:8], wd)


# ------------------------------------------------------------------ residual norm
# rows, dim, gate rows (0: none, -1: [dim]): widths of every team, ragged ones,
# groups of one row, of all rows and between, more groups than segments
_NORM = [(1, 1, 0), (1, 8, 1), (3, 7, 3), (5, 64, -1), (64, 100, 4), (33, 512, 1), (40, 513, 0),
         (70, 1000, 7), (30, 1001, 2), (12, 2048, 1), (9, 2056, 3), (20, 4096, 4), (3, 4100, 1),
         (6, 8192, 2), (4, 8191, 1), (3, 16384, 1), (2, 9000, 2), (1300, 64, 1300), (2000, 24, 500),
         (1500, 16, 1), (1025, 136, 5)]


def _norm_ops(rows, dim, gates, dt, on):
    g = _gen(rows, dim, gates)
    vec = lambda m, s: _normal(g, (dim,), torch.float32, s, m)  # noqa: E731
    o = dict(x=_normal(g, (rows, dim), dt), branch=_normal(g, (rows, dim), dt, 1.5, 0.25), gate=None,
             scale=vec(1.0, 0.1), post_weight=vec(1.0, 0.2), post_bias=vec(0.0, 0.2),
             next_weight=vec(1.0, 0.2), next_bias=vec(0.0, 0.2))
    if gates:
        o["gate"] = _normal(g, (dim,) if gates < 0 else (gates, dim), dt, 0.3, 0.5)
    for key in list(o):
        if key not in ("x", "branch", "gate") and key not in on:
            o[key] = None
    for key in ("post", "next"):
        if o[key + "_weight"] is None:
            o[key + "_bias"] = None
    o["dy"] = _normal(g, (rows, dim), dt)
    o["dn"] = _normal(g, (rows, dim), dt) if o["next_weight"] is not None else None
    return o


_FULL = ("scale", "post_weight", "post_bias", "next_weight", "next_bias")


def _check_norm(o, kind, eps, p, seed, counter, dt, grads=True):
    call = {k: v for k, v in o.items() if k not in ("x", "branch", "dy", "dn")}
    call.update(norm=kind, eps=eps, p=p, seed=seed, counter=counter)
    ref, size = plain.residual_norm(o, kind, eps, p, seed, counter)
    y0, n0 = mj.residual_norm(o["x"], o["branch"], **call)
    y, n, saved = mj.residual_norm_train(o["x"], o["branch"], **call)
    assert torch.equal(y0, y) and (n is None or torch.equal(n0, n))
    got = {"y": y, "n": n}
    if grads:
        got.update({"d_" + k: v for k, v in mj.residual_norm_backward(o["dy"], o["dn"], saved).items()})
    unit = 2.0 ** -8 if dt == torch.bfloat16 else 2.0 ** -24
    for name, want in ref.items():
        have = got[name]
        if name == "d_gate" and have.dim() == 1:
            have = have[None]
        # a row's fp32 arithmetic: some ten roundings of values up to its largest, and
        # its sums' relative error on every element; sums over rows and differences
        # that cancel: of their terms
        rows_err = 2.0 ** -19 * (want.abs() + want.abs().max(-1, keepdim=True).values + 1e-3)
        if name in size:
            rows_err = 2.0 ** -18 * (size[name] + size[name].max(-1, keepdim=True).values)
        u = unit if have.dtype == torch.bfloat16 else 2.0 ** -24
        _close(have, want, u * want.abs() * 1.01 + rows_err, name)
    return got


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows,dim,gates", _NORM)
def test_residual_norm(dev, rows, dim, gates, kind, dtype):
    if kind == "layer" and dim == 1:
        pytest.skip("the variance of one value is zero: only eps is left")
    o = _norm_ops(rows, dim, gates, DT[dtype], _FULL)
    _check_norm(o, kind, 1e-3, 0.25 if rows % 2 else 0.0, 12345, 7, DT[dtype])


@pytest.mark.parametrize("on", [(), ("post_weight",), ("next_weight",), ("scale", "next_weight"),
                                ("post_weight", "next_weight"), ("post_weight", "post_bias", "scale")])
@pytest.mark.parametrize("gates", [0, 2])
def test_residual_norm_parts(dev, on, gates):
    """Each part alone and in pairs."""
    o = _norm_ops(34, 264, gates, torch.bfloat16, on)
    _check_norm(o, "rms", 1e-6, 0.1, 3, 0, torch.bfloat16)


@pytest.mark.parametrize("rows,dim,gates,on", [
    (600, 8200, 600, _FULL), (530, 8201, 265, _FULL), (20, 8193, 0, ("post_weight",)),
    (20, 12288, 2, ("next_weight", "scale")), (300, 10000, 3, ("post_weight", "next_weight")),
    (7, 16384, 7, ())])
def test_residual_norm_wide_rows(dev, rows, dim, gates, on):
    """Above 8192 columns, where the backward walks the rows twice: a gate row for every
    row and for two, segments inside groups, each part alone."""
    o = _norm_ops(rows, dim, gates, torch.bfloat16, on)
    _check_norm(o, "layer" if rows % 3 else "rms", 1e-3, 0.25, 99, 3, torch.bfloat16)


@pytest.mark.parametrize("scale", [False, True])
def test_residual_norm_without_branch(dev, scale):
    """The norm before the first block; without a scale y is x itself."""
    o = _norm_ops(21, 200, 0, torch.bfloat16, ("next_weight", "next_bias") + (("scale",) if scale else ()))
    o["branch"] = None
    got = _check_norm(o, "layer", 1e-5, 0.0, 0, 0, torch.bfloat16)
    assert scale or got["y"] is o["x"]


def test_residual_norm_missing_gradients(dev):
    """dy or dn None stands for zero."""
    o = _norm_ops(19, 136, 1, torch.float32, _FULL)
    for gone in ("dy", "dn"):
        part = dict(o)
        part[gone] = None
        _check_norm(part, "rms", 1e-6, 0.0, 0, 0, torch.float32)


def test_residual_norm_misaligned(dev):
    """Operands one element off a 16-byte boundary, and other strides."""
    o = _norm_ops(17, 264, 1, torch.bfloat16, _FULL)
    want = _check_norm(o, "rms", 1e-6, 0.25, 1, 2, torch.bfloat16)

    def off(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        flat[1:] = t.reshape(-1)
        return flat[1:].reshape(t.shape)

    moved = {k: None if v is None else off(v) for k, v in o.items()}
    got = _check_norm(moved, "rms", 1e-6, 0.25, 1, 2, torch.bfloat16)
    assert torch.equal(got["y"], want["y"]) and torch.equal(got["n"], want["n"])
    turned = dict(o)
    for k in ("x", "branch", "dy", "dn"):
        turned[k] = o[k].t().contiguous().t()
    got = _check_norm(turned, "rms", 1e-6, 0.25, 1, 2, torch.bfloat16)
    assert all(torch.equal(got[k], want[k]) for k in want)


def test_residual_norm_zero_rows_and_extremes(dev):
    """A zero branch row gives 0 / sqrt(eps); a NaN in a dropped place stays out
    where no norm reads it; an infinite row spoils itself only."""
    dim = 256
    x = torch.ones((4, dim), device=dev)
    b = torch.zeros((4, dim), device=dev)
    w = torch.ones(dim, device=dev)
    y, n = mj.residual_norm(x, b, post_weight=w, next_weight=w)
    assert torch.equal(y, x) and bool((n - 1).abs().max() < 1e-5)
    k = torch.from_numpy(plain.keep(4 * dim, 0.5, 9, 1)).reshape(4, dim).to(dev)
    b = torch.where(k, 2.0, float("nan")).to(dev)
    y, _ = mj.residual_norm(x, b, p=0.5, seed=9, counter=1)
    assert torch.equal(y, torch.where(k, 5.0, 1.0))
    b = torch.ones((4, dim), device=dev)
    b[2, 5] = float("inf")
    y, n = mj.residual_norm(x, b, post_weight=w, next_weight=w)
    assert bool(torch.isfinite(y[[0, 1, 3]]).all()) and bool(torch.isfinite(n[[0, 1, 3]]).all())
    assert bool(torch.isnan(y[2]).any())


def test_residual_norm_large_mean(dev):
    """The layer norm's variance comes from differences from the mean: a mean 1000
    times the spread costs its 2^-24 relative to the mean, no more."""
    g = _gen("mean")
    x = _normal(g, (8, 1024), torch.float32, 1.0, 1000.0)
    w = torch.ones(1024, device=dev)
    _, n = mj.residual_norm(x, next_weight=w, norm="layer", eps=1e-6)
    want, _ = plain.norm(x.double().cpu(), "layer", 1e-6)
    _close(n, want, torch.full_like(want, 1000 * 2.0 ** -21), "n")


def test_residual_norm_gradient_against_differences(dev):
    o = _norm_ops(6, 40, 2, torch.float32, _FULL)
    names = ("x", "branch", "gate", "scale", "post_weight", "post_bias", "next_weight", "next_bias")
    kw = dict(norm="layer", eps=1e-3, p=0.25, seed=4, counter=2)
    run = lambda t: mj.residual_norm(t["x"], t["branch"], **{k: t[k] for k in names[2:]}, **kw)  # noqa: E731
    loss = lambda y, n: float((y.double() * o["dy"]).sum() + (n.double() * o["dn"]).sum())  # noqa: E731
    _, _, saved = mj.residual_norm_train(o["x"], o["branch"], **{k: o[k] for k in names[2:]}, **kw)
    grads = mj.residual_norm_backward(o["dy"], o["dn"], saved)
    g, e = _gen("norm diff"), 0.02
    for name in names:
        d = torch.randn(o[name].shape, generator=g, device=dev)
        d = d / d.norm()
        ends = [loss(*run({**o, name: o[name] + s * d})) for s in (e, -e)]
        want = float((grads[name].double() * d.double()).sum())
        assert abs((ends[0] - ends[1]) / (2 * e) - want) <= 2e-2 * float(grads[name].double().norm()) + 1e-3, name


def test_residual_norm_empty(dev):
    x = torch.empty((0, 64), dtype=torch.bfloat16, device=dev)
    w = torch.ones(64, device=dev)
    y, n, saved = mj.residual_norm_train(x, x, post_weight=w, next_weight=w)
    grads = mj.residual_norm_backward(y, n, saved)
    assert y.shape == n.shape == (0, 64) and not bool(grads["post_weight"].any())


def test_residual_norm_refusals(dev):
    x = torch.zeros((6, 32), device=dev)
    w = torch.ones(32, device=dev)
    with pytest.raises(mj.MomijoHipError):
        mj.residual_norm(x, x, gate=torch.ones((4, 32), device=dev))       # 4 does not divide 6
    with pytest.raises(ValueError):
        mj.residual_norm(x, x, gate=torch.ones((2, 16), device=dev))
    with pytest.raises(ValueError):
        mj.residual_norm(x, x, next_weight=w[:8])
    with pytest.raises(ValueError):
        mj.residual_norm(x, x[:3], next_weight=w)
    with pytest.raises(ValueError):
        mj.residual_norm(x, x, next_weight=w, norm="batch")
    with pytest.raises(TypeError):
        mj.residual_norm(x, x.bfloat16(), next_weight=w)
    with pytest.raises(mj.MomijoHipError):
        mj.residual_norm(x, x, p=1.5)
    with pytest.raises(mj.MomijoHipError):
        mj.residual_norm(x, x, post_bias=w)
    with pytest.raises(mj.MomijoHipError):
        mj.residual_norm(x, None, post_weight=w, next_weight=w)
    with pytest.raises(mj.MomijoHipError):
        wide = torch.zeros((1, 16392), device=dev)
        mj.residual_norm(wide, wide)
    _, _, saved = mj.residual_norm_train(x, x, post_weight=w)
    with pytest.raises(ValueError):
        mj.residual_norm_backward(x, x, saved)                             # no next norm


# ------------------------------------------------------------------ dropout
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n", [1, 7, 8, 9, 255, 2048, 8191, 8200, 100003])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
def test_dropout(dev, n, p, dtype):
    dt = DT[dtype]
    x = _normal(_gen(n), (n,), dt)
    seed, counter = (1 << 40) + 17, (1 << 33) + n
    got = mj.dropout(x, p, seed, counter)
    k = torch.from_numpy(plain.keep(n, p, seed, counter)).to(dev)
    want = torch.where(k, x.float() * np.float32(plain.keep_scale(p)), 0.0).to(dt)
    assert torch.equal(got, want)
    assert torch.equal(mj.dropout_backward(x, p, seed, counter), want)


def test_dropout_probability_steps(dev):
    """p below half a step still drops, p just below 1 still keeps."""
    x = torch.ones(1 << 20, device=dev)
    for p in (1e-9, 1.0 - 1e-7):
        got = mj.dropout(x, p, 5)
        k = torch.from_numpy(plain.keep(x.numel(), p, 5, 0)).to(dev)
        assert torch.equal(got != 0, k) and bool(k.any()) and not bool(k.all())
    for p in (0.1, 0.5):
        assert abs(float((mj.dropout(x, p, 8) == 0).double().mean()) - p) < 4 * (p * (1 - p) / x.numel()) ** 0.5 + 2.0 ** -17


def test_dropout_special_values_places_and_strides(dev):
    n = 4099
    x = _normal(_gen("special"), (n,), torch.float32)
    k = torch.from_numpy(plain.keep(n, 0.5, 3, 0)).to(dev)
    bad = torch.where(k, x, torch.tensor([float("nan"), float("inf")], device=dev).repeat(n)[:n])
    assert torch.equal(mj.dropout(bad, 0.5, 3), torch.where(k, x * 2, 0.0))
    off = torch.empty(n + 1, device=dev)
    off[1:] = x
    want = mj.dropout(x, 0.5, 3)
    assert torch.equal(mj.dropout(off[1:], 0.5, 3), want)
    two = x[:4096].reshape(64, 64)
    assert torch.equal(mj.dropout(two.t(), 0.5, 3), mj.dropout(two.t().contiguous(), 0.5, 3))
    assert torch.equal(mj.dropout(x, 0.5, 3, out=x), want)           # in place
    assert mj.dropout(x[:0], 0.5, 3).numel() == 0


def test_dropout_device_seed_in_a_graph(dev):
    """A captured call draws from the device's {seed, counter}: each replay another
    mask, checked against the eager call."""
    x = _normal(_gen("graph"), (5000,), torch.bfloat16)
    state = torch.tensor([77, 0], dtype=torch.int64, device=dev)
    out = torch.empty_like(x)
    mj.dropout(x, 0.3, state, out=out)
    torch.cuda.synchronize()
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        g.capture_begin()
        mj.dropout(x, 0.3, state, out=out)
        g.capture_end()
    for c in (0, 1, 5, 2 ** 40):
        state[1] = c
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, mj.dropout(x, 0.3, 77, c))


def test_dropout_class_and_refusals(dev):
    layer = mj.Dropout(0.25, seed=6)
    x = torch.ones(1000, device=dev)
    (a, ca), (b, cb) = layer.forward(x), layer.forward(x)
    assert (ca, cb) == (0, 1) and not torch.equal(a, b)
    assert torch.equal(layer.backward(x, ca), a) and torch.equal(layer.backward(x, cb), b)
    layer.training = False
    assert layer.forward(x)[0] is x
    with pytest.raises(ValueError):
        mj.Dropout(1.5)
    with pytest.raises(mj.MomijoHipError):
        mj.dropout(x, -0.1, 0)
    with pytest.raises(mj.MomijoHipError):
        mj.dropout(x, float("nan"), 0)
    with pytest.raises(TypeError):
        mj.dropout(x.double(), 0.1, 0)
    with pytest.raises(ValueError):
        mj.dropout(x, 0.1, torch.zeros(2, device=dev))
    with pytest.raises(ValueError):
        mj.dropout(x, 0.1, 0, out=x[:5])


# ------------------------------------------------------------------ streams, graphs
def test_block_on_another_stream_and_in_a_graph(dev):
    """The training step runs on the current stream and can be captured; every
    replay gives the eager step's bits."""
    m, k, i = 70, 264, 520
    x, wg, wu, wd, dy = _mlp_inputs(m, k, i, k, torch.bfloat16)
    w = torch.ones(k, device=dev)

    def step():
        y, n, s0 = mj.residual_norm_train(x, next_weight=w)
        b, s1 = mj.gated_mlp_train(n, wg, wu, wd)
        y, n, s2 = mj.residual_norm_train(y, b, post_weight=w, next_weight=w, p=0.1, seed=3)
        d2 = mj.residual_norm_backward(dy, dy, s2)
        d1 = mj.gated_mlp_backward(d2["branch"], s1)
        d0 = mj.residual_norm_backward(d2["x"], d1[0], s0)
        return [y, n, d0["x"], d0["next_weight"], d2["post_weight"], *d1]

    want = [t.clone() for t in step()]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        other = step()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        g.capture_begin()
        out = step()
        g.capture_end()
    for _ in range(3):
        for t in out:
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        step()
        torch.cuda.synchronize()
