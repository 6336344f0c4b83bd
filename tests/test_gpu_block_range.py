"""The residual norm and the gated MLP over more rows than one dimension of a grid holds (2^32 threads), up to
the last that the ABI takes (bounds as in test_gpu_block.py).  Only the last rows hold
anything: the others' outputs are zeros."""
import pytest
import torch

import _block as plain
import momijo_amd as mj
from test_gpu_block import _close, _gen, _normal

pytestmark = pytest.mark.gpu

LAST = 40


@pytest.fixture(autouse=True)
def release():
    """What a test held goes back before the next one allocates."""
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def _zeros_but_last(g, rows, dim):
    t = torch.zeros((rows, dim), dtype=torch.bfloat16, device="cuda")
    t[-LAST:] = _normal(g, (LAST, dim), torch.bfloat16)
    return t


def _room(nbytes):
    if torch.cuda.mem_get_info()[0] < nbytes:
        pytest.skip(f"needs {nbytes >> 30} GiB of device memory")


# 2^26 rows of up to 512 columns, a wave each, are 2^32 threads; 2^31 - 1 is the last number
# of rows, whose segments (or groups of one row) end past 2^31.  gates: gate rows
@pytest.mark.parametrize("rows,dim,gates", [((1 << 26) + 5, 8, 0), ((1 << 31) - 1, 1, 0), ((1 << 31) - 1, 1, -1)])
def test_residual_norm_rows_past_a_grid_dimension(dev, rows, dim, gates):
    _room(rows * (8 * dim * 2 + 40))
    g = _gen("grid", rows, gates)
    x, branch = _zeros_but_last(g, rows, dim), _zeros_but_last(g, rows, dim)
    w = _normal(g, (dim,), torch.float32, 0.2, 1.0)
    gate = _zeros_but_last(g, rows, dim) if gates else None
    kw = dict(scale=w, next_weight=w, eps=1e-3)
    y, n, saved = mj.residual_norm_train(x, branch, gate=gate, **kw)
    dn = _zeros_but_last(g, rows, dim)
    grads = mj.residual_norm_backward(None, dn, saved)
    o = dict(dict.fromkeys(("post_weight", "post_bias", "next_bias", "dy")), scale=w, next_weight=w,
             x=x[-LAST:], branch=branch[-LAST:], gate=gate[-LAST:] if gates else None, dn=dn[-LAST:])
    ref, size = plain.residual_norm(o, "rms", 1e-3, 0.0, 0, 0)
    got = dict(y=y[-LAST:], n=n[-LAST:], d_x=grads["x"][-LAST:], d_branch=grads["branch"][-LAST:],
               d_scale=grads["scale"], d_next_weight=grads["next_weight"])
    if gates:
        got["d_gate"] = grads["gate"][-LAST:]
    for name, have in got.items():
        want = ref[name]
        err = 2.0 ** -19 * (want.abs() + want.abs().max(-1, keepdim=True).values + 1e-3)
        if name in size:
            err = 2.0 ** -18 * (size[name] + size[name].max(-1, keepdim=True).values)
        u = 2.0 ** -8 if have.dtype == torch.bfloat16 else 2.0 ** -24
        _close(have, want, u * want.abs() * 1.01 + err, name)
    for t in (y, n, grads["x"], grads["branch"]) + ((grads["gate"],) if gates else ()):
        assert not bool(t[:-LAST].any())


@pytest.mark.parametrize("dim,backward", [(4104, False), (8200, True)])
def test_residual_norm_wide_rows_past_a_grid_dimension(dev, dim, backward):
    """2^22 rows of a workgroup of 1024 threads each."""
    rows = (1 << 22) + 3
    _room(rows * dim * 2 * (3 if backward else 2) + (1 << 32))
    g = _gen("wide grid", dim)
    x = _zeros_but_last(g, rows, dim)
    w = _normal(g, (dim,), torch.float32, 0.2, 1.0)
    y, n, saved = mj.residual_norm_train(x, next_weight=w, eps=1e-3)
    assert y is x and not bool(n[:-LAST].any())
    o = dict(dict.fromkeys(("branch", "gate", "scale", "post_weight", "post_bias", "next_bias", "dy")),
             next_weight=w, x=x[-LAST:], dn=None)
    last = n[-LAST:].clone()
    if backward:  # n's memory is dn's: gradient n
        o["dn"] = last
    else:
        o["dn"] = torch.zeros_like(last)
    ref, size = plain.residual_norm(o, "rms", 1e-3, 0.0, 0, 0)
    got = dict(n=last)
    if backward:
        grads = mj.residual_norm_backward(None, n, saved)
        got.update(d_x=grads["x"][-LAST:], d_next_weight=grads["next_weight"])
        assert not bool(grads["x"][:-LAST].any())
    for name, have in got.items():
        want = ref[name]
        err = 2.0 ** -19 * (want.abs() + want.abs().max(-1, keepdim=True).values + 1e-3)
        if name in size:
            err = 2.0 ** -18 * (size[name] + size[name].max(-1, keepdim=True).values)
        u = 2.0 ** -8 if have.dtype == torch.bfloat16 else 2.0 ** -24
        _close(have, want, u * want.abs() * 1.01 + err, name)


@pytest.mark.parametrize("rows,k,i,h", [((1 << 30) + 5, 8, 8, 8), ((1 << 29) + 3, 8, 40, 8)])
def test_gated_mlp_rows_past_a_grid_dimension(dev, rows, k, i, h):
    """2^30 rows are 2^24 tiles of 64 rows, 2^32 threads: larger tiles take them."""
    _room(rows * 2 * (k + i + h) + (4 << 30))
    g = _gen("mlp grid", rows)
    x = _zeros_but_last(g, rows, k)
    x[:LAST] = x[-LAST:]
    wg, wu = (_normal(g, (i, k), torch.bfloat16, k ** -0.5) for _ in range(2))
    wd = _normal(g, (h, i), torch.bfloat16, i ** -0.5)
    y = mj.gated_mlp(x, wg, wu, wd)
    ref = plain.mlp(x[-LAST:], wg, wu, wd, torch.zeros((LAST, h), device=dev), "silu", 2.0 ** -8, 2.0 ** -18)["y"]
    for part in (y[-LAST:], y[:LAST]):
        _close(part, ref[0], ref[1] + 1e-30, "y")
    assert not bool(y[LAST:-LAST].any())


def test_products_past_a_grid_dimension_are_refused(dev):
    """The fp32 tiles of 2^29 rows (512 threads for 64 rows) are 2^32 threads: an error, where
    a launch of a few more runs those few and leaves the other outputs; 2^28 rows run."""
    k = 8
    _room(3 << 35)
    g = _gen("f32 grid")
    w = _normal(g, (k, k), torch.float32, k ** -0.5)
    x = torch.zeros(((1 << 29) + 64, k), device=dev)
    with pytest.raises(mj.MomijoHipError):
        mj.gated_mlp(x, w, w, w)
    x = x[:1 << 28]
    x[-LAST:] = _normal(g, (LAST, k), torch.float32)
    y = mj.gated_mlp(x, w, w, w)
    ref = plain.mlp(x[-LAST:], w, w, w, torch.zeros((LAST, k), device=dev), "silu", 2.0 ** -24, 2.0 ** -20)["y"]
    _close(y[-LAST:], ref[0], ref[1] + 1e-30, "y")
    assert not bool(y[:-LAST].any())
    with pytest.raises(mj.MomijoHipError):   # a wave a row
        mj.quantize_rowwise_int8(torch.zeros(((1 << 26) + 8, 4), device=dev))
