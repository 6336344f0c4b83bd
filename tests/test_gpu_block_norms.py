"""The residual norm's backward in each of its forms: with and without biases (kernels of
their own: other registers, vectors in LDS and workgroups), the team of each width, one and
two chunks a thread, 16-byte rows and others, segments of a gate row's rows and runs of
whole groups (bounds as in test_gpu_block.py)."""
import pytest
import torch

import momijo_amd as mj
from test_gpu_block import DT, _check_norm, _norm_ops

pytestmark = pytest.mark.gpu

_VECTORS = {True: ("scale", "post_weight", "post_bias", "next_weight", "next_bias"),
            False: ("scale", "post_weight", "next_weight")}
# teams of 1, 2, 4, 8 waves and 8 with two chunks; multiples of 8 and not
_DIMS = [37, 512, 513, 1001, 1024, 1030, 2041, 2048, 2050, 3001, 4096, 4100, 6000, 8191, 8192]


def _off(t):
    """The same values one element off a 16-byte boundary."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    flat[1:] = t.reshape(-1)
    return flat[1:].reshape(t.shape)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("gates", ["none", "few", "each"])
@pytest.mark.parametrize("dim", _DIMS)
def test_residual_norm_forms(dev, dim, gates, bias, dtype):
    """Rows for more than one round of every team: 2 gate rows (segments), or one for every
    row or three (whole groups)."""
    rows = 66 if dim > 1024 else 1206
    groups = {"none": 0, "few": 2, "each": rows if dim % 2 else rows // 3}[gates]
    o = _norm_ops(rows, dim, groups, DT[dtype], _VECTORS[bias])
    kind = "layer" if (dim + len(gates)) % 2 else "rms"
    _check_norm(o, kind, 1e-3, 0.0 if gates == "few" else 0.25, 31, 6, DT[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("dim", [264, 1024, 2048, 4096, 8192])
def test_residual_norm_forms_misaligned(dev, dim, bias, dtype):
    o = _norm_ops(33, dim, 3, DT[dtype], _VECTORS[bias])
    want = _check_norm(o, "layer", 1e-3, 0.1, 31, 6, DT[dtype])
    moved = {k: None if v is None else _off(v) for k, v in o.items()}
    got = _check_norm(moved, "layer", 1e-3, 0.1, 31, 6, DT[dtype])
    assert torch.equal(got["y"], want["y"]) and torch.equal(got["n"], want["n"])


@pytest.mark.parametrize("dim", [1001, 4096, 8192])
def test_residual_norm_parts_of_each_width(dev, dim):
    """Without biases: each norm alone, the plain sum before the next norm, and no branch."""
    for on in (("post_weight",), ("next_weight",), ("scale", "next_weight"), ()):
        _check_norm(_norm_ops(40, dim, 0, torch.bfloat16, on), "rms", 1e-6, 0.1, 3, 0, torch.bfloat16)
    o = _norm_ops(40, dim, 0, torch.bfloat16, ("next_weight",))
    o["branch"] = None
    _check_norm(o, "layer", 1e-5, 0.0, 0, 0, torch.bfloat16)


@pytest.mark.parametrize("dim,rows", [(4096, 1500), (1001, 5000), (512, 9000)])
def test_residual_norm_repeats(dev, dim, rows):
    """The same inputs give the same bits."""
    o = _norm_ops(rows, dim, 2, torch.bfloat16, _VECTORS[False])
    kw = {k: o[k] for k in ("gate", "scale", "post_weight", "next_weight")}
    first = None
    for _ in range(3):
        y, n, saved = mj.residual_norm_train(o["x"], o["branch"], p=0.1, seed=5, **kw)
        now = [y, n] + list(mj.residual_norm_backward(o["dy"], o["dn"], saved).values())
        first = first or now
        assert all(torch.equal(a, b) for a, b in zip(first, now))
