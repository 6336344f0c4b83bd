"""The quantizer against its definition by arithmetic on fractions, without the steps of any floating-point unit:

    a = max(the block's largest magnitude, 2^-100), scale = a (1 / 448), values = e4m3(v (448 (1 / a)))

with each operation in parentheses rounded to Float32, ties to even.  Against the quotients a / 448 and
v 448 / a themselves: the scale has two roundings more, 2 x 2^-24 of it, and the number that is rounded to
e4m3 three, so that a value is e4m3's neighbour on the other side only if the quotient lies that near to the
middle between two."""
from fractions import Fraction

import numpy as np
import pytest
import torch

import _experts as plain


def _nearest(x, bits, low):
    """x to `bits` bits of mantissa, ties to even; exponents below `low` share its steps."""
    if x == 0:
        return x
    e = abs(x).numerator.bit_length() - abs(x).denominator.bit_length()
    if abs(x) < Fraction(2) ** e:
        e -= 1
    step = Fraction(2) ** (max(e, low) - bits + 1)
    return round(x / step) * step     # (Python rounds a fraction's ties to even)


def _f32(x):
    return _nearest(x, 24, -126)


def _e4m3(x):
    v = _nearest(x, 4, -6)
    assert abs(v) <= 448
    return v


def _block(values):
    """(values as e4m3 numbers, scale) of a block, and a."""
    v = [Fraction(float(t)) for t in values]
    a = max([Fraction(1, 2 ** 100)] + [abs(t) for t in v])
    factor = _f32(448 * _f32(1 / a))
    return [_e4m3(_f32(t * factor)) for t in v], _f32(a * _f32(Fraction(1, 448))), a


def _input():
    """Rows of two blocks and a part of one: magnitudes from 2^-130 to 2^127, 8-bit mantissas (ties are
    frequent), whole steps and middles of e4m3, zeros."""
    r = np.random.default_rng(5)
    x = r.standard_normal((14, 272)).astype(np.float32)
    x[::2] = torch.from_numpy(x[::2]).bfloat16().float().numpy()
    x *= np.exp2(np.array([0, -40, 20, -90, 60, -99, -101, -110, 3, -20, 0, 1, -3, 0], np.float32))[:, None]
    x[10, :128] = np.arange(128) * 3.5            # (largest 444.5)
    x[11, :128] = 448 - np.arange(128) * 3.5      # a is 448: values as they are
    x[12, :128] = 0
    x[13, 128:256] *= np.float32(3e38) / np.abs(x[13, 128:256]).max()
    return x


@pytest.fixture(scope="module")
def expected():
    x = _input()
    q, s = np.empty_like(x), np.empty((3, x.shape[0]), np.float32)
    for m in range(x.shape[0]):
        for b in range(3):
            at = slice(128 * b, min(128 * b + 128, x.shape[1]))
            v, scale, a = _block(x[m, at])
            q[m, at], s[b, m] = [float(t) for t in v], float(scale)
            near = Fraction(301, 100) / 2 ** 24
            assert abs(scale - a / 448) <= (Fraction(201, 100) / 2 ** 24) * a / 448 + Fraction(1, 2 ** 149)
            for t, got in zip(x[m, at], v):
                want = Fraction(float(t)) * 448 / a
                assert got in (_e4m3(want), *(_nearest(want * (1 + d * near), 4, -6) for d in (-1, 1)))
    return x, q, s


def test_the_tests_plain_form(expected):
    x, q, s = expected
    rq, rs = plain.quantize_rows(x)
    assert np.array_equal(rq, q) and np.array_equal(rs, s)


def test_blocks_of_a_matrix():
    x = _input()[:3, :144]
    rq, rs = plain.quantize_blocks(x)
    for b, at in enumerate((slice(0, 128), slice(128, 144))):
        v, scale, _ = _block(x[:, at].reshape(-1))
        assert rs[0, b] == float(scale) and rq[:, at].reshape(-1).tolist() == [float(t) for t in v]


@pytest.mark.gpu
def test_the_kernels(dev, expected):
    import momijo_amd as mj
    x, q, s = expected
    gq, gs = mj.quantize_rows_fp8(torch.from_numpy(x).cuda())
    assert np.array_equal(gq.float().cpu().numpy(), q) and np.array_equal(gs.cpu().numpy(), s)
    plan = mj.sort_experts(torch.zeros(x.shape[0], 1, dtype=torch.int32, device="cuda"), 1)
    dq, ds = mj.dispatch_fp8(torch.from_numpy(x).cuda(), plan)
    assert torch.equal(dq.view(torch.uint8), gq.view(torch.uint8)) and torch.equal(ds, gs)
    w = x[:3, :144]
    wq, ws = mj.quantize_blocks_fp8(torch.from_numpy(w).cuda())
    rq, rs = plain.quantize_blocks(w)
    assert np.array_equal(wq.float().cpu().numpy(), rq) and np.array_equal(ws.cpu().numpy(), rs)
