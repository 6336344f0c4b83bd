"""Host-side checks of the feed-forward block's operators: the generator's plain form
against its published vectors, and the C ABI's refusals, before any device work."""
import ctypes

import numpy as np
import pytest

import _block as plain
from momijo_amd import _lib


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def test_philox_published_vectors():
    """Philox4x32-10 for the zero and the all-ones counter and key."""
    got = plain.philox4x32(np.array([0], np.uint64), 0, 0)
    assert [hex(v) for v in got[0]] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]
    ones = (1 << 64) - 1
    got = plain.philox4x32(np.array([ones], np.uint64), ones, ones)
    assert [hex(v) for v in got[0]] == ["0x408f276d", "0x41c83b0e", "0xa20bc7c6", "0x6d5451fd"]


def test_dropout_status_codes(lib):
    p = ctypes.c_void_p(16)  # never dereferenced
    assert lib.mj_dropout(7, p, p, 4, 0.1, 0, 0, None, None) == _lib.MJ_ERR_ARG
    assert lib.mj_dropout(0, p, p, -1, 0.1, 0, 0, None, None) == _lib.MJ_ERR_ARG
    assert lib.mj_dropout(0, p, p, 4, 1.1, 0, 0, None, None) == _lib.MJ_ERR_ARG
    assert lib.mj_dropout(0, None, p, 4, 0.1, 0, 0, None, None) == _lib.MJ_ERR_ARG
    assert lib.mj_dropout(0, None, None, 0, 0.1, 0, 0, None, None) == _lib.MJ_OK


def _norm(lib, **kw):
    a = dict(dtype=0, norm=0, x=16, b=16, gate=None, gate_rows=0, scale=None, wp=None, bp=None,
             wn=None, bn=None, eps=1e-6, p=0.0, seed=0, counter=0, state=None, y=16, n=None,
             stats=None, rows=4, dim=8, stream=None)
    a.update(kw)
    return lib.mj_residual_norm(*a.values())


def test_residual_norm_status_codes(lib):
    assert _norm(lib, dtype=3) == _lib.MJ_ERR_ARG
    assert _norm(lib, norm=2) == _lib.MJ_ERR_ARG
    assert _norm(lib, rows=-1) == _lib.MJ_ERR_ARG
    assert _norm(lib, dim=16385) == _lib.MJ_ERR_UNSUPPORTED
    assert _norm(lib, x=None) == _lib.MJ_ERR_ARG
    assert _norm(lib, b=None, wp=16) == _lib.MJ_ERR_ARG
    assert _norm(lib, bp=16) == _lib.MJ_ERR_ARG
    assert _norm(lib, eps=-1.0) == _lib.MJ_ERR_ARG
    assert _norm(lib, gate=16, gate_rows=3) == _lib.MJ_ERR_SHAPE
    assert _norm(lib, gate=16, gate_rows=0) == _lib.MJ_ERR_SHAPE
    assert _norm(lib, y=None) == _lib.MJ_ERR_ARG
    assert _norm(lib, n=16) == _lib.MJ_ERR_ARG
    assert _norm(lib, rows=0) == _lib.MJ_OK and _norm(lib, dim=0) == _lib.MJ_OK


def test_residual_norm_backward_needs_its_work(lib):
    need = lib.mj_residual_norm_work_bytes(100, 64, 0)  # for a call without a gate, as below
    assert need > 0 and need % (64 * 4) == 0
    assert lib.mj_residual_norm_work_bytes(100, 64, 3) == 0
    assert lib.mj_residual_norm_work_bytes(0, 64, 0) == 0
    args = [0, 0, 16, 16, None, 0, None, None, None, None, 0.0, 0, 0, None, 16, 16, None, 16, 16,
            None, None, None, None, None, None, 100, 64]
    assert lib.mj_residual_norm_backward(*args, 16, need - 1, None) == _lib.MJ_ERR_ARG
    assert lib.mj_residual_norm_backward(*args, None, need, None) == _lib.MJ_ERR_ARG
    args[14] = None  # no stats
    assert lib.mj_residual_norm_backward(*args, 16, need, None) == _lib.MJ_ERR_ARG


def test_gated_mlp_status_codes(lib):
    p = ctypes.c_void_p(16)
    big = 1 << 40
    fwd = lambda act, m, k, i, h, x=p, g=None: lib.mj_gated_mlp_bf16(  # noqa: E731
        x, p, p, p, act, p, g, None, p, m, k, i, h, p, big, None)
    assert fwd(4, 4, 8, 8, 8) == _lib.MJ_ERR_UNSUPPORTED      # no gradient for the approximations
    assert fwd(42, 4, 8, 8, 8) == _lib.MJ_ERR_ARG
    assert fwd(3, -1, 8, 8, 8) == _lib.MJ_ERR_ARG
    assert fwd(3, 4, 12, 8, 8) == _lib.MJ_ERR_UNSUPPORTED
    assert fwd(3, 4, 8, 8, 1 << 22) == _lib.MJ_ERR_UNSUPPORTED
    assert fwd(3, 4, 8, 8, 8, ctypes.c_void_p(8)) == _lib.MJ_ERR_UNSUPPORTED
    assert fwd(3, 4, 8, 8, 8, None) == _lib.MJ_ERR_ARG
    assert fwd(3, 4, 8, 8, 8, p, p) == _lib.MJ_ERR_ARG        # g without u
    assert fwd(3, 0, 8, 8, 8) == _lib.MJ_OK
    need = lib.mj_gated_mlp_work_bytes(64, 512, 4096, 64, 0)
    assert need > 0
    assert lib.mj_gated_mlp_bf16(p, p, p, p, 3, p, None, None, p, 64, 512, 4096, 64, p, need - 1,
                                 None) == _lib.MJ_ERR_ARG


def test_gated_mlp_f32_status_codes(lib):
    p, odd = ctypes.c_void_p(16), ctypes.c_void_p(20)
    big = 1 << 40
    fwd = lambda m, k, i, h, g=p, y=p, work=p, nbytes=big, act=3: lib.mj_gated_mlp_f32(  # noqa: E731
        p, p, p, p, act, p, g, p, y, m, k, i, h, work, nbytes, None)
    assert fwd(4, 8, 8, 8, act=42) == _lib.MJ_ERR_ARG
    assert fwd(4, 8, -8, 8) == _lib.MJ_ERR_ARG
    assert fwd(4, 8, 8, 8, g=None) == _lib.MJ_ERR_ARG
    assert fwd(4, 8, 8, 8, y=None) == _lib.MJ_ERR_ARG
    assert fwd(4, 8, 8, 8, g=odd) == _lib.MJ_ERR_UNSUPPORTED
    assert fwd(4, 8, 8, 8, y=odd) == _lib.MJ_ERR_UNSUPPORTED
    assert fwd(0, 8, 8, 8) == _lib.MJ_OK
    need = lib.mj_gated_mlp_f32_work_bytes(64, 64, 4096, 64, 0)
    assert need > 0
    assert fwd(64, 64, 4096, 64, work=None) == _lib.MJ_ERR_ARG
    assert fwd(64, 64, 4096, 64, nbytes=need - 1) == _lib.MJ_ERR_ARG
    assert lib.mj_gated_mlp_f32_work_bytes(0, 64, 4096, 64, 0) == 0


@pytest.mark.parametrize("name", ["mj_gated_mlp_backward_bf16", "mj_gated_mlp_backward_f32"])
def test_gated_mlp_backward_status_codes(lib, name):
    p, odd = 16, 20
    work = lib.mj_gated_mlp_work_bytes if name.endswith("bf16") else lib.mj_gated_mlp_f32_work_bytes

    def bwd(M=64, K=64, I=4096, H=64, act=3, work=p, nbytes=1 << 40, **at):
        a = dict(x=p, Wg=p, Wu=p, Wd=p, h=p, g=p, u=p, dy=p, dg=p, du=p, dx=p, dWg=p, dWu=p, dWd=p)
        a.update(at)
        return getattr(lib, name)(a["x"], a["Wg"], a["Wu"], a["Wd"], act, a["h"], a["g"], a["u"],
                                  a["dy"], a["dg"], a["du"], a["dx"], a["dWg"], a["dWu"], a["dWd"],
                                  M, K, I, H, work, nbytes, None)

    assert bwd(act=4) == _lib.MJ_ERR_UNSUPPORTED
    assert bwd(M=-1) == _lib.MJ_ERR_ARG
    for operand in ("x", "Wg", "Wd", "g", "dy", "dg", "h"):
        assert bwd(**{operand: None}) == _lib.MJ_ERR_ARG, operand
    for operand in ("g", "u", "dg", "du", "dx"):
        assert bwd(**{operand: odd}) == _lib.MJ_ERR_UNSUPPORTED, operand
    need = work(64, 64, 4096, 64, 1)
    assert need > 0
    assert bwd(work=None) == _lib.MJ_ERR_ARG
    assert bwd(nbytes=need - 1) == _lib.MJ_ERR_ARG


def test_copy_rows_status_codes(lib):
    ptrs = (ctypes.c_void_p * 1)(16)
    call = lambda n, *z: lib.mj_copy_rows_bf16(n, ptrs, ptrs, (ctypes.c_int64 * 6)(*z), None)  # noqa: E731
    assert call(0, 1, 1, 1, 1, 1, 1) == _lib.MJ_ERR_ARG
    assert call(5, 1, 1, 1, 1, 1, 1) == _lib.MJ_ERR_ARG
    assert call(1, -1, 1, 1, 1, 1, 1) == _lib.MJ_ERR_ARG
    assert call(1, 2, 4, 3, 2, 4, 4) == _lib.MJ_ERR_SHAPE     # source rows overlap
    assert call(1, 2, 4, 4, 2, 8, 4) == _lib.MJ_ERR_SHAPE
    assert lib.mj_copy_rows_bf16(1, None, ptrs, (ctypes.c_int64 * 6)(), None) == _lib.MJ_ERR_ARG
    null = (ctypes.c_void_p * 1)()
    assert lib.mj_copy_rows_bf16(1, null, ptrs, (ctypes.c_int64 * 6)(2, 2, 2, 2, 2, 2), None) == _lib.MJ_ERR_ARG
    assert call(1, 0, 0, 0, 0, 0, 0) == _lib.MJ_OK


@pytest.mark.parametrize("M,I,N", [(200, 6912, 2560), (64, 4096, 64), (48, 11008, 4096)])
def test_gated_mlp_work_of_a_zero_width(lib, M, I, N):
    """y [M, N] (or dx) is summed in K slices whatever the width it does not depend on:
    with that width zero it needs the same work, and a call without is refused."""
    p, big = ctypes.c_void_p(16), 1 << 40
    need = lib.mj_gated_mlp_work_bytes(M, 64, I, N, 0)
    assert need > 0
    assert lib.mj_gated_mlp_work_bytes(M, 0, I, N, 0) == need
    assert lib.mj_gated_mlp_bf16(None, p, p, p, 3, p, None, None, p, M, 0, I, N, None, 0,
                                 None) == _lib.MJ_ERR_ARG
    need = lib.mj_gated_mlp_work_bytes(M, N, I, 64, 1)
    assert need > 0
    assert lib.mj_gated_mlp_work_bytes(M, N, I, 0, 1) == need
    assert lib.mj_gated_mlp_backward_bf16(p, p, p, p, 3, p, p, p, None, p, p, p, p, p, p, M, N, I, 0,
                                          None, big, None) == _lib.MJ_ERR_ARG
    for zero in ((0, N, I, N), (M, N, 0, N)):
        assert lib.mj_gated_mlp_work_bytes(*zero, 0) == lib.mj_gated_mlp_work_bytes(*zero, 1) == 0
    assert lib.mj_gated_mlp_work_bytes(M, N, I, 0, 0) == lib.mj_gated_mlp_work_bytes(M, 0, I, N, 1) == 0


def test_gated_mlp_most_rows(lib):
    """Beyond 2^31 - 1024 rows the tiles' row numbers would overflow: refused."""
    p = ctypes.c_void_p(16)
    for m, status in (((1 << 31) - 1023, _lib.MJ_ERR_UNSUPPORTED), ((1 << 31) - 1, _lib.MJ_ERR_UNSUPPORTED),
                      (0, _lib.MJ_OK)):
        assert lib.mj_gated_mlp_bf16(p, p, p, p, 3, p, None, None, p, m, 8, 8, 8, None, 0, None) == status
        assert lib.mj_gated_mlp_backward_bf16(p, p, p, p, 3, p, p, p, p, p, p, None, None, None, None, m, 8,
                                              8, 8, None, 0, None) == status


def test_residual_norm_of_x_itself(lib):
    """y = x is no work, but the other arguments are checked as in any call."""
    alone = dict(b=None, x=16, y=16)
    assert _norm(lib, **alone) == _lib.MJ_OK
    for bad in (dict(p=0.5), dict(p=2.0), dict(gate=16, gate_rows=1), dict(wp=16), dict(bp=16), dict(bn=16),
                dict(eps=-1.0), dict(dim=16385), dict(norm=2), dict(n=16)):
        assert _norm(lib, **{**alone, **bad}) != _lib.MJ_OK, bad
