"""Host checks of the mixture of experts and the 8-bit products that need no GPU: the C ABI's
refusals and sizes (before any device work), and the plain forms that the GPU tests compare
with, against torch's autograd and its 8-bit type."""
import ctypes

import numpy as np
import pytest
import torch

import _experts as plain
import momijo_amd as mj
from momijo_amd import _lib


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


P, ODD = 16, 24          # pointers that no call dereferences: validation fails first
ROWS = (1 << 31) - 1024  # most slots
OK, ARG, BAD = _lib.MJ_OK, _lib.MJ_ERR_ARG, _lib.MJ_ERR_UNSUPPORTED


def _call(lib, name, order, **at):
    return getattr(lib, name)(*[at[k] for k in order], None)


# ------------------------------------------------------------------ rows
def test_sort_status_codes(lib):
    def sort(**at):
        a = dict(ids=P, size=8, slots=16, experts=4, pos=P, offsets=P, work=None, nbytes=0)
        a.update(at)
        return _call(lib, "mj_sort_experts", a, **a)

    for bad in (dict(size=2), dict(experts=0), dict(experts=1025), dict(slots=-1), dict(ids=None),
                dict(pos=None), dict(offsets=None), dict(slots=8193), dict(slots=8193, work=P, nbytes=8)):
        assert sort(**bad) == ARG, bad
    assert sort(slots=ROWS + 1) == BAD
    work = lib.mj_sort_experts_work_bytes
    assert work(8192, 64) == 0 and work(8193, 64) > 0 and work(8193, 0) == 0 == work(0, 64)
    assert work(8193, 1024) == 4 * (3 + 1) * 1025      # 4096 slots a workgroup, and the totals


def test_row_status_codes(lib):
    shared = dict(pos=P, offsets=P, experts=4)

    def dispatch(**at):
        a = dict(dtype=1, x=P, weights=None, **shared, xs=P, ws=None, tokens=3, topk=2, dim=8)
        a.update(at)
        return _call(lib, "mj_dispatch", a, **a)

    def combine(**at):
        a = dict(dtype=1, to=1, ys=P, weights=None, **shared, y=P, tokens=3, topk=2, dim=8)
        a.update(at)
        return _call(lib, "mj_combine", a, **a)

    def backward(**at):
        a = dict(dtype=1, dy=P, ys=P, weights=P, **shared, dys=P, dw=P, tokens=3, topk=2, dim=8)
        a.update(at)
        return _call(lib, "mj_combine_backward", a, **a)

    for call in (dispatch, combine, backward):
        for bad in (dict(dtype=2), dict(experts=0), dict(experts=1025), dict(tokens=-1), dict(topk=-1),
                    dict(dim=-1), dict(pos=None), dict(offsets=None)):
            assert call(**bad) == ARG, (call, bad)
        assert call(tokens=ROWS // 2 + 1) == BAD
        assert call(tokens=0) == OK
    for bad in (dict(x=None), dict(xs=None), dict(weights=P), dict(ws=P)):
        assert dispatch(**bad) == ARG, bad
    assert dispatch(topk=0) == OK == dispatch(dim=0)
    assert combine(ys=None) == ARG == combine(y=None) and combine(to=7) == ARG
    assert combine(to=0) == BAD                        # bf16 rows do not give fp32 sums
    assert combine(dim=0) == OK
    for bad in (dict(dy=None), dict(ys=None), dict(dys=None), dict(dw=None), dict(weights=None)):
        assert backward(**bad) == ARG, bad
    assert backward(topk=0) == OK


# ------------------------------------------------------------------ the experts' block
_FWD = ["xs", "offsets", "experts", "wg", "wu", "wd", "act", "weights", "h", "g", "u", "ys", "R", "K", "I", "H"]
_BWD = _FWD[:11] + ["dys", "dg", "du", "dxs", "dwg", "dwu", "dwd", "pos", "slots", "dots", "dw", "R", "K", "I", "H"]


def _mlp(lib, name, order, **at):
    a = dict.fromkeys(order, P)
    a.update(experts=4, act=3, slots=8, R=8, K=16, I=24, H=8, weights=None)
    a.update(at)
    return _call(lib, name, order, **a)


@pytest.mark.parametrize("name,order", [("mj_experts_mlp_bf16", _FWD), ("mj_experts_mlp_backward_bf16", _BWD)])
def test_experts_mlp_status_codes(lib, name, order):
    call = lambda **at: _mlp(lib, name, order, **at)  # noqa: E731
    for bad in (dict(act=42), dict(experts=0), dict(experts=1025), dict(R=-1), dict(K=-8), dict(offsets=None)):
        assert call(**bad) == ARG, bad
    for bad in (dict(act=4), dict(K=12), dict(I=20), dict(H=4), dict(H=1 << 22), dict(R=ROWS + 1), dict(xs=ODD),
                dict(wg=ODD), dict(h=ODD), dict(g=ODD)):
        assert call(**bad) == BAD, bad
    need = ("xs", "wg", "wu", "wd", "h", "ys") if order is _FWD else ("xs", "wg", "wd", "h", "g", "u", "dys", "dg",
                                                                    "pos", "dots")
    for operand in need:
        assert call(**{operand: None}) == ARG, operand
    if order is _FWD:
        assert call(g=None) == ARG and call(R=0) == OK
    else:
        assert call(slots=-1) == ARG


def test_experts_mlp_dots(lib):
    dots = lib.mj_experts_mlp_dots
    assert dots(0, 4, 16, 24, 8) == 0 == dots(8, 4, 16, 0, 8) == dots(8, 0, 16, 24, 8)
    for R, E, I, H in ((8, 4, 24, 8), (1000, 7, 712, 104), (8192, 8, 5504, 4096), (300, 1024, 8, 8)):
        n = dots(R, E, 16, I, H)
        assert n % R == 0 and I / 64 <= n // R <= max(8, I / 32 + 8)   # one for each wave of 32 or 64 columns


# ------------------------------------------------------------------ 8-bit floating point
def test_f8_status_codes(lib):
    q = lib.mj_quantize_rows_f8
    assert q(2, P, P, P, 4, 16, None) == ARG and q(1, P, P, P, -1, 16, None) == ARG
    assert q(1, P, P, P, 4, 24, None) == BAD == q(1, ODD, P, P, 4, 16, None) == q(1, P, P, P, ROWS + 1, 16, None)
    assert q(1, None, P, P, 4, 16, None) == ARG and q(1, None, None, None, 0, 16, None) == OK
    b = lib.mj_quantize_blocks_f8
    assert b(1, P, P, P, -1, 4, 16, None) == ARG and b(1, P, P, P, 1, 4, 8, None) == BAD
    assert b(1, P, P, None, 1, 4, 16, None) == ARG and b(0, None, None, None, 1, 0, 16, None) == OK
    d = lib.mj_dispatch_f8
    assert d(1, P, P, P, 0, P, P, 4, 2, 16, None) == ARG and d(1, P, P, P, 4, P, P, 4, 2, 24, None) == BAD
    assert d(1, P, P, P, 4, None, P, 4, 2, 16, None) == ARG and d(1, P, P, P, 4, P, P, 0, 2, 16, None) == OK
    big = 1 << 40

    def gemm(x=P, sx=P, w=P, sw=P, bias=None, act=0, y=P, M=4, N=8, K=16, work=P, nbytes=big):
        return lib.mj_gemm_f8(x, sx, w, sw, bias, act, y, M, N, K, work, nbytes, None)

    for bad in (dict(act=42), dict(M=-1), dict(N=-1), dict(x=None), dict(sx=None), dict(w=None), dict(sw=None),
                dict(y=None)):
        assert gemm(**bad) == ARG, bad
    for bad in (dict(act=4), dict(K=24), dict(K=1 << 22), dict(M=ROWS + 1), dict(x=ODD), dict(w=ODD), dict(y=ODD)):
        assert gemm(**bad) == BAD, bad
    assert gemm(M=0) == OK == gemm(N=0)
    need = lib.mj_gemm_f8_work_bytes(48, 4096, 11008)  # K slices
    assert need > 0 and gemm(M=48, N=4096, K=11008, nbytes=need - 1) == ARG

    def linear(dtype=1, x=P, w=P, sw=P, act=0, y=P, M=64, N=512, K=1024, work=P, nbytes=big):
        return lib.mj_linear_f8(dtype, x, w, sw, None, act, y, M, N, K, work, nbytes, None)

    for bad in (dict(dtype=2), dict(act=42), dict(x=None), dict(w=None), dict(sw=None), dict(y=None), dict(work=None),
                dict(nbytes=lib.mj_linear_f8_work_bytes(64, 512, 1024) - 1)):
        assert linear(**bad) == ARG, bad
    for bad in (dict(act=4), dict(K=24), dict(x=ODD), dict(work=ODD), dict(y=ODD)):
        assert linear(**bad) == BAD, bad
    assert lib.mj_linear_f8_work_bytes(64, 512, 1024) >= 64 * 1024 + 4 * 64 * 8
    assert lib.mj_linear_f8_work_bytes(1, 512, 1024) == 0      # quantized by the product's workgroups

    def experts(x=P, sx=P, offsets=P, E=4, w=P, sw=P, y=P, R=8, N=16, K=16):
        return lib.mj_experts_gemm_f8(x, sx, offsets, E, w, sw, y, R, N, K, None)

    for bad in (dict(x=None), dict(offsets=None), dict(E=0), dict(E=1025), dict(w=None), dict(y=None), dict(R=-1)):
        assert experts(**bad) == ARG, bad
    assert experts(K=8) == BAD == experts(y=ODD) and experts(R=0) == OK

    def gate(x=P, E=4, wg=P, wu=P, su=P, act=3, hq=P, R=8, I=16, K=16, work=P, nbytes=big):
        return lib.mj_experts_gate_f8(x, P, P, E, wg, P, wu, su, act, hq, P, R, I, K, work, nbytes, None)

    for bad in (dict(act=42), dict(E=0), dict(wg=None), dict(wu=None), dict(su=None), dict(hq=None), dict(work=None),
                dict(nbytes=4 * 8 * 16 - 1)):
        assert gate(**bad) == ARG, bad
    for bad in (dict(act=4), dict(I=8), dict(K=8), dict(hq=ODD), dict(wu=ODD)):
        assert gate(**bad) == BAD, bad
    assert lib.mj_experts_gate_f8_work_bytes(8192, 8, 5504, 4096) == 0     # h quantized by the product's tiles


def test_classes_refuse_on_the_host():
    z = torch.zeros
    with pytest.raises(ValueError):
        mj.ExpertsMLP(z(2, 8, 8), z(2, 8, 8), z(3, 8, 8))
    with pytest.raises(ValueError):
        mj.sort_experts(z(4, 2, dtype=torch.int64), 4)          # not on the GPU
    with pytest.raises(ValueError):
        mj.ExpertPlan(z(4, 2, dtype=torch.int64), z(5, dtype=torch.int32))
    with pytest.raises(ValueError):
        mj.F8Linear(z(32, 48), z(1, 1))
    with pytest.raises(ValueError):
        mj.F8Linear(z(32, 48).to(torch.float8_e4m3fn), z(1, 2))
    plan = mj.ExpertPlan(z(4, 2, dtype=torch.int32), z(5, dtype=torch.int32))
    assert (plan.tokens, plan.topk, plan.rows, plan.experts) == (4, 2, 8, 4)
    for bad in (lambda: mj.dispatch(z(4, 8), plan), lambda: mj.combine(z(8, 8), None, plan),
                lambda: mj.dispatch_fp8(z(4, 16), plan), lambda: mj.quantize_rows_fp8(z(4, 16)),
                lambda: mj.F8Linear(z(32, 48).to(torch.float8_e4m3fn), z(1, 1)).forward(z(2, 48))):
        with pytest.raises(ValueError):
            bad()


# ------------------------------------------------------------------ the plain forms
def test_plain_sort():
    ids = torch.tensor([[2, 0], [5, 2], [-1, 1], [0, 2]])
    pos, offsets = plain.sort(ids, 3)
    assert pos.tolist() == [[3, 0], [6, 4], [7, 2], [1, 5]] and offsets.tolist() == [0, 2, 3, 6]


@pytest.mark.parametrize("act", ["silu", "gelu", "relu", "none"])
def test_plain_mlp_against_autograd(act):
    g = torch.Generator().manual_seed(len(act))
    T, k, E, K, I, H = 9, 2, 4, 6, 5, 7
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    ids = torch.randint(-1, E, (T, k), generator=g)
    v = dict(x=r(T, K), weights=r(T, k), gate=r(E, I, K), up=r(E, I, K), down=r(E, H, I))
    dy = r(T, H)
    pos, offsets = plain.sort(ids, E)
    ref = plain.mlp(v["x"], pos, offsets, v["weights"], v["gate"], v["up"], v["down"], dy, act, 0.0, 0.0)
    for t in v.values():
        t.requires_grad_(True)
    f = {"relu": torch.relu, "silu": torch.nn.functional.silu, "none": lambda t: t,
         "gelu": lambda t: torch.nn.functional.gelu(t, approximate="tanh")}[act]
    y = torch.zeros(T, H, dtype=torch.float64)
    for t in range(T):
        for j in range(k):
            e = int(ids[t, j])
            if e >= 0:
                x = v["x"][t]
                h = f(v["gate"][e] @ x) * (v["up"][e] @ x)
                y = y + torch.nn.functional.one_hot(torch.tensor(t), T).double()[:, None] * (
                    v["weights"][t, j] * (v["down"][e] @ h))
    assert torch.allclose(ref["y"][0], y.detach(), rtol=1e-12, atol=1e-12)
    for name, d in zip(v, torch.autograd.grad(y, list(v.values()), dy)):
        assert torch.allclose(ref[name][0], d, rtol=1e-11, atol=1e-11), name


def test_plain_e4m3_is_torchs():
    """Every e4m3 value, the middles between neighbours and their float32 neighbours."""
    v = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    mid = (v[:-1] + v[1:]) / 2
    x = np.concatenate([v, mid, np.nextafter(mid, np.float32(0)), np.nextafter(mid, np.float32(999))]).astype(np.float32)
    x = np.concatenate([x, -x])
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(plain.e4m3(x), want)


def test_plain_quantization_keeps_its_bound():
    """A value is off by at most half a step: 2^-4 of it, or 2^-10 of the scale near zero."""
    x = np.random.default_rng(3).standard_normal((20, 300)).astype(np.float32) * np.float32(10) ** np.arange(-8, 12)[:, None]
    q, s = plain.quantize_rows(x)
    wide = np.repeat(s.T, 128, axis=1)[:, :300].astype(np.float64)
    assert np.all(np.abs(q * wide - x) <= np.maximum(np.abs(x) * (2.0 ** -4 + 2.0 ** -20), wide * 2.0 ** -10 * 1.001))
    assert np.abs(q).max() == 448
