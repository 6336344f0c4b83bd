"""The block-scaled 8-bit Linear and experts on the GPU against 64-bit plain forms.

Quantization is exact to the bit: its Float32 steps are the definition.  A product's bound: its sum
is off by what _experts.f8_error derives, the activation by 2^-18 and the output by a rounding
to bf16, 2^-8 relative.
"""
import zlib

import numpy as np
import pytest
import torch

import _block as block
import _experts as plain
import momijo_amd as mj

pytestmark = pytest.mark.gpu

ACTS = {"none": mj.EPI_NONE, "relu": mj.EPI_RELU, "gelu": mj.EPI_GELU_TANH, "silu": mj.EPI_SILU}
F8 = torch.float8_e4m3fn


def _gen(*key):
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(repr(key).encode()))


def _normal(g, shape, dt=torch.float32, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dt)


def _close(got, want, bound, name):
    got = got.to(want.device, torch.float64)
    assert got.shape == want.shape, (name, got.shape, want.shape)
    bad = ~((got - want).abs() <= bound)
    assert not bool(bad.any()), (
        f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {float((got - want).abs().max()):.3e}, "
        f"first at {torch.nonzero(bad)[0].tolist()}")


def _bits(q, want):
    """q holds want's values, zeros of any sign alike."""
    return np.array_equal(q.float().cpu().numpy(), want)


# ------------------------------------------------------------------ quantization
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,K", [(0, 16), (1, 16), (3, 128), (5, 144), (17, 4096), (300, 1040), (33, 11008)])
def test_quantize_rows(dev, M, K, dt):
    x = _normal(_gen(M, K), (M, K), dt)
    x *= torch.exp2(torch.randint(-30, 30, (M, 1), generator=_gen(K), device="cuda")).to(dt)
    q, s = mj.quantize_rows_fp8(x)
    rq, rs = plain.quantize_rows(x.float().cpu().numpy())
    assert q.dtype is F8 and np.array_equal(s.cpu().numpy(), rs) and _bits(q, rq)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 16), (128, 128), (130, 144), (300, 1040), (3, 200, 272)])
def test_quantize_blocks(dev, shape, dt):
    w = _normal(_gen(shape), shape, dt, 0.02)
    q, s = mj.quantize_blocks_fp8(w)
    for i in range(shape[0] if len(shape) == 3 else 1):
        at = i if len(shape) == 3 else ...
        rq, rs = plain.quantize_blocks(w[at].float().cpu().numpy())
        assert np.array_equal(s[at].cpu().numpy(), rs) and _bits(q[at], rq)


def test_quantize_special_values(dev):
    """Every tie and step of e4m3, blocks of zeros, tiny and huge blocks; NaN and infinity."""
    x = torch.zeros(9, 128, device="cuda")
    x[0, :127] = torch.arange(127, device="cuda") * 0.25 / 512      # steps below the normal numbers, ties
    x[0, 127] = 448.0
    x[1, :100] = torch.arange(1, 101, device="cuda") * 0.53125
    x[1, 100] = -448.0
    x[3] = 2.0 ** -120
    x[4] = 3e38
    x[5, 3] = 1e-38
    x[6, 5], x[6, 6] = float("nan"), 2.0
    x[7, 5], x[7, 6] = float("inf"), 2.0
    x[8] = -2.0 ** -100
    q, s = mj.quantize_rows_fp8(x)
    keep = [0, 1, 2, 3, 4, 5, 8]
    rq, rs = plain.quantize_rows(x[keep].cpu().numpy())
    assert _bits(q[keep], rq) and np.array_equal(s[:, keep].cpu().numpy(), rs)
    f = q.float().cpu()
    assert not bool(f[2].any()) and bool(torch.isnan(f[6, 5])) and float(f[6, 6]) == 448.0
    assert bool(torch.isnan(f[7, 5])) and float(s[0, 7]) == float("inf")


# ------------------------------------------------------------------ products
# rows, N, K: one row, few rows, across the few-row kernel, the tiles and their edges, widths that
# end inside a block, odd N, K slices, one and several rounds of large tiles
_LINEAR = [(1, 1, 16), (1, 64, 128), (1, 11008, 4096), (2, 40, 4096), (3, 129, 144), (16, 300, 1040),
           (17, 256, 272), (33, 1000, 512), (48, 4096, 11008), (65, 72, 4112), (100, 129, 160),
           (128, 128, 128), (129, 640, 2048), (257, 333, 528), (300, 1000, 1040), (1000, 3000, 1040),
           (513, 2048, 4096), (2048, 4096, 1024), (4096, 4104, 528)]


@pytest.mark.parametrize("M,N,K", _LINEAR)
def test_linear(dev, M, N, K):
    act = ["none", "silu", "gelu", "relu"][(M + N) % 4]
    g = _gen(M, N, K)
    x = _normal(g, (M, K), torch.bfloat16 if M % 2 else torch.float32)
    q, s = mj.quantize_blocks_fp8(_normal(g, (N, K), std=K ** -0.5))
    bias = _normal(g, (N,)) if N % 3 == 0 else None
    lin = mj.F8Linear(q, s, bias, ACTS[act])
    y = lin.forward(x)
    xq, xs = mj.quantize_rows_fp8(x)
    assert torch.equal(y, mj.gemm_fp8_nt(xq, xs, q, s, bias, ACTS[act]))
    a, w = plain.rows_f64(xq, xs), plain.blocks_f64(q, s)
    v, e = a @ w.t(), plain.f8_error(a, w)
    if bias is not None:
        v = v + bias.double()
    e = 1.2 * (e + 2.0 ** -24 * v.abs())   # |act'| <= 1.2
    v = block.act(act, v)[0]
    _close(y, v, e + 2.0 ** -18 * v.abs() + 2.0 ** -8 * (v.abs() + e) + 1e-30, "y")


def test_linear_shapes(dev):
    g = _gen("shapes")
    lin = mj.F8Linear.from_float(_normal(g, (72, 160)))
    x = _normal(g, (2, 3, 160), torch.bfloat16)
    y = lin.forward(x)
    assert y.shape == (2, 3, 72) and torch.equal(y.reshape(6, 72), lin.forward(x.reshape(6, 160)))
    assert torch.equal(lin.forward(x[0, 0]), y[0, 0])
    assert lin.forward(x[:0]).shape == (0, 3, 72)
    off = torch.empty(6 * 160 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(2, 3, 160).copy_(x)
    assert torch.equal(lin.forward(off), y)
    assert torch.equal(lin.forward(x.transpose(0, 1).contiguous().transpose(0, 1)), y)


def test_linear_scales_span_fp32(dev):
    """Rows and blocks far apart in magnitude: each output to its own size."""
    g = _gen("span")
    x, w = _normal(g, (40, 512)), _normal(g, (300, 512))
    x *= torch.exp2(torch.arange(40, device="cuda") * 2.0 - 40)[:, None]
    x[:, 128:256] *= 2.0 ** -20
    w[128:256] *= 2.0 ** 30
    w[:, 256:384] *= 2.0 ** -30
    q, s = mj.quantize_blocks_fp8(w)
    xq, xs = mj.quantize_rows_fp8(x)
    y = mj.gemm_fp8_nt(xq, xs, q, s)
    a, b = plain.rows_f64(xq, xs), plain.blocks_f64(q, s)
    v, e = a @ b.t(), plain.f8_error(a, b)
    _close(y, v, e + 2.0 ** -8 * (v.abs() + e), "y")


def test_linear_nan_and_inf_stay_in_their_row(dev):
    g = _gen("nan")
    for M in (5, 40, 300):
        lin = mj.F8Linear.from_float(_normal(g, (200, 272)))
        x = _normal(g, (M, 272), torch.bfloat16)
        y = lin.forward(x)
        x[1, 7], x[3, 260] = float("nan"), float("inf")
        z = lin.forward(x)
        keep = [i for i in range(M) if i not in (1, 3)]
        assert torch.equal(z[keep], y[keep]) and not bool(torch.isfinite(z[[1, 3]]).any())


def test_linear_captured(dev):
    g = _gen("captured")
    for M in (1, 48, 300):
        lin = mj.F8Linear.from_float(_normal(g, (520, 4096)))
        x = _normal(g, (M, 4096), torch.bfloat16)
        lin.forward(x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = lin.forward(x)
        for _ in range(3):
            x.copy_(_normal(g, (M, 4096), torch.bfloat16))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, lin.forward(x))


# ------------------------------------------------------------------ experts
def _ids(g, T, k, E, kind):
    ids = torch.randint(0, E, (T, k), generator=g, device="cuda")
    if kind == "one":
        ids.fill_(E - 1)
    elif kind == "drop":
        ids = torch.where(torch.randint(0, 3, (T, k), generator=g, device="cuda") == 0, -1, ids)
    elif kind == "none":
        ids.fill_(-1)
    return ids


_EXPERTS = [(1, 1, 1, 16, 16, 16, "even"), (1, 2, 8, 4096, 1376, 512, "even"), (7, 3, 5, 144, 272, 80, "drop"),
            (48, 2, 8, 512, 704, 512, "even"), (40, 2, 4, 272, 144, 272, "one"), (300, 2, 3, 528, 400, 336, "drop"),
            (1000, 3, 16, 256, 512, 256, "drop"), (700, 2, 70, 128, 144, 128, "even"),
            (2048, 2, 4, 1040, 2064, 1056, "drop"), (33, 2, 4, 64, 64, 64, "none")]


@pytest.mark.parametrize("T,k,E,K,I,H,kind", _EXPERTS)
def test_experts(dev, T, k, E, K, I, H, kind):
    """Each step from the step before as it is on the device, so that a value next to a border of
    e4m3 falls on one side in both: dispatch exact, h within its quantization, y as a product."""
    act = ["silu", "gelu", "relu", "none"][(T + K) % 4]
    g = _gen(T, k, E, K, I, H)
    ids, w = _ids(g, T, k, E, kind), _normal(g, (T, k))
    x = _normal(g, (T, K), torch.bfloat16)
    f = mj.F8Experts.from_float(*(_normal(g, s, std=s[2] ** -0.5) for s in ((E, I, K), (E, I, K), (E, H, I))),
                                ACTS[act])
    plan = mj.sort_experts(ids, E)
    pos, offsets = plan.pos.long(), plan.offsets.tolist()
    kept = offsets[-1]
    q, s = mj.dispatch_fp8(x, plan)
    xq, xs = mj.quantize_rows_fp8(x)
    for j in range(k):
        on = pos[:, j] < kept
        assert torch.equal(q.view(torch.uint8)[pos[on, j]], xq.view(torch.uint8)[on])
        assert torch.equal(s[:, pos[on, j]], xs[:, on])
    assert not bool(q[kept:].float().any())
    hq, hs = mj.experts_gate_fp8(q, s, plan, f.gate, f.gate_scales, f.up, f.up_scales, f.act)
    ys = mj.experts_gemm_fp8(hq, hs, plan, f.down, f.down_scales)
    assert not bool(hq[kept:].float().any()) and not bool(ys[kept:].any())
    a, hv = plain.rows_f64(q, s), plain.rows_f64(hq, hs)
    for e in range(E):
        r = slice(offsets[e], offsets[e + 1])
        if r.start == r.stop:
            continue
        wg, wu, wd = (plain.blocks_f64(m[e], c[e]) for m, c in
                      ((f.gate, f.gate_scales), (f.up, f.up_scales), (f.down, f.down_scales)))
        v, u = a[r] @ wg.t(), a[r] @ wu.t()
        ev, eu = plain.f8_error(a[r], wg), plain.f8_error(a[r], wu)
        av = block.act(act, v)[0]
        eav = 1.2 * ev + 2.0 ** -18 * av.abs()
        h, eh = av * u, eav * u.abs() + av.abs() * eu + eav * eu + 2.0 ** -24 * (av * u).abs()
        # a value moves by half a step: 2^-4 of it, or 2^-10 of the scale below e4m3's normal
        # numbers; the scale is that of the block's largest, which may be off by its own error
        step = hs[:, r].double().t().repeat_interleave(128, 1)[:, :I] * 2.0 ** -10
        _close(hv[r], h, eh + (h.abs() + eh) * (2.0 ** -4 * (1 + 2.0 ** -20)) + step * 1.001, "h")
        top = torch.nn.functional.pad(h.abs() + eh, (0, -I % 128)).reshape(-1, hs.shape[0], 128).amax(2)
        low = torch.nn.functional.pad(h.abs() - eh, (0, -I % 128)).reshape(-1, hs.shape[0], 128).amax(2)
        sc = hs[:, r].double().t() * 448
        assert bool((sc <= top.clamp_min(2.0 ** -100) * (1 + 2.0 ** -22)).all())
        assert bool((sc >= low * (1 - 2.0 ** -22)).all())
        y, ey = hv[r] @ wd.t(), plain.f8_error(hv[r], wd)
        _close(ys[r], y, ey, "ys")
    assert torch.equal(f.forward(x, ids, w), mj.combine(ys, w, plan, torch.bfloat16))


def test_experts_captured(dev):
    g = _gen("experts captured")
    T, k, E, K, I = 70, 2, 5, 144, 272
    f = mj.F8Experts.from_float(*(_normal(g, s, std=0.1) for s in ((E, I, K), (E, I, K), (E, K, I))))
    fresh = lambda: (_normal(g, (T, K), torch.bfloat16), _ids(g, T, k, E, "drop"), _normal(g, (T, k)))  # noqa: E731
    held = fresh()
    f.forward(*held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = f.forward(*held)
    for _ in range(3):
        new = fresh()
        for a, b in zip(held, new):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, f.forward(*new))


def test_refusals(dev):
    w = torch.zeros(32, 48, device="cuda")
    q, s = mj.quantize_blocks_fp8(w)
    xq, xs = mj.quantize_rows_fp8(torch.zeros(4, 48, device="cuda"))
    lin = mj.F8Linear(q, s)
    plan = mj.sort_experts(torch.zeros(2, 2, dtype=torch.int64, device="cuda"), 1)
    for bad in (lambda: mj.F8Linear(w, s), lambda: mj.F8Linear(q, s[:, :0]), lambda: mj.F8Linear(q, s.double()),
                lambda: mj.F8Linear(q, s, torch.zeros(31, device="cuda")),
                lambda: mj.F8Linear(q, s, None, mj.EPI_SILU_APPROX).forward(torch.zeros(4, 48, device="cuda")),
                lambda: lin.forward(torch.zeros(4, 32, device="cuda")),
                lambda: lin.forward(torch.zeros(4, 48, device="cuda").half()), lambda: lin.forward(torch.zeros(4, 48)),
                lambda: mj.quantize_rows_fp8(torch.zeros(4, 24, device="cuda")),
                lambda: mj.quantize_blocks_fp8(torch.zeros(4, 24, device="cuda")),
                lambda: mj.quantize_rows_fp8(torch.zeros(48, device="cuda")),
                lambda: mj.gemm_fp8_nt(xq, xs.t(), q, s), lambda: mj.gemm_fp8_nt(xq[:, :32], xs, q, s),
                lambda: mj.gemm_fp8_nt(xq, xs, q[None], s[None]),
                lambda: mj.experts_gemm_fp8(xq, xs, plan, q, s),
                lambda: mj.experts_gemm_fp8(xq[:3], xs[:, :3], plan, q[None], s[None]),
                lambda: mj.experts_gemm_fp8(xq, xs, plan, torch.cat([q, q]).view(2, 32, 48), torch.stack([s, s])),
                lambda: mj.F8Experts(q[None], s[None], q[None], s[None], q[None], s[None])):
        with pytest.raises((TypeError, ValueError, mj.MomijoHipError)):
            bad()
