"""The mixture of experts on the GPU against its 64-bit plain forms: sort, dispatch,
combine and the experts' gated blocks, forward and backward.

Bounds, derived per element: a rounding to bf16 is off by up to 2^-8 relative (fp32
2^-24); a sum of n fp32 terms one after another by up to n 2^-24 of the sum of their
magnitudes; sums on the matrix cores and the activations by 2^-18 of it (as the feed-forward
block's tests).  The sort, copies and zeros are exact.
"""
import zlib

import pytest
import torch

import _experts as plain
import momijo_amd as mj

pytestmark = pytest.mark.gpu

ACTS = {"none": mj.EPI_NONE, "relu": mj.EPI_RELU, "gelu": mj.EPI_GELU_TANH, "silu": mj.EPI_SILU}
DT = {"bf16": torch.bfloat16, "f32": torch.float32}
UNIT = {"bf16": 2.0 ** -8, "f32": 2.0 ** -24}


def _gen(*key):
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(repr(key).encode()))


def _normal(g, shape, dt=torch.float32, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dt)


def _ids(g, T, k, E, kind="even"):
    """Experts of T tokens: even, all of one expert (one), half of them dropped (drop), all
    dropped (none), each token's the same one k times (same), or so many of each expert and,
    last, so many dropped (a tuple)."""
    if isinstance(kind, tuple):
        all_ids = torch.repeat_interleave(torch.arange(E + 1), torch.tensor(kind)).to("cuda")
        return all_ids[torch.randperm(T * k, generator=g, device="cuda")].reshape(T, k)
    ids = torch.randint(0, E, (T, k), generator=g, device="cuda")
    if kind == "one":
        ids.fill_(E // 2)
    elif kind == "drop":
        off = torch.randint(0, 4, (T, k), generator=g, device="cuda")
        ids = torch.where(off == 0, -1, torch.where(off == 1, E + ids, ids))
    elif kind == "none":
        ids.fill_(E)
    elif kind == "same":
        ids = ids[:, :1].expand(T, k)
    return ids


def _close(got, want, bound, name):
    got = got.to(want.device, torch.float64)
    assert got.shape == want.shape, (name, got.shape, want.shape)
    bad = ~((got - want).abs() <= bound)
    assert not bool(bad.any()), (
        f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {float((got - want).abs().max()):.3e}, "
        f"first at {torch.nonzero(bad)[0].tolist()}")


# ------------------------------------------------------------------ sort
# slots across the workgroup's 1024, 4096 and 8192, and over more workgroups than a scan's 256
@pytest.mark.parametrize("T,k,E", [(0, 2, 4), (1, 1, 1), (1, 8, 64), (5, 0, 3), (63, 1, 2), (64, 16, 7),
                                   (1000, 1, 1000), (1025, 1, 64), (4096, 1, 65), (1366, 3, 128),
                                   (1024, 8, 1024), (8193, 1, 5), (8192, 8, 64), (200000, 6, 1024)])
@pytest.mark.parametrize("kind", ["even", "one", "drop"])
def test_sort(dev, T, k, E, kind):
    ids = _ids(_gen(T, k, E), T, k, E, kind)
    for t in (torch.int64, torch.int32):
        plan = mj.sort_experts(ids.to(t), E)
        pos, offsets = plain.sort(ids, E)
        assert torch.equal(plan.offsets.cpu(), offsets)
        assert torch.equal(plan.pos.cpu(), pos)


def test_sort_of_far_numbers_and_strides(dev):
    """int64 entries beyond 32 bits are outside, not wrapped; a strided view is a matrix."""
    ids = torch.tensor([[0, 1 << 32], [(1 << 40) + 1, 2], [-(1 << 32), 3], [1, -1]], device="cuda")
    plan = mj.sort_experts(ids.t().contiguous().t(), 3)
    pos, offsets = plain.sort(ids, 3)
    assert torch.equal(plan.pos.cpu(), pos) and torch.equal(plan.offsets.cpu(), offsets)


# ------------------------------------------------------------------ rows
_ROWS = [(1, 1, 1, 1), (1, 2, 8, 4096), (3, 5, 4, 7), (7, 4, 3, 8), (33, 8, 64, 520), (100, 3, 10, 1001),
         (257, 2, 5, 513), (64, 17, 20, 136), (500, 6, 32, 8200), (2000, 8, 64, 1024)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T,k,E,D", _ROWS)
@pytest.mark.parametrize("kind", ["even", "drop", "same"])
def test_rows(dev, T, k, E, D, kind, dtype):
    g, dt, unit, e = _gen(T, k, E, D), DT[dtype], UNIT[dtype], 2.0 ** -24
    ids = _ids(g, T, k, E, kind)
    plan = mj.sort_experts(ids, E)
    pos, kept = plan.pos, int(plan.offsets[-1])
    x, dy = _normal(g, (T, D), dt), _normal(g, (T, D), dt)
    ys, w = _normal(g, (T * k, D), dt), _normal(g, (T, k))
    xs, ws = mj.dispatch(x, plan, w)
    want = torch.zeros_like(ys)
    on = pos < kept
    for j in range(k):
        want[pos[:, j].long()] = torch.where(on[:, j, None], x, torch.zeros_like(x))
    assert torch.equal(xs, want) and torch.equal(mj.dispatch(x, plan), want)
    assert torch.equal(ws[pos.long()], torch.where(on, w, 0.0))
    y, size = plain.combine(ys, w, pos, kept)
    _close(mj.combine(ys, w, plan), y, (k + 1) * e * size + unit * y.abs(), "y")
    if dtype == "f32":
        _close(mj.combine(ys, w, plan, torch.bfloat16), y, (k + 1) * e * size + 2.0 ** -8 * y.abs(), "y")
    dx, size = plain.combine(ys, None, pos, kept)
    _close(mj.dispatch_backward(ys, plan), dx, (k + 1) * e * size + unit * dx.abs(), "dx")
    dys, dw = mj.combine_backward(dy, ys, w, plan)
    rdys, rdw, size = plain.combine_backward(dy, ys, w, pos, kept)
    _close(dys, rdys, e * rdys.abs() + unit * rdys.abs(), "dys")
    _close(dw, rdw, (D + 8) * e * size, "dw")


def test_dropped_rows_may_hold_anything(dev):
    """A slot without an expert adds nothing to its token, whatever its row and weight hold."""
    g = _gen("dropped")
    ids = _ids(g, 50, 3, 6, "drop")
    plan = mj.sort_experts(ids, 6)
    kept = int(plan.offsets[-1])
    off = plan.pos >= kept
    ys, dy, w = _normal(g, (150, 72), torch.bfloat16), _normal(g, (50, 72), torch.bfloat16), _normal(g, (50, 3))
    bad, wbad = ys.clone(), w.clone()
    bad[kept:] = float("nan")
    wbad[off] = float("inf")
    assert torch.equal(mj.combine(bad, wbad, plan), mj.combine(ys, w, plan))
    for a, b in zip(mj.combine_backward(dy, bad, wbad, plan), mj.combine_backward(dy, ys, w, plan)):
        assert torch.equal(a, b)
    assert not bool(mj.dispatch(dy, plan, wbad)[1][kept:].any())


def test_empty(dev):
    for T, k, D in ((0, 2, 8), (3, 0, 8), (3, 2, 0)):
        plan = mj.sort_experts(torch.zeros(T, k, dtype=torch.int64, device="cuda"), 4)
        x = torch.ones(T, D, device="cuda", dtype=torch.bfloat16)
        w = torch.ones(T, k, device="cuda")
        xs, ws = mj.dispatch(x, plan, w)
        assert xs.shape == (T * k, D) and torch.equal(ws, torch.ones(T * k, device="cuda"))
        y = mj.combine(xs, w, plan)
        assert y.shape == (T, D) and (k == 0) <= (not bool(y.any()))
        dys, dw = mj.combine_backward(x, xs, w, plan)
        assert dys.shape == xs.shape and dw.shape == (T, k) and (D > 0 or not bool(dw.any()))


# ------------------------------------------------------------------ the experts' block
# tokens, topk, E, K, I, H: few rows an expert (one token; a segment of 16 that ends inside, and over
# it), tiles of 64, 128 and 256 rows, experts without rows, ragged widths, all rows in one expert
_MLP = [(1, 1, 1, 8, 8, 8, "even"), (1, 2, 8, 256, 704, 256, "even"), (5, 3, 4, 72, 136, 40, "drop"),
        (24, 2, 64, 128, 96, 128, "even"), (60, 2, 8, 264, 520, 136, "one"), (100, 2, 3, 200, 328, 96, "drop"),
        (300, 2, 5, 520, 264, 392, "even"), (1000, 3, 16, 136, 712, 104, "drop"), (700, 2, 70, 64, 64, 64, "even"),
        (900, 2, 2, 1024, 1400, 1024, "even"), (2048, 2, 4, 1032, 2056, 1048, "drop"),
        (3000, 1, 130, 256, 512, 256, "one"), (40, 2, 6, 64, 128, 64, "none"), (30, 4, 5, 96, 64, 96, "same")]


@pytest.mark.parametrize("T,k,E,K,I,H,kind", _MLP)
def test_experts(dev, T, k, E, K, I, H, kind):
    act = ["silu", "gelu", "relu", "none"][(T + K) % 4]
    g, dt = _gen(T, k, E, K, I, H), torch.bfloat16
    ids, w = _ids(g, T, k, E, kind), torch.rand((T, k), generator=g, device="cuda") + 0.1
    x, dy = _normal(g, (T, K), dt), _normal(g, (T, H), dt)
    wg, wu = _normal(g, (E, I, K), dt, K ** -0.5), _normal(g, (E, I, K), dt, K ** -0.5)
    wd = _normal(g, (E, H, I), dt, I ** -0.5)
    layer = mj.ExpertsMLP(wg, wu, wd, ACTS[act])
    y0 = layer.forward(x, ids, w)
    y, saved = layer.forward_train(x, ids, w)
    grads = layer.backward(dy, saved)
    assert torch.equal(y, y0)
    pos, offsets = (t.to("cuda") for t in plain.sort(ids, E))
    ref = plain.mlp(x, pos, offsets, w, wg, wu, wd, dy, act, 2.0 ** -8, 2.0 ** -18)
    _close(y, *ref["y"], "y")
    for name, got in grads.items():
        assert got.dtype == (torch.float32 if name == "weights" else dt)
        _close(got, ref[name][0], ref[name][1] + 1e-30, name)


def test_experts_without_weights(dev):
    """Rows as they are: ys and its gradients equal those with weights of one; rows of dropped
    slots are zeros, and what the gradient holds there is not read."""
    g, dt = _gen("plain"), torch.bfloat16
    T, k, E, K, I = 200, 2, 5, 136, 264
    plan = mj.sort_experts(_ids(g, T, k, E, "drop"), E)
    kept = int(plan.offsets[-1])
    xs = mj.dispatch(_normal(g, (T, K), dt), plan)
    m = [_normal(g, s, dt, s[2] ** -0.5) for s in ((E, I, K), (E, I, K), (E, K, I))]
    ys, saved = mj.experts_mlp_train(xs, plan, *m)
    one, saved1 = mj.experts_mlp_train(xs, plan, *m, weights=torch.ones(T * k, device="cuda"))
    assert torch.equal(ys, one) and torch.equal(mj.experts_mlp(xs, plan, *m), ys)
    assert not bool(ys[kept:].any()) and bool(ys[:kept].any())
    dys = _normal(g, (T * k, K), dt)
    dys[kept:] = float("nan")
    a, b = mj.experts_mlp_backward(dys, saved), mj.experts_mlp_backward(dys, saved1)
    for u, v in zip(a[:4], b[:4]):
        assert torch.equal(u, v) and bool(torch.isfinite(u).all())
    assert a[4] is None and bool(torch.isfinite(b[4]).all()) and not bool(a[0][kept:].any())


def test_experts_gradients_by_differences(dev):
    """The gradients against central differences of the layer in float64 (its plain form), in
    random directions: a check of the formulas themselves."""
    g = _gen("differences")
    T, k, E, K, I = 6, 2, 3, 16, 24
    ids = _ids(g, T, k, E, "drop")
    pos, offsets = (t.to("cuda") for t in plain.sort(ids, E))
    v = dict(x=_normal(g, (T, K)), w=_normal(g, (T, k)), gate=_normal(g, (E, I, K), std=0.3),
             up=_normal(g, (E, I, K), std=0.3), down=_normal(g, (E, K, I), std=0.3))
    v = {n: t.to(torch.bfloat16).float() for n, t in v.items()}
    dy = _normal(g, (T, K), torch.bfloat16)
    f = lambda d: plain.mlp(d["x"], pos, offsets, d["w"], d["gate"], d["up"], d["down"], dy,  # noqa: E731
                            "silu", 0.0, 0.0)["y"][0]
    ref = plain.mlp(v["x"], pos, offsets, v["w"], v["gate"], v["up"], v["down"], dy, "silu", 2.0 ** -8, 2.0 ** -18)
    b = {n: t.to(torch.bfloat16) for n, t in v.items()}
    _, saved = mj.ExpertsMLP(b["gate"], b["up"], b["down"]).forward_train(b["x"], ids, v["w"])
    grads = mj.ExpertsMLP.backward(dy, saved)
    for name, key in (("x", "x"), ("w", "weights"), ("gate", "gate"), ("up", "up"), ("down", "down")):
        way = _normal(g, v[name].shape).double()
        h = 1e-5
        up, down = ({**{n: t.double() for n, t in v.items()}, name: v[name].double() + s * h * way}
                    for s in (1, -1))
        slope = ((f(up) - f(down)) * dy.double()).sum() / (2 * h)
        got = (grads[key].double() * way).sum()
        bound = (ref[key][1] * way.abs()).sum() + 1e-7 * (ref[key][0] * way).abs().sum()
        assert abs(float(got - slope)) <= float(bound), (name, float(got), float(slope), float(bound))


def test_captured_and_replayed(dev):
    """A captured step draws its plan anew: replayed with other tokens, experts and weights, with
    eager work between, it gives what eager calls give."""
    g, dt = _gen("graph"), torch.bfloat16
    T, k, E, K, I = 130, 2, 6, 64, 136
    m = [_normal(g, s, dt, 0.1) for s in ((E, I, K), (E, I, K), (E, K, I))]
    layer = mj.ExpertsMLP(*m)

    def fresh():
        return _normal(g, (T, K), dt), _ids(g, T, k, E, "drop"), _normal(g, (T, k)), _normal(g, (T, K), dt)

    def step(x, ids, w, dy):
        y, saved = layer.forward_train(x, ids, w)
        return [y, *layer.backward(dy, saved).values()]

    held = fresh()
    step(*held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*held)
    for _ in range(3):
        new = fresh()
        for a, b in zip(held, new):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step(*new)):
            assert torch.equal(a, b)


def test_strides_and_streams(dev):
    """Transposed and offset operands are copied; a call on another stream runs there."""
    g, dt = _gen("strides"), torch.bfloat16
    T, k, E, K, I = 40, 2, 4, 64, 72
    m = [_normal(g, s, dt, 0.1) for s in ((E, I, K), (E, I, K), (E, K, I))]
    x, ids, w = _normal(g, (T, K), dt), _ids(g, T, k, E), _normal(g, (T, k))
    y = mj.ExpertsMLP(*m).forward(x, ids, w)
    off = torch.empty(T * K + 1, dtype=dt, device="cuda")[1:].view(T, K).copy_(x)
    odd = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in m]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        y2 = mj.ExpertsMLP(*odd).forward(off, ids.t().contiguous().t(), w.t().contiguous().t())
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(y, y2)


def test_refusals(dev):
    x = torch.zeros(4, 16, dtype=torch.bfloat16, device="cuda")
    ids, w = torch.zeros(4, 2, dtype=torch.int64, device="cuda"), torch.ones(4, 2, device="cuda")
    m = [torch.zeros(3, 16, 16, dtype=torch.bfloat16, device="cuda") for _ in range(3)]
    plan = mj.sort_experts(ids, 3)
    for bad in (lambda: mj.sort_experts(ids.float(), 3), lambda: mj.sort_experts(ids[0], 3),
                lambda: mj.sort_experts(ids.cpu(), 3), lambda: mj.sort_experts(ids, 0),
                lambda: mj.sort_experts(ids, 1025), lambda: mj.dispatch(x[:3], plan),
                lambda: mj.dispatch(x.half(), plan), lambda: mj.dispatch(x, plan, w.double()),
                lambda: mj.dispatch(x, plan, w[:, :1]), lambda: mj.combine(x, w, plan),
                lambda: mj.combine(mj.dispatch(x, plan), w, plan, torch.float32),
                lambda: mj.combine_backward(x, x, w, plan), lambda: mj.ExpertsMLP(m[0], m[1][:2], m[2]),
                lambda: mj.ExpertsMLP(*m).forward(x.float(), ids, w),
                lambda: mj.ExpertsMLP(*m, mj.EPI_SILU_APPROX).forward(x, ids, w),
                lambda: mj.experts_mlp(mj.dispatch(x, plan), plan, m[0][:2], m[1][:2], m[2][:2]),
                lambda: mj.experts_mlp(mj.dispatch(x[:, :12], plan), plan, *[t[:, :12, :12] for t in m])):
        with pytest.raises((TypeError, ValueError, mj.MomijoHipError)):
            bad()
