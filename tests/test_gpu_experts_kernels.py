"""Every kernel that the plans of the experts' block and of the 8-bit products can choose,
against the 64-bit plain forms (test_experts_kernels.py asserts on the host that these sizes
reach them), widths of zero, many experts, and arrays past 2^32 bytes."""
import pytest
import torch

import _experts as plain
import momijo_amd as mj
import test_gpu_experts as experts
import test_gpu_fp8 as fp8

pytestmark = pytest.mark.gpu

# rows, N, K
LINEAR = [(16, 4104, 1040), (12, 520, 2704), (9, 1000, 4112), (31, 300, 272), (197, 8220, 144), (130, 3614, 3744),
          (898, 8300, 144), (131, 6746, 5360), (1561, 7342, 144), (1000, 11000, 1040), (391, 5382, 5696),
          (102, 303, 1424)]
# tokens, topk, experts, K, I, H
F8_EXPERTS = [(407, 1, 22, 144, 1424, 144), (50, 2, 2, 144, 336, 160), (4975, 1, 2, 144, 1168, 144),
              (56, 2, 8, 144, 320, 330), (1863, 2, 2, 160, 144, 545), (2291, 2, 2, 160, 144, 1763),
              (4661, 1, 3, 144, 160, 2305), (3000, 2, 4, 1040, 2064, 3001)]
EXPERTS = [(3519, 1, 2, 208, 560, 128), (4457, 1, 2, 120, 352, 96), (3529, 1, 2, 96, 1504, 112),
           (3067, 1, 2, 96, 368, 112), (869, 2, 3, 160, 96, 2208), (941, 2, 2, 184, 104, 1712),
           (4401, 1, 4, 120, 104, 1840), (4504, 1, 2, 128, 1360, 104), (3173, 1, 5, 104, 944, 104),
           (3844, 1, 2, 144, 2592, 96), (1945, 1, 2, 2056, 96, 128), (2551, 1, 2, 1192, 112, 168),
           (4963, 1, 3, 1816, 96, 128), (59, 3, 24, 944, 96, 144), (95, 5, 22, 280, 152, 96),
           (494, 2, 7, 2440, 136, 176), (139, 1, 26, 200, 104, 104), (4001, 2, 4, 1032, 3000, 1096)]
# rows of each expert, dropped rows, then K, I, H: what the whole rounds of 256 x 256 tiles leave over,
# in quarters (up to half a round: one tile, quarters past the rows and the columns) or in whole tiles
ROUNDS = [((1500, 2050, 1300, 250), 3376, 3376, 3376), ((4090, 1, 2049, 900), 4088, 4088, 4088),
          ((1400, 2600, 2060, 10), 3240, 3304, 3240), ((1400, 2600, 1290, 10), 4088, 3376, 4088),
          ((2000, 2600, 3000, 250), 4088, 3376, 4088)]


@pytest.mark.parametrize("counts,K,I,H", ROUNDS)
def test_rounds_of_experts(dev, counts, K, I, H):
    experts.test_experts(dev, sum(counts), 1, len(counts) - 1, K, I, H, counts)


@pytest.mark.parametrize("M,N,K", LINEAR)
def test_linear(dev, M, N, K):
    fp8.test_linear(dev, M, N, K)


@pytest.mark.parametrize("T,k,E,K,I,H", F8_EXPERTS)
def test_f8_experts(dev, T, k, E, K, I, H):
    fp8.test_experts(dev, T, k, E, K, I, H, "drop" if T % 2 else "even")


@pytest.mark.parametrize("T,k,E,K,I,H", EXPERTS)
def test_experts(dev, T, k, E, K, I, H):
    experts.test_experts(dev, T, k, E, K, I, H, "drop" if T % 2 else "even")


def test_many_experts(dev):
    """More experts than a wave has lanes, most of them without rows."""
    experts.test_experts(dev, 40, 2, 1024, 16, 16, 16, "even")
    experts.test_experts(dev, 3000, 8, 700, 24, 16, 16, "drop")
    fp8.test_experts(dev, 40, 2, 1024, 16, 16, 16, "even")
    fp8.test_experts(dev, 5000, 8, 700, 16, 32, 16, "drop")


@pytest.mark.parametrize("T", [3, 90])
@pytest.mark.parametrize("K,I,H", [(0, 16, 16), (16, 0, 16), (16, 16, 0), (0, 0, 16)])
def test_experts_of_zero_width(dev, T, K, I, H):
    """An empty sum is zero, and so are the gradients it feeds; nothing of other shapes is written."""
    z = lambda *s: torch.ones(*s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    ids = torch.arange(T * 2, device="cuda").reshape(T, 2) % 3
    w = torch.ones(T, 2, device="cuda")
    layer = mj.ExpertsMLP(z(3, I, K), z(3, I, K), z(3, H, I))
    y, saved = layer.forward_train(z(T, K), ids, w)
    assert y.shape == (T, H) and not bool(y.any())
    g = layer.backward(z(T, H), saved)
    for name, shape in (("x", (T, K)), ("weights", (T, 2)), ("gate", (3, I, K)), ("up", (3, I, K)), ("down", (3, H, I))):
        assert g[name].shape == shape and not bool(g[name].any()), name


@pytest.mark.parametrize("M", [3, 40, 300])
def test_linear_of_zero_width(dev, M):
    bias = torch.randn(72, device="cuda")
    lin = mj.F8Linear.from_float(torch.zeros(72, 0, device="cuda"), bias)
    y = lin.forward(torch.zeros(M, 0, device="cuda"))
    assert torch.equal(y, bias.bfloat16().expand(M, 72))
    assert mj.F8Linear.from_float(torch.zeros(0, 64, device="cuda")).forward(torch.zeros(M, 64, device="cuda")).shape == (M, 0)


def test_no_tokens(dev):
    m = [torch.ones(3, 16, 16, dtype=torch.bfloat16, device="cuda") for _ in range(3)]
    x, ids, w = m[0].new_empty((0, 16)), torch.empty(0, 2, dtype=torch.int64, device="cuda"), torch.empty(0, 2, device="cuda")
    y, saved = mj.ExpertsMLP(*m).forward_train(x, ids, w)
    g = mj.ExpertsMLP.backward(y, saved)
    assert y.shape == (0, 16) and g["x"].shape == (0, 16) and g["weights"].shape == (0, 2)
    assert not any(bool(g[n].any()) for n in ("gate", "up", "down"))
    assert mj.F8Experts.from_float(*m).forward(x, ids, w).shape == (0, 16)


def test_another_current_device(dev, monkeypatch):
    """Tensors of a device that is not the current one are refused, with saved operands too."""
    T, k, E, K = 6, 2, 3, 32
    m = [torch.ones(*s, dtype=torch.bfloat16, device="cuda") for s in ((E, 16, K), (E, 16, K), (E, K, 16))]
    x, w = torch.ones(T, K, dtype=torch.bfloat16, device="cuda"), torch.ones(T, k, device="cuda")
    ids = torch.zeros(T, k, dtype=torch.int32, device="cuda")
    plan = mj.sort_experts(ids, E)
    xs, ws = mj.dispatch(x, plan, w)
    ys, saved = mj.experts_mlp_train(xs, plan, *m, weights=ws)
    f8, (q, s), lin = mj.F8Experts.from_float(*m), mj.dispatch_fp8(x, plan), mj.F8Linear.from_float(m[0][0])
    rows = mj.quantize_rows_fp8(x)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1)
    for call in (lambda: mj.sort_experts(ids, E), lambda: mj.dispatch(x, plan, w), lambda: mj.combine(ys, w, plan),
                 lambda: mj.dispatch_backward(ys, plan), lambda: mj.combine_backward(x, xs, w, plan),
                 lambda: mj.experts_mlp(xs, plan, *m), lambda: mj.experts_mlp_backward(xs, saved),
                 lambda: mj.quantize_rows_fp8(x), lambda: mj.quantize_blocks_fp8(m[0]), lambda: lin.forward(x),
                 lambda: mj.gemm_fp8_nt(*rows, lin.q, lin.scales), lambda: mj.dispatch_fp8(x, plan),
                 lambda: mj.experts_gate_fp8(q, s, plan, f8.gate, f8.gate_scales, f8.up, f8.up_scales),
                 lambda: mj.experts_gemm_fp8(q, s, plan, f8.gate, f8.gate_scales)):
        with pytest.raises(ValueError, match="current device"):
            call()


@pytest.mark.parametrize("T,k,E,K", [(9, 2, 4, 64), (400, 3, 5, 272), (5000, 1, 3, 1040)])
def test_plans_that_are_none(dev, T, k, E, K):
    """A caller's own plan, or one that was overwritten: results mean nothing, but what lies around
    the sorted rows stays as it was, and so do the operands."""
    g = torch.Generator(device="cuda").manual_seed(T)
    big = 2 ** 31 - 1
    rows = T * k
    pos = torch.randint(-2 * rows, 3 * rows, (T, k), generator=g, device="cuda", dtype=torch.int32)
    pos[0, 0], pos[-1, -1], pos[1, 0] = big, -big - 1, rows
    m = [torch.randn(*s, generator=g, device="cuda").bfloat16() for s in ((E, 80, K), (E, 80, K), (E, K, 80))]
    x, dy = (torch.randn(T, K, generator=g, device="cuda").bfloat16() for _ in range(2))
    w = torch.rand(T, k, generator=g, device="cuda")
    before = [t.clone() for t in (x, dy, w, *m)]
    f8 = mj.F8Experts.from_float(*m)
    for ends in ([0, big, -5, 7], [rows + 1, rows, 0, -big - 1], [0, rows, 0, rows], [5, 5, 3, big]):
        offsets = torch.tensor([ends[i % 4] for i in range(E + 1)], dtype=torch.int32, device="cuda")
        plan = mj.ExpertPlan(pos, offsets)
        xs, ws = mj.dispatch(x, plan, w)
        ys, saved = mj.experts_mlp_train(xs, plan, *m, weights=ws)
        mj.experts_mlp_backward(mj.dispatch(dy, plan), saved)
        mj.combine(ys, w, plan)
        mj.combine_backward(dy, xs, w, plan)
        q, s = mj.dispatch_fp8(x, plan)
        hq, hs = mj.experts_gate_fp8(q, s, plan, f8.gate, f8.gate_scales, f8.up, f8.up_scales)
        mj.experts_gemm_fp8(hq, hs, plan, f8.down, f8.down_scales)
        guard = torch.full((rows + 8, K), 7.0, dtype=torch.bfloat16, device="cuda")
        wide = torch.full((rows + 8,), 7.0, device="cuda")
        mj._lib.call("mj_dispatch", 1, x.data_ptr(), w.data_ptr(), *plan._args, guard[4:].data_ptr(),
                     wide[4:].data_ptr(), T, k, K, None)
        mj._lib.call("mj_combine_backward", 1, dy.data_ptr(), xs.data_ptr(), w.data_ptr(), *plan._args,
                     guard[4:].data_ptr(), w.clone().data_ptr(), T, k, K, None)
        for t in (guard, wide):
            assert bool((t[:4] == 7).all()) and bool((t[-4:] == 7).all())
        assert all(torch.equal(a, b) for a, b in zip(before, (x, dy, w, *m)))


def test_rows_past_2_32_bytes(dev):
    """Sorted rows of more than 2^32 bytes and 2^31 elements: the last ones are the tokens'."""
    T, k, D = 70000, 4, 8200
    ids = (torch.arange(T * k, device="cuda").reshape(T, k) * 7919) % 5
    ids[::1000, 1] = -1
    plan = mj.sort_experts(ids, 5)
    x = torch.randn(T, D, device="cuda").bfloat16()
    xs = mj.dispatch(x, plan)
    kept = int(plan.offsets[-1])
    pos = plan.pos.long()
    for j in range(k):
        at = torch.arange(0, T, 997, device="cuda")
        on = pos[at, j] < kept
        assert torch.equal(xs[pos[at, j]], torch.where(on[:, None], x[at], torch.zeros_like(x[at])))
    y = mj.combine(xs, None, plan)
    n = (plan.pos < kept).sum(1, keepdim=True)
    for a in range(0, T, 7000):
        want = (x[a:a + 7000].double() * n[a:a + 7000])
        assert bool(((y[a:a + 7000].double() - want).abs() <= 2.0 ** -8 * want.abs()).all())


def test_f8_products_past_2_32_elements(dev):
    """y of more than 2^32 bytes, x and the weights' scales far from their start: rows repeat, and
    so do their outputs."""
    M, N, K = 131328, 16512, 128
    g = torch.Generator(device="cuda").manual_seed(11)
    x = torch.randn(513, K, generator=g, device="cuda").bfloat16()
    lin = mj.F8Linear.from_float(torch.randn(N, K, generator=g, device="cuda"))
    y = lin.forward(x.repeat(256, 1))
    one = lin.forward(x)
    a, w = plain.rows_f64(*mj.quantize_rows_fp8(x)), plain.blocks_f64(lin.q, lin.scales)
    v, e = a @ w.t(), plain.f8_error(a, w)
    assert bool(((one.double() - v).abs() <= e + 2.0 ** -8 * (v.abs() + e)).all())
    for b in (0, 100, 255):
        assert bool(((y[513 * b:513 * (b + 1)].double() - v).abs() <= e + 2.0 ** -8 * (v.abs() + e)).all()), b
