"""What the experts' and the 8-bit entry points write: every output lies between two guards that stay as they were,
with plans that a sort gave and with others, and holds what the Python entry points give.  Also few-row
segments behind an expert's first."""
import pytest
import torch

import momijo_amd as mj
import test_gpu_experts as experts
import test_gpu_fp8 as fp8
from momijo_amd import _lib

pytestmark = pytest.mark.gpu

GUARD = 1024  # bytes on either side
BF, F32, F8, I32 = torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.int32


class Guarded:
    """Output tensors, filled with 0x5A bytes as their surroundings are."""

    def __init__(self):
        self.held = {}

    def __call__(self, name, shape, dtype):
        t = torch.empty(shape, dtype=dtype, device="meta")
        n = t.numel() * t.element_size()
        raw = torch.full((n + 2 * GUARD,), 0x5A, dtype=torch.uint8, device="cuda")
        self.held[name] = raw, raw[GUARD:GUARD + n].view(dtype).view(shape)
        return raw.data_ptr() + GUARD  # (an empty tensor's address too)

    def __getitem__(self, name):
        return self.held[name][1]

    def check(self):
        torch.cuda.synchronize()
        for name, (raw, _) in self.held.items():
            for part in (raw[:GUARD], raw[-GUARD:]):
                assert bool((part == 0x5A).all()), f"bytes around {name} were written"


def _operands(T, k, E, K, I, H):
    g = torch.Generator(device="cuda").manual_seed(T + K)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    m = [r(E, I, K) * K ** -0.5, r(E, I, K) * K ** -0.5, r(E, H, I) * I ** -0.5]
    return g, r(T, K).bfloat16(), r(T, H).bfloat16(), r(T, k), [t.bfloat16() for t in m]


def _plans(g, T, k, E):
    """A sort's, then two that are none."""
    ids = torch.randint(-1, E, (T, k), generator=g, device="cuda")
    yield mj.sort_experts(ids, E), True
    rows, big = T * k, 2 ** 31 - 1
    pos = torch.randint(-2 * rows, 3 * rows, (T, k), generator=g, device="cuda", dtype=I32)
    pos[0, 0], pos[-1, -1], pos[1, 0] = big, -big - 1, rows
    for ends in ([0, big, -5, 7], [rows + 1, rows, 0, -big - 1]):
        offsets = torch.tensor([ends[i % 4] for i in range(E + 1)], dtype=I32, device="cuda")
        yield mj.ExpertPlan(pos, offsets), False


def _call(name, *args):
    _lib.call(name, *[a.data_ptr() if isinstance(a, torch.Tensor) else a for a in args], None)


def _same(got, want):
    assert got.shape == want.shape and got.dtype == want.dtype
    assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))


# few rows an expert, small tiles, 256 x 256 tiles with a second launch
SIZES = [(9, 2, 4, 64, 80, 72), (60, 2, 8, 72, 144, 328), (400, 3, 5, 272, 400, 136), (2500, 2, 3, 1040, 272, 520)]


@pytest.mark.parametrize("T,k,E,K,I,H", SIZES)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows(dev, T, k, E, K, I, H, dtype):
    g, x, _, w, _ = _operands(T, k, E, K, I, H)
    x, code, R = x.to(dtype), _lib.BF16 if dtype is BF else _lib.F32, T * k
    ys = torch.randn(R, K, generator=g, device="cuda").to(dtype)
    for plan, real in _plans(g, T, k, E):
        o = Guarded()
        p = (plan.pos, plan.offsets, E)
        _call("mj_dispatch", code, x, w, *p, o("xs", (R, K), dtype), o("ws", (R,), F32), T, k, K)
        _call("mj_combine", code, code, ys, w, *p, o("y", (T, K), dtype), T, k, K)
        _call("mj_combine", code, _lib.BF16, ys, None, *p, o("y16", (T, K), BF), T, k, K)
        _call("mj_combine_backward", code, x, ys, w, *p, o("dys", (R, K), dtype), o("dw", (T, k), F32), T, k, K)
        o.check()
        if real:
            xs, ws = mj.dispatch(x, plan, w)
            dys, dw = mj.combine_backward(x, ys, w, plan)
            for name, want in dict(xs=xs, ws=ws, y=mj.combine(ys, w, plan), y16=mj.combine(ys, None, plan, BF), dys=dys,
                                   dw=dw).items():
                _same(o[name], want)


@pytest.mark.parametrize("slots", [1, 1000, 1025, 8192, 8193, 20000])
@pytest.mark.parametrize("E", [1, 7, 1024])
def test_sort(dev, slots, E):
    ids = torch.randint(-1, E + 1, (slots, 1), device="cuda", generator=torch.Generator("cuda").manual_seed(slots))
    o = Guarded()
    n = _lib.load().mj_sort_experts_work_bytes(slots, E)
    _call("mj_sort_experts", ids, 8, slots, E, o("pos", (slots, 1), I32), o("offsets", (E + 1,), I32),
          o("work", (n,), torch.uint8), n)
    o.check()
    plan = mj.sort_experts(ids, E)
    _same(o["pos"], plan.pos)
    _same(o["offsets"], plan.offsets)


@pytest.mark.parametrize("T,k,E,K,I,H", SIZES)
def test_experts(dev, T, k, E, K, I, H):
    g, x, dy, w, m = _operands(T, k, E, K, I, H)
    R, act = T * k, _lib.EPI_SILU
    for plan, real in _plans(g, T, k, E):
        o = Guarded()
        xs, ws = mj.dispatch(x, plan, w)
        dys = mj.dispatch(dy, plan)
        dots = _lib.load().mj_experts_mlp_dots(R, E, K, I, H)
        _call("mj_experts_mlp_bf16", xs, plan.offsets, E, *m, act, ws, o("h", (R, I), BF), o("g", (R, I), F32),
              o("u", (R, I), F32), o("ys", (R, H), F32), R, K, I, H)
        if not real:  # (rows that no tile wrote: numbers all the same)
            for name in ("h", "g", "u"):
                o[name].fill_(0.5)
        _call("mj_experts_mlp_backward_bf16", xs, plan.offsets, E, *m, act, ws, o["h"], o["g"], o["u"], dys,
              o("dg", (R, I), BF), o("du", (R, I), BF), o("dxs", (R, K), F32), o("dwg", m[0].shape, BF),
              o("dwu", m[1].shape, BF), o("dwd", m[2].shape, BF), plan.pos, R, o("dots", (dots,), F32),
              o("dw", (T, k), F32), R, K, I, H)
        o.check()
        if real:
            ys, saved = mj.experts_mlp_train(xs, plan, *m, weights=ws)
            dxs, dwg, dwu, dwd, dw = mj.experts_mlp_backward(dys, saved)
            for name, want in dict(ys=ys, dxs=dxs, dwg=dwg, dwu=dwu, dwd=dwd, dw=dw).items():
                _same(o[name], want)
            kept = int(plan.offsets[-1])
            for name in ("h", "g", "u", "dg", "du"):  # the dropped slots' rows stay as they were
                assert bool((o[name][kept:].view(torch.uint8) == 0x5A).all()), name


@pytest.mark.parametrize("T,k,E,K,I,H", SIZES)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_f8_experts(dev, T, k, E, K, I, H, dtype):
    K, I, R, act = -(-K // 16) * 16, -(-I // 16) * 16, T * k, _lib.EPI_SILU
    g, x, _, _, m = _operands(T, k, E, K, I, H)
    x, f = x.to(dtype), mj.F8Experts.from_float(*m)
    for plan, real in _plans(g, T, k, E):
        o = Guarded()
        bk, bi = -(-K // 128), -(-I // 128)
        _call("mj_dispatch_f8", _lib.BF16 if dtype is BF else _lib.F32, x, plan.pos, plan.offsets, E,
              o("q", (R, K), F8), o("s", (bk, R), F32), T, k, K)
        if not real:
            o["q"].view(torch.uint8).fill_(0x30)
            o["s"].fill_(1.0)
        n = _lib.load().mj_experts_gate_f8_work_bytes(R, E, I, K)
        _call("mj_experts_gate_f8", o["q"], o["s"], plan.offsets, E, f.gate, f.gate_scales, f.up, f.up_scales, act,
              o("hq", (R, I), F8), o("hs", (bi, R), F32), R, I, K, o("work", (n,), torch.uint8), n)
        _call("mj_experts_gemm_f8", o["hq"], o["hs"], plan.offsets, E, f.down, f.down_scales, o("ys", (R, H), F32), R, H,
              I)
        o.check()
        if real:
            q, s = mj.dispatch_fp8(x, plan)
            hq, hs = mj.experts_gate_fp8(q, s, plan, f.gate, f.gate_scales, f.up, f.up_scales, act)
            for name, want in dict(q=q, s=s, hq=hq, hs=hs,
                                   ys=mj.experts_gemm_fp8(hq, hs, plan, f.down, f.down_scales)).items():
                _same(o[name], want)


# few rows, small tiles with and without K slices, large tiles with and without; odd widths
@pytest.mark.parametrize("M,N,K", [(1, 301, 272), (9, 1000, 4112), (31, 300, 272), (50, 129, 144), (102, 303, 1424),
                                   (65, 72, 4112), (1000, 3001, 1040), (131, 6746, 5360), (1561, 7342, 144)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_f8_linear(dev, M, N, K, dtype):
    g = torch.Generator(device="cuda").manual_seed(M)
    x = torch.randn(M, K, generator=g, device="cuda").to(dtype)
    W, bias = torch.randn(N, K, generator=g, device="cuda"), torch.randn(N, generator=g, device="cuda")
    code, b = _lib.BF16 if dtype is BF else _lib.F32, -(-K // 128)
    o = Guarded()
    _call("mj_quantize_blocks_f8", _lib.F32, W, o("w", (N, K), F8), o("ws", (-(-N // 128), b), F32), 1, N, K)
    _call("mj_quantize_rows_f8", code, x, o("q", (M, K), F8), o("s", (b, M), F32), M, K)
    n = _lib.load().mj_gemm_f8_work_bytes(M, N, K)
    _call("mj_gemm_f8", o["q"], o["s"], o["w"], o["ws"], bias, _lib.EPI_GELU_TANH, o("y", (M, N), BF), M, N, K,
          o("work", (n,), torch.uint8), n)
    n = _lib.load().mj_linear_f8_work_bytes(M, N, K)
    _call("mj_linear_f8", code, x, o["w"], o["ws"], bias, _lib.EPI_GELU_TANH, o("y2", (M, N), BF), M, N, K,
          o("work2", (n,), torch.uint8), n)
    o.check()
    lin = mj.F8Linear.from_float(W, bias, _lib.EPI_GELU_TANH)
    _same(o["w"], lin.q)
    _same(o["ws"], lin.scales)
    _same(o["y"], lin.forward(x))
    _same(o["y2"], o["y"])


# an expert's rows, or the dropped ones, over several segments of 16 and of 32, the last one not full; widths
# that end inside 32 columns
@pytest.mark.parametrize("T,name", [(20, b"16 rows"), (60, b"32 rows")])
@pytest.mark.parametrize("kind", ["one", "none"])
@pytest.mark.parametrize("K,I,H", [(272, 144, 330), (1040, 400, 1009)])
def test_f8_segments(dev, T, name, kind, K, I, H):
    kernel = _lib.load().mj_gemm_f8_kernel
    assert kernel(2 * T, I, K, 8, 1) == name == kernel(2 * T, H, I, 8, 0)
    fp8.test_experts(dev, T, 2, 8, K, I, H, kind)


@pytest.mark.parametrize("counts", [(0, 40, 0, 1, 17, 0, 32, 38), (3, 0, 0, 0, 0, 0, 90, 35), (1, 0, 127, 0, 0, 0, 0, 0)])
@pytest.mark.parametrize("K,I,H", [(72, 136, 40), (264, 520, 1000)])
def test_segments(dev, counts, K, I, H):
    """So many rows of each of eight experts and, last, so many dropped."""
    counts = (*counts[:7], 0, counts[7])
    T = sum(counts)
    assert all(_lib.load().mj_experts_mlp_kernel(T, 8, K, I, H, p) == b"16 rows" for p in (0, 1))
    experts.test_experts(dev, T, 1, 8, K, I, H, counts)
