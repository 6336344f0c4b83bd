"""Few rows an expert through layers so wide that the few-row kernels need more than 2^32 threads: 2^18 column
tiles for each of 33 and more segments of rows."""
import pytest
import torch

import momijo_amd as mj
import test_gpu_experts as experts
import test_gpu_fp8 as fp8
from momijo_amd import _lib

pytestmark = pytest.mark.gpu

WIDE = 1 << 22                     # (the first width that is refused)
# tokens, experts, K, I, H
BF16 = [(33, 33, 8, WIDE - 8, 8), (33, 33, 8, 8, WIDE - 8)]
F8 = [(33, 33, 16, WIDE - 16, 16), (33, 33, 16, 16, WIDE - 3), (500, 60, 16, WIDE - 16, 16),
      (500, 60, 16, 16, WIDE - 3)]


@pytest.mark.parametrize("T,E,K,I,H", BF16)
def test_experts(dev, T, E, K, I, H):
    """Each step from the one before as it is on the device.  A sum of n products is off by fewer than n + 8
    roundings of Float32 where n terms are added one after another: K for g and u, and I / 256 + 64 for ys (8
    waves, 32 products an addition)."""
    for product in (0, 1):
        assert _lib.load().mj_experts_mlp_kernel(T, E, K, I, H, product) == b"16 rows"
    g = torch.Generator(device="cuda").manual_seed(I)
    r = lambda *s: torch.randn(s, generator=g, device="cuda", dtype=torch.float32).bfloat16()  # noqa: E731
    wg, wu, wd = r(E, I, K), r(E, I, K), r(E, H, I)
    plan = mj.sort_experts(torch.randint(0, E, (T, 1), generator=g, device="cuda"), E)
    xs, ws = mj.dispatch(r(T, K), plan, torch.rand(T, 1, generator=g, device="cuda") + 0.1)
    ys, saved = mj.experts_mlp_train(xs, plan, wg, wu, wd, mj.EPI_NONE, ws)
    n = 4 * T * I
    gk, uk = (saved.buf[at:at + n].view(torch.float32).view(T, I) for at in (0, n))
    hk = saved.buf[2 * n:].view(torch.bfloat16)[:T * I].view(T, I)
    ends, unit = plan.offsets.tolist(), 2.0 ** -24
    for e in range(E):
        for m in range(ends[e], ends[e + 1]):
            x = xs[m].double()
            for got, w in ((gk, wg), (uk, wu)):
                t = w[e].double() * x
                experts._close(got[m], t.sum(1), (K + 8) * unit * t.abs().sum(1), "g or u")
            h = gk[m].double() * uk[m].double() * ws[m].double()
            experts._close(hk[m], h, (2.0 ** -8 + 4 * unit) * h.abs(), "h")
            t = wd[e].double() * hk[m].double()
            experts._close(ys[m], t.sum(1), (I / 256 + 64) * unit * t.abs().sum(1), "ys")


@pytest.mark.parametrize("T,E,K,I,H", F8)
def test_f8_experts(dev, T, E, K, I, H):
    name = b"16 rows" if T <= 8 * E else b"32 rows"
    assert _lib.load().mj_gemm_f8_kernel(T, I, K, E, 1) == name == _lib.load().mj_gemm_f8_kernel(T, H, I, E, 0)
    fp8.test_experts(dev, T, 1, E, K, I, H, "even")
