"""64-bit plain forms of the mixture of experts and of the block-scaled 8-bit products,
for the tests."""
import numpy as np
import torch

import _block as block


def sort(ids, experts):
    """pos and offsets by a stable sort of the slots."""
    e = np.asarray(ids.cpu()).reshape(-1).astype(np.int64)
    key = np.where((e >= 0) & (e < experts), e, experts)
    order = np.argsort(key, kind="stable")
    pos = np.empty(e.size, np.int32)
    pos[order] = np.arange(e.size, dtype=np.int32)
    offsets = np.searchsorted(key[order], np.arange(experts + 1), side="left").astype(np.int32)
    return torch.from_numpy(pos.reshape(ids.shape)), torch.from_numpy(offsets)


def combine(ys, w, pos, kept):
    """(y, the sum of its terms' magnitudes) in float64; w None: ones."""
    T, k = pos.shape
    y = torch.zeros(T, ys.shape[1], dtype=torch.float64, device=ys.device)
    size = torch.zeros_like(y)
    for j in range(k):
        on = pos[:, j] < kept
        t = ys[pos[:, j].long().clamp_max(max(ys.shape[0] - 1, 0))].double()
        if w is not None:
            t = t * w[:, j, None].double()
        t = torch.where(on[:, None], t, 0.0)
        y, size = y + t, size + t.abs()
    return y, size


def combine_backward(dy, ys, w, pos, kept):
    """dys, dw and the sum of dw's terms' magnitudes."""
    T, k = pos.shape
    dys = torch.zeros(T * k, dy.shape[1], dtype=torch.float64, device=dy.device)
    dw = torch.zeros(T, k, dtype=torch.float64, device=dy.device)
    size = torch.zeros_like(dw)
    for j in range(k):
        on, at = pos[:, j] < kept, pos[:, j].long()
        dys[at] = torch.where(on[:, None], w[:, j, None].double() * dy.double(), 0.0)
        t = torch.where(on[:, None], dy.double() * ys[at].double(), 0.0)
        dw[:, j], size[:, j] = t.sum(1), t.abs().sum(1)
    return dys, dw, size


def mlp(x, pos, offsets, w, wg, wu, wd, dy, act, unit, e32):
    """{name: (value, bound)} of the experts' layer and its gradients in float64, in the way
    of _block.mlp: h, dg, du and the outputs are rounded to the operands' type (relative
    error `unit`), ys and dxs stay fp32; e32 is the relative error of an fp32 sum against the sum of its
    terms' magnitudes."""
    x, w, wg, wu, wd, dy = (t.double() for t in (x, w, wg, wu, wd, dy))
    T, k = pos.shape
    E, I, K = wg.shape
    H = wd.shape[1]
    kept = int(offsets[-1])
    R = T * k
    new = lambda *s: torch.zeros(*s, dtype=torch.float64, device=x.device)  # noqa: E731
    token = torch.empty(R, dtype=torch.long, device=x.device)
    token[pos.reshape(-1).long()] = torch.arange(R, device=x.device) // k
    rw = new(R)
    rw[pos.reshape(-1).long()] = w.reshape(-1)
    ys, eys, dxs, edxs, dwr, edwr = new(R, H), new(R, H), new(R, K), new(R, K), new(R), new(R)
    out = {n: (new(*s), new(*s)) for n, s in (("gate", wg.shape), ("up", wg.shape), ("down", wd.shape))}
    for e in range(E):
        a, b = int(offsets[e]), int(offsets[e + 1])
        if a == b:
            continue
        xe, d, we = x[token[a:b]], dy[token[a:b]], rw[a:b, None]
        g, u, dh = xe @ wg[e].t(), xe @ wu[e].t(), d @ wd[e]
        eg, eu = e32 * (xe.abs() @ wg[e].abs().t()), e32 * (xe.abs() @ wu[e].abs().t())
        edh = e32 * (d.abs() @ wd[e].abs())
        f, df = block.act(act, g)
        # |act'| <= 1.2, |act''| <= 1.2 for these activations (relu: where g's sign is sure)
        ef, edf = 1.2 * eg + e32 * f.abs(), 1.2 * eg + e32
        if act == "relu":
            edf = torch.where(g.abs() <= eg, 1.0, 0.0) + e32 * df
        hu = f * u
        ehu = ef * u.abs() + f.abs() * eu + ef * eu
        dg, du = we * dh * u * df, we * dh * f
        edg = we.abs() * (edh * (u * df).abs() + dh.abs() * (eu * df.abs() + u.abs() * edf)) + 6 * e32 * dg.abs()
        edu = we.abs() * (edh * f.abs() + dh.abs() * ef) + 6 * e32 * du.abs()
        dwr[a:b] = (dh * hu).sum(1)
        edwr[a:b] = (edh * hu.abs() + dh.abs() * ehu + e32 * (dh * hu).abs()).sum(1)
        h = we * hu
        eh = we.abs() * ehu + (2 * e32 + unit) * h.abs()
        edg, edu = edg + unit * dg.abs(), edu + unit * du.abs()

        def product(p, ep, q, unit=unit):
            v = p @ q
            return v, ep @ q.abs() + e32 * (p.abs() @ q.abs()) + unit * v.abs()

        ys[a:b], eys[a:b] = product(h, eh, wd[e].t(), 0.0)
        (v0, b0), (v1, b1) = product(dg, edg, wg[e], 0.0), product(du, edu, wu[e], 0.0)
        dxs[a:b], edxs[a:b] = v0 + v1, b0 + b1
        for name, p, ep, q in (("gate", dg, edg, xe), ("up", du, edu, xe)):
            out[name][0][e], out[name][1][e] = product(p.t(), ep.t(), q)
        out["down"][0][e], out["down"][1][e] = product(d.t(), torch.zeros_like(d.t()), h)
        out["down"][1][e] += d.abs().t() @ eh

    def back(v, ev):
        y, size = combine(v, None, pos, kept)
        return y, combine(ev, None, pos, kept)[0] + e32 * size + unit * y.abs()

    out["y"], out["x"] = back(ys, eys), back(dxs, edxs)
    at = pos.long()
    on = pos < kept
    out["weights"] = torch.where(on, dwr[at], 0.0), torch.where(on, edwr[at], 0.0)
    return out


# ------------------------------------------------------------------ 8-bit floating point
def e4m3(v):
    """float32 numbers to the nearest e4m3 (ties to even), as float32 (numpy)."""
    v = np.asarray(v, np.float32).astype(np.float64)
    m = np.abs(v)
    with np.errstate(divide="ignore"):
        e = np.floor(np.log2(np.maximum(m, 2.0 ** -6)))
    step = 2.0 ** (e - 3)
    return (np.rint(v / step) * step).astype(np.float32)


def _scaled(v, a):
    a = np.maximum(a, np.float32(2.0 ** -100)).astype(np.float32)
    return e4m3(v * (np.float32(448) * (np.float32(1) / a))), a * (np.float32(1) / np.float32(448))


def quantize_rows(x):
    """(values [M, K], scales [K / 128, M]) of float32 x, in numpy."""
    x = np.asarray(x, np.float32)
    M, K = x.shape
    q, s = np.empty_like(x), np.empty((-(-K // 128), M), np.float32)
    for b in range(s.shape[0]):
        v = x[:, 128 * b:128 * b + 128]
        q[:, 128 * b:128 * b + 128], c = _scaled(v, np.abs(v).max(1, keepdims=True))
        s[b] = c[:, 0]
    return q, s


def quantize_blocks(w):
    w = np.asarray(w, np.float32)
    N, K = w.shape
    q, s = np.empty_like(w), np.empty((-(-N // 128), -(-K // 128)), np.float32)
    for a in range(s.shape[0]):
        for b in range(s.shape[1]):
            at = np.s_[128 * a:128 * a + 128, 128 * b:128 * b + 128]
            q[at], c = _scaled(w[at], np.abs(w[at]).max(keepdims=True))
            s[a, b] = c[0, 0]
    return q, s


def rows_f64(q, s):
    """The values that quantized rows stand for."""
    wide = s.double().t().repeat_interleave(128, 1)[:, :q.shape[1]]
    return q.double() * wide


def blocks_f64(q, s):
    N, K = q.shape[-2:]
    wide = s.double().repeat_interleave(128, -2)[..., :N, :].repeat_interleave(128, -1)[..., :K]
    return q.double() * wide


def f8_error(x, w):
    """How far the matrix cores' sums of 8-bit products x w^T may be off (x, w float64 with
    their scales).  They add 8 consecutive products as multiples of 2^-13 of the largest one's
    power of two, cutting the others off toward zero, and the sums of 8 in fp32.  A product is at
    least the power of two of its factors' exponents, and the largest of 8 has no bits below
    2^-6 of that: at most 7 of 8 are cut, each by less than 2^-13 of the largest.  The largest
    of 8 products is at most the product of the largest factors."""
    K = x.shape[1]
    top = lambda v: torch.nn.functional.pad(v.abs(), (0, -K % 8)).reshape(v.shape[0], -1, 8).amax(2)  # noqa: E731
    return 7 * 2.0 ** -13 * (top(x) @ top(w).t()) + (K / 8 + 8) * 2.0 ** -24 * (x.abs() @ w.abs().t())
