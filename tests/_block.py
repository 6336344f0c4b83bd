"""64-bit plain forms of the feed-forward block's operators, for the tests."""
import math

import numpy as np
import torch

_LOW = 0xFFFFFFFF


def philox4x32(block, counter, seed):
    """Philox4x32-10 of counter words (block, block >> 32, counter, counter >> 32)
    keyed by seed, for an array of block numbers; uint32 [blocks, 4]."""
    b = np.asarray(block, np.uint64)
    low, sh = np.uint64(_LOW), np.uint64(32)
    c = [b & low, b >> sh, np.full_like(b, counter & _LOW), np.full_like(b, (counter >> 32) & _LOW)]
    k0, k1 = seed & _LOW, (seed >> 32) & _LOW
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> sh) ^ c[1] ^ np.uint64(k0), p1 & low, (p0 >> sh) ^ c[3] ^ np.uint64(k1), p0 & low]
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    return np.stack(c, 1).astype(np.uint32)


def threshold(p):
    return 0 if p == 0 else 65536 if p == 1 else min(65535, max(1, round(p * 65536)))


def keep(n, p, seed, counter):
    """Boolean keep mask of n elements."""
    w = philox4x32(np.arange((n + 7) // 8), counter & (1 << 64) - 1, seed & (1 << 64) - 1)
    return w.view(np.uint16).reshape(-1)[:n] >= threshold(p)   # little endian: low half first


def keep_scale(p):
    t = threshold(p)
    return 0.0 if t == 65536 else 65536 / (65536 - t)


def act(name, v):
    """act(v) and act'(v) in float64."""
    if name == "none":
        return v, torch.ones_like(v)
    if name == "relu":
        return v.clamp_min(0), (v > 0).double()
    if name == "silu":
        s = torch.sigmoid(v)
        return v * s, s * (1 + v * (1 - s))
    c = math.sqrt(2 / math.pi)
    th = torch.tanh(c * (v + 0.044715 * v ** 3))
    return 0.5 * v * (1 + th), 0.5 * (1 + th) + 0.5 * v * (1 - th * th) * c * (1 + 3 * 0.044715 * v * v)


def mlp(x, wg, wu, wd, dy, name, unit, e32):
    """{name: (value, bound)} of the gated MLP and its gradients in float64.  `unit`
    is the relative error of a rounding to the operands' type (2^-8 for bf16's 8
    significant bits: h, dg, du and the outputs), e32 the relative error of an fp32 sum
    against the sum of its terms' magnitudes."""
    x, wg, wu, wd, dy = (t.double() for t in (x, wg, wu, wd, dy))
    g, u, dh = x @ wg.t(), x @ wu.t(), dy @ wd
    eg, eu = e32 * (x.abs() @ wg.abs().t()), e32 * (x.abs() @ wu.abs().t())
    edh = e32 * (dy.abs() @ wd.abs())
    a, da = act(name, g)
    # |act'| <= 1.2, |act''| <= 1.2 for these activations (relu: where g's sign is sure)
    ea, eda = 1.2 * eg + e32 * a.abs(), 1.2 * eg + e32
    if name == "relu":
        eda = torch.where(g.abs() <= eg, 1.0, 0.0) + e32 * da
    h, dg, du = a * u, dh * u * da, dh * a
    eh = ea * u.abs() + a.abs() * eu + ea * eu
    edg = edh * (u * da).abs() + dh.abs() * (eu * da.abs() + u.abs() * eda) + 4 * e32 * dg.abs()
    edu = edh * a.abs() + dh.abs() * ea + 4 * e32 * du.abs()
    eh, edg, edu = eh + unit * h.abs(), edg + unit * dg.abs(), edu + unit * du.abs()

    def product(p, ep, q):
        v = p @ q
        return v, ep @ q.abs() + e32 * (p.abs() @ q.abs()) + unit * v.abs()

    y = product(h, eh, wd.t())
    dx0, dx1 = product(dg, edg, wg), product(du, edu, wu)
    out = dict(y=y, dx=(dx0[0] + dx1[0], dx0[1] + dx1[1] + unit * (dx0[0] + dx1[0]).abs()))
    out["dgate"] = product(dg.t(), edg.t(), x)
    out["dup"] = product(du.t(), edu.t(), x)
    out["ddown"] = product(dy.t(), torch.zeros_like(dy.t()), h)
    out["ddown"] = (out["ddown"][0], out["ddown"][1] + dy.abs().t() @ eh)
    return out


def norm(v, kind, eps):
    d = v - v.mean(1, keepdim=True) if kind == "layer" else v
    r = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + eps)
    return d * r, r


def norm_back(dv, vhat, r, kind):
    d = dv - vhat * (dv * vhat).mean(1, keepdim=True)
    if kind == "layer":
        d = d - dv.mean(1, keepdim=True)
    return d * r


def norm_back_size(dv, vhat, r):
    """The magnitudes of norm_back's terms, which cancel where a row is narrow."""
    return r * (dv + vhat.abs() * (dv * vhat.abs()).mean(1, keepdim=True) + dv.mean(1, keepdim=True))


def residual_norm(o, kind, eps, p, seed, counter):
    """Values, and for the sums over rows and d_x, d_branch the terms' magnitudes.  o: dict of
    x, branch, gate [groups, dim], scale, post_weight, ..., dy, dn; absent ones None."""
    o = {k: None if v is None else v.double().cpu() for k, v in o.items()}
    x, b = o["x"], o["branch"]
    rows, dim = x.shape
    one = torch.ones(dim, dtype=torch.float64)
    out, size = {}, {}
    gate = None if o["gate"] is None else o["gate"].reshape(-1, dim).repeat_interleave(
        rows // o["gate"].reshape(-1, dim).shape[0], 0)
    s = one if o["scale"] is None else o["scale"]
    k = torch.from_numpy(keep(rows * dim, p, seed, counter)).reshape(rows, dim) if p else None
    sc = keep_scale(p)
    y = x * s
    if b is not None:
        c, bhat = b, b
        if o["post_weight"] is not None:
            bhat, rb = norm(b, kind, eps)
            c = bhat * o["post_weight"] + (0 if o["post_bias"] is None else o["post_bias"])
        z = c if gate is None else c * gate
        if k is not None:
            z = torch.where(k, z * sc, 0.0)
        y = y + z
    out["y"] = y
    if o["next_weight"] is not None:
        yh, ry = norm(y, kind, eps)
        out["n"] = yh * o["next_weight"] + (0 if o["next_bias"] is None else o["next_bias"])
    if o.get("dy") is None and o.get("dn") is None:
        return out, size
    d = torch.zeros_like(x) if o["dy"] is None else o["dy"]
    dn = o.get("dn")
    sd = d.abs()
    if dn is not None:
        d = d + norm_back(dn * o["next_weight"], yh, ry, kind)
        sd = sd + norm_back_size((dn * o["next_weight"]).abs(), yh, ry)

    def total(name, t):
        out[name], size[name] = t.sum(0), t.abs().sum(0)

    if o["next_weight"] is not None:
        total("d_next_weight", torch.zeros_like(x) if dn is None else dn * yh)
        if o["next_bias"] is not None:
            total("d_next_bias", torch.zeros_like(x) if dn is None else dn)
    out["d_x"], size["d_x"] = d * s, sd * s.abs()
    if o["scale"] is not None:
        total("d_scale", d * x)
    if b is None:
        return out, size
    dz = d if k is None else torch.where(k, d * sc, 0.0)
    sd = sd * max(sc, 1.0) if p else sd
    if gate is not None:
        groups = o["gate"].reshape(-1, dim).shape[0]
        t = (dz * c).reshape(groups, rows // groups, dim)
        out["d_gate"], size["d_gate"] = t.sum(1), t.abs().sum(1)
        dz, sd = dz * gate, sd * gate.abs()
    if o["post_weight"] is not None:
        total("d_post_weight", dz * bhat)
        if o["post_bias"] is not None:
            total("d_post_bias", dz)
        dz = norm_back(dz * o["post_weight"], bhat, rb, kind)
        sd = norm_back_size(sd * o["post_weight"].abs(), bhat, rb)
    out["d_branch"], size["d_branch"] = dz, sd
    return out, size
