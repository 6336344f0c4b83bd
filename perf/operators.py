"""The operators of a transformer's feed-forward block, as timed cases.

Each case is one forward pass or one training step (forward, then backward)
through the public entry points, on resident device inputs.  ``own`` chooses
the framework's kernels (True) or the plain form in elementary 32-bit torch
operations (False).  ``exact`` computes the same outputs from the definitions
in 64 bits.

mlp            y = (act(x Wg^T) * (x Wu^T)) Wd^T with its gradients
residual_norm  y = scale * x + dropout(gate * norm(branch)), n = norm(y), with
               the gradients of x, the branch and every parameter
dropout        y = x * keep / (1 - p), the keep mask drawn from a counter-based
               generator, and its backward pass (the same mask, drawn again)

The mask.  Philox4x32-10 (Salmon et al., "Parallel random numbers: as easy as
1, 2, 3", 2011) with key = the 64-bit seed and counter words (block, block >>
32, counter, counter >> 32) gives block b's four words; element 8 b + i takes
half i of them (low half of word i / 2 for even i).  It is kept where its 16
bits are >= T = round(65536 p) (at least 1 for p > 0, at most 65535 for p < 1)
and then multiplied by 65536 / (65536 - T).
"""
import math

import numpy as np
import torch

own = False

BF16, F32 = "bf16", "f32"
_DT = {BF16: torch.bfloat16, F32: torch.float32}


def listed():
    return [
        # decode: one token through the FFN of a 4096 -> 11008 -> 4096 layer
        dict(name="mlp_token", kind="mlp", tokens=1, k=4096, i=11008, h=4096, act="silu",
             dtype=BF16, train=False),
        # batched decode: 48 sequences, one token each
        dict(name="mlp_batch", kind="mlp", tokens=48, k=4096, i=11008, h=4096, act="silu",
             dtype=BF16, train=False),
        # prefill of 2048 tokens
        dict(name="mlp_prefill", kind="mlp", tokens=2048, k=4096, i=11008, h=4096, act="silu",
             dtype=BF16, train=False),
        # a training step of 4096 tokens: the largest case
        dict(name="mlp_train", kind="mlp", tokens=4096, k=4096, i=11008, h=4096, act="silu",
             dtype=BF16, train=True),
        # a training step on a ragged batch of a middle-sized layer
        dict(name="mlp_train_ragged", kind="mlp", tokens=1000, k=1040, i=2808, h=1040, act="gelu",
             dtype=BF16, train=True),
        # the Float32 layer that the framework's tape trains
        dict(name="mlp_train_f32", kind="mlp", tokens=1024, k=1024, i=2752, h=1024, act="silu",
             dtype=F32, train=True),
        # decode: the norms at a block boundary for one token
        dict(name="norm_token", kind="residual_norm", rows=1, dim=4096, groups=1, norm="rms",
             post=True, next=True, bias=False, scale=False, p=0.0, dtype=BF16, train=False),
        # training: four sequences of 2048 tokens, a gate of its own for each
        # sequence, dropout on the branch
        dict(name="norm_train", kind="residual_norm", rows=8192, dim=4096, groups=4, norm="rms",
             post=True, next=True, bias=False, scale=True, p=0.1, dtype=BF16, train=True),
        # training of a layer-norm model in Float32, one gate vector
        dict(name="norm_layer_f32", kind="residual_norm", rows=4096, dim=1024, groups=1,
             norm="layer", post=True, next=True, bias=True, scale=False, p=0.0, dtype=F32,
             train=True),
        # an odd width and a ragged batch
        dict(name="norm_odd", kind="residual_norm", rows=1000, dim=1001, groups=1, norm="rms",
             post=False, next=True, bias=False, scale=False, p=0.1, dtype=BF16, train=True),
        # the hidden activations of a training batch
        dict(name="dropout_hidden", kind="dropout", rows=8192, cols=11008, p=0.1, dtype=BF16,
             train=False),
        # forward and backward on a Float32 batch
        dict(name="dropout_train_f32", kind="dropout", rows=1000, cols=1001, p=0.5, dtype=F32,
             train=True),
    ]


def draw(rng):
    def size(lo, hi):
        """Log-uniform in [lo, hi]; half of the draws from 64 on are multiples
        of 64, as most layer widths are, and the rest are what comes."""
        v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        if v >= 64 and rng.random() < 0.5:
            v = v // 64 * 64
        return max(lo, min(hi, v))

    while True:
        kind = rng.choice(["mlp", "mlp", "residual_norm", "dropout"])
        dtype = rng.choice([BF16, BF16, BF16, F32])
        if kind == "mlp":
            k = size(64, 4096)
            c = dict(kind=kind, tokens=size(1, 8192), k=k, i=size(64, 11008),
                     h=rng.choice([k, k, size(64, 4096)]), act=rng.choice(["silu", "gelu", "relu"]),
                     dtype=dtype, train=rng.random() < 0.5)
            if c["tokens"] * c["i"] * (2 * k + c["h"]) > 4096 * 11008 * 3 * 4096:
                continue
            if dtype == F32 and c["tokens"] * c["i"] * (2 * k + c["h"]) > 4 * 1024 ** 4:
                continue
            return c
        if kind == "residual_norm":
            groups = rng.choice([0, 1, 1, 2, 7])
            rows = size(1, 8192)
            rows = max(1, rows // max(1, groups)) * max(1, groups)
            c = dict(kind=kind, rows=rows, dim=size(16, 8192), groups=groups,
                     norm=rng.choice(["rms", "layer"]), post=rng.random() < 0.7,
                     next=rng.random() < 0.8, bias=rng.random() < 0.3, scale=rng.random() < 0.5,
                     p=rng.choice([0.0, 0.1, 0.25]), dtype=dtype, train=rng.random() < 0.6)
            if c["rows"] * c["dim"] > 8192 * 4096 * (1 if dtype == BF16 else 0.5):
                continue
            return c
        c = dict(kind=kind, rows=size(1, 8192), cols=size(16, 11008),
                 p=rng.choice([0.05, 0.1, 0.25, 0.5]), dtype=dtype, train=rng.random() < 0.5)
        if c["rows"] * c["cols"] <= 8192 * 11008 // (2 if c["train"] or dtype == F32 else 1):
            return c


class _Gen:
    """Seeded device tensors: the same seed gives the same sequence."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(1000003 * int(seed) + 29)

    def normal(self, shape, dtype=torch.float32, mean=0.0, std=1.0):
        t = torch.randn(shape, generator=self.g, device="cuda")
        return (t * std + mean).to(dtype)


def prepare(case, seed):
    g, kind, dt = _Gen(seed), case["kind"], _DT[case["dtype"]]
    s = dict(case=case, seed=10007 * int(seed) + 3, counter=int(seed) % 1000)
    if kind == "mlp":
        m, k, i, h = case["tokens"], case["k"], case["i"], case["h"]
        s.update(x=g.normal((m, k), dt), gate=g.normal((i, k), dt, std=k ** -0.5),
                 up=g.normal((i, k), dt, std=k ** -0.5), down=g.normal((h, i), dt, std=i ** -0.5))
        if case["train"]:
            s["dy"] = g.normal((m, h), dt)
        return s
    if kind == "residual_norm":
        m, d = case["rows"], case["dim"]
        s.update(x=g.normal((m, d), dt), branch=g.normal((m, d), dt, mean=0.1))
        s["gate"] = g.normal((case["groups"], d), dt, mean=0.5, std=0.2) if case["groups"] else None
        s["scale"] = g.normal((d,), mean=1.0, std=0.05) if case["scale"] else None
        for name in ("post", "next"):
            on = case[name]
            s[name + "_weight"] = g.normal((d,), mean=1.0, std=0.1) if on else None
            s[name + "_bias"] = g.normal((d,), std=0.1) if on and case["bias"] else None
        if case["train"]:
            s["dy"] = g.normal((m, d), dt)
            s["dn"] = g.normal((m, d), dt) if case["next"] else None
        return s
    s["x"] = g.normal((case["rows"], case["cols"]), dt)
    if case["train"]:
        s["dy"] = g.normal((case["rows"], case["cols"]), dt)
    return s


# ------------------------------------------------------------------ plain forms
_LOW = 0xFFFFFFFF


def _keep(shape, p, seed, counter, device):
    """The scaled keep mask (0 or 65536 / (65536 - T)) in 32 bits."""
    n = math.prod(shape)
    t = min(65535, max(1, round(p * 65536)))
    block = torch.arange((n + 7) // 8, dtype=torch.int64, device=device)
    c0, c1, c2, c3 = block & _LOW, block >> 32, counter & _LOW, (counter >> 32) & _LOW
    k0, k1 = seed & _LOW, (seed >> 32) & _LOW
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # modulo 2^64: both halves are right
        c0, c1, c2, c3 = ((b >> 32) & _LOW) ^ c1 ^ k0, b & _LOW, ((a >> 32) & _LOW) ^ c3 ^ k1, a & _LOW
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    c1, c3 = torch.broadcast_to(torch.as_tensor(c1, device=device), c0.shape), c3
    words = torch.stack([c0, c1, c2, c3], dim=1)
    halves = torch.stack([words & 0xFFFF, words >> 16], dim=2).reshape(-1)[:n]
    return ((halves >= t).float() * (65536.0 / (65536 - t))).reshape(shape)


def _act_plain(name, v):
    """act(v) and its derivative."""
    if name == "relu":
        on = (v > 0).float()
        return v * on, on
    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-v))
        return v * s, s * (1.0 + v * (1.0 - s))
    c = math.sqrt(2.0 / math.pi)  # GELU in its tanh form, tanh(t) = 2 / (1 + exp(-2 t)) - 1
    t = c * (v + 0.044715 * v * v * v)
    th = 2.0 / (1.0 + torch.exp(-2.0 * t)) - 1.0
    return 0.5 * v * (1.0 + th), 0.5 * (1.0 + th) + 0.5 * v * (1.0 - th * th) * c * (1.0 + 3 * 0.044715 * v * v)


def _mlp_plain(s):
    case, dt = s["case"], s["x"].dtype
    x, wg, wu, wd = (s[n].float() for n in ("x", "gate", "up", "down"))
    g, u = x @ wg.t(), x @ wu.t()
    a, da = _act_plain(case["act"], g)
    h = a * u
    out = dict(y=(h @ wd.t()).to(dt))
    if case["train"]:
        dy = s["dy"].float()
        dh = dy @ wd
        dg, du = dh * u * da, dh * a
        out.update(dx=(dg @ wg + du @ wu).to(dt), dgate=(dg.t() @ x).to(dt), dup=(du.t() @ x).to(dt),
                   ddown=(dy.t() @ h).to(dt))
    return out


_EPS = 1e-6


def _norm_plain(v, kind):
    """(v - mean) / std (layer) or v / rms, and 1 / std or 1 / rms of each row."""
    if kind == "layer":
        v = v - v.mean(dim=1, keepdim=True)
    r = 1.0 / torch.sqrt((v * v).mean(dim=1, keepdim=True) + _EPS)
    return v * r, r


def _norm_back_plain(dv, v, r, kind):
    """The gradient of _norm_plain's input; v is the normalised row."""
    d = dv - v * (dv * v).mean(dim=1, keepdim=True)
    if kind == "layer":
        d = d - dv.mean(dim=1, keepdim=True)
    return d * r


def _residual_norm_plain(s):
    case = s["case"]
    kind, dt, rows, dim = case["norm"], s["x"].dtype, case["rows"], case["dim"]
    x, b = s["x"].float(), s["branch"].float()
    groups = max(1, case["groups"])
    per = rows // groups
    wide = lambda t: t.float().repeat_interleave(per, dim=0)  # noqa: E731
    z = b
    if case["post"]:
        bhat, rb = _norm_plain(b, kind)
        z = bhat * s["post_weight"]
        if case["bias"]:
            z = z + s["post_bias"]
    c = z
    gate = wide(s["gate"]) if case["groups"] else None
    if gate is not None:
        z = z * gate
    keep = _keep((rows, dim), case["p"], s["seed"], s["counter"], x.device) if case["p"] else None
    if keep is not None:
        z = z * keep
    y = (x * s["scale"] if case["scale"] else x) + z
    out = dict(y=y.to(dt))
    if case["next"]:
        yhat, ry = _norm_plain(y, kind)
        n = yhat * s["next_weight"]
        out["n"] = (n + s["next_bias"] if case["bias"] else n).to(dt)
    if not case["train"]:
        return out
    dy = s["dy"].float()
    if case["next"]:
        dn = s["dn"].float()
        dy = dy + _norm_back_plain(dn * s["next_weight"], yhat, ry, kind)
        out["d_next_weight"] = (dn * yhat).sum(dim=0)
        if case["bias"]:
            out["d_next_bias"] = dn.sum(dim=0)
    out["d_x"] = (dy * s["scale"] if case["scale"] else dy).to(dt)
    if case["scale"]:
        out["d_scale"] = (dy * x).sum(dim=0)
    dz = dy if keep is None else dy * keep
    if gate is not None:
        out["d_gate"] = (dz * c).reshape(groups, per, dim).sum(dim=1).to(dt)
        dz = dz * gate
    if case["post"]:
        out["d_post_weight"] = (dz * bhat).sum(dim=0)
        if case["bias"]:
            out["d_post_bias"] = dz.sum(dim=0)
        dz = _norm_back_plain(dz * s["post_weight"], bhat, rb, kind)
    out["d_branch"] = dz.to(dt)
    return out


def _dropout_plain(s):
    case = s["case"]
    dt = s["x"].dtype
    shape = (case["rows"], case["cols"])
    out = dict(y=(s["x"].float() * _keep(shape, case["p"], s["seed"], s["counter"], s["x"].device)).to(dt))
    if case["train"]:  # the mask is not kept between the passes: drawn again
        out["dx"] = (s["dy"].float() * _keep(shape, case["p"], s["seed"], s["counter"], s["x"].device)).to(dt)
    return out


# ------------------------------------------------------------------ the framework's
def _mlp_own(s):
    import momijo_amd as mj

    case = s["case"]
    act = {"silu": mj.EPI_SILU, "gelu": mj.EPI_GELU_TANH, "relu": mj.EPI_RELU}[case["act"]]
    if not case["train"]:
        return dict(y=mj.gated_mlp(s["x"], s["gate"], s["up"], s["down"], act))
    y, saved = mj.gated_mlp_train(s["x"], s["gate"], s["up"], s["down"], act)
    dx, dgate, dup, ddown = mj.gated_mlp_backward(s["dy"], saved)
    return dict(y=y, dx=dx, dgate=dgate, dup=dup, ddown=ddown)


def _residual_norm_own(s):
    import momijo_amd as mj

    case = s["case"]
    kw = dict(gate=s["gate"], scale=s["scale"], post_weight=s["post_weight"],
              post_bias=s["post_bias"], next_weight=s["next_weight"], next_bias=s["next_bias"],
              norm=case["norm"], eps=_EPS, p=case["p"], seed=s["seed"], counter=s["counter"])
    if not case["train"]:
        y, n = mj.residual_norm(s["x"], s["branch"], **kw)
        return dict(y=y, n=n) if case["next"] else dict(y=y)
    y, n, saved = mj.residual_norm_train(s["x"], s["branch"], **kw)
    grads = mj.residual_norm_backward(s["dy"], s["dn"], saved)
    out = {"d_" + name: v for name, v in grads.items()}
    out["y"] = y
    if case["next"]:
        out["n"] = n
    return out


def _dropout_own(s):
    import momijo_amd as mj

    case = s["case"]
    out = dict(y=mj.dropout(s["x"], case["p"], s["seed"], s["counter"]))
    if case["train"]:
        out["dx"] = mj.dropout_backward(s["dy"], case["p"], s["seed"], s["counter"])
    return out


_PLAIN = dict(mlp=_mlp_plain, residual_norm=_residual_norm_plain, dropout=_dropout_plain)
_OWN = dict(mlp=_mlp_own, residual_norm=_residual_norm_own, dropout=_dropout_own)


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["kind"]](state)


# ------------------------------------------------------------------ work and 64 bits
def work(case):
    kind, e = case["kind"], 2 if case["dtype"] == BF16 else 4
    if kind == "mlp":
        m, k, i, h = case["tokens"], case["k"], case["i"], case["h"]
        nbytes, flops = e * (m * k + 2 * i * k + h * i + m * h), 2 * m * i * (2 * k + h)
        if case["train"]:  # dy read; dx and the weights' gradients written
            nbytes += e * (m * h + m * k + 2 * i * k + h * i)
            flops *= 3
        return dict(bytes=nbytes, flops=flops)
    if kind == "residual_norm":
        m, d = case["rows"], case["dim"]
        wide = 3 + case["next"]                       # x, branch; y, n
        gates = e * case["groups"] * d
        vectors = 4 * d * (case["scale"] + (case["post"] + case["next"]) * (1 + case["bias"]))
        flops = m * d * (4 + 4 * case["post"] + 4 * case["next"])
        if case["train"]:  # dy, dn read; dx, dbranch written
            wide += 3 + case["next"]
            gates *= 2
            vectors *= 2
            flops *= 3
        return dict(bytes=e * m * d * wide + gates + vectors, flops=flops)
    n = case["rows"] * case["cols"]
    times = 2 if case["train"] else 1
    return dict(bytes=2 * e * n * times, flops=2 * n * times)


def _mask_exact(n, p, seed, counter):
    """Philox4x32-10 in numpy's unsigned words; the scaled mask in 64 bits."""
    m0, m1, low, half = np.uint64(0xD2511F53), np.uint64(0xCD9E8D57), np.uint64(_LOW), np.uint64(32)
    blocks = -(-n // 8)
    b = np.arange(blocks, dtype=np.uint64)
    w = [b & low, b >> half, np.full(blocks, counter & _LOW, np.uint64),
         np.full(blocks, (counter >> 32) & _LOW, np.uint64)]
    key = [seed & _LOW, (seed >> 32) & _LOW]
    for _ in range(10):
        p0, p1 = w[0] * m0, w[2] * m1
        w = [(p1 >> half) ^ w[1] ^ np.uint64(key[0]), p1 & low,
             (p0 >> half) ^ w[3] ^ np.uint64(key[1]), p0 & low]
        key = [(key[0] + 0x9E3779B9) & _LOW, (key[1] + 0xBB67AE85) & _LOW]
    bits = np.empty((blocks, 8), np.uint16)
    for j in range(4):
        bits[:, 2 * j] = (w[j] & np.uint64(0xFFFF)).astype(np.uint16)
        bits[:, 2 * j + 1] = (w[j] >> np.uint64(16)).astype(np.uint16)
    t = min(65535, max(1, round(p * 65536)))
    keep = torch.from_numpy(bits.reshape(-1)[:n] >= t).to("cuda")
    return keep.double() * (65536 / (65536 - t))


def exact(case, seed):
    """The definitions in float64, the gradients by differentiating them."""
    s = prepare(case, seed)
    kind = case["kind"]
    wide = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if kind == "dropout":
        mask = _mask_exact(s["x"].numel(), case["p"], s["seed"], s["counter"]).reshape(s["x"].shape)
        out = dict(y=wide["x"] * mask)
        if case["train"]:
            out["dx"] = wide["dy"] * mask
        return out
    leaves = [k for k in wide if k not in ("dy", "dn")]
    if case["train"]:
        for k in leaves:
            wide[k].requires_grad_(True)
    if kind == "mlp":
        g = wide["x"] @ wide["gate"].t()
        act = {"relu": torch.relu, "silu": torch.nn.functional.silu,
               "gelu": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}[case["act"]]
        y = (act(g) * (wide["x"] @ wide["up"].t())) @ wide["down"].t()
        if not case["train"]:
            return dict(y=y)
        d = torch.autograd.grad(y, [wide[k] for k in ("x", "gate", "up", "down")], wide["dy"])
        return dict(y=y.detach(), dx=d[0], dgate=d[1], dup=d[2], ddown=d[3])

    def norm(v, name):
        if case["norm"] == "layer":
            v = torch.nn.functional.layer_norm(v, (v.shape[1],), eps=_EPS)
        else:
            v = v * torch.rsqrt(v.square().mean(1, keepdim=True) + _EPS)
        v = v * wide[name + "_weight"]
        return v + wide[name + "_bias"] if name + "_bias" in wide else v

    rows, dim = case["rows"], case["dim"]
    z = norm(wide["branch"], "post") if case["post"] else wide["branch"]
    if case["groups"]:
        z = (z.reshape(case["groups"], -1, dim) * wide["gate"][:, None, :]).reshape(rows, dim)
    if case["p"]:
        z = z * _mask_exact(rows * dim, case["p"], s["seed"], s["counter"]).reshape(rows, dim)
    y = (wide["x"] * wide["scale"] if case["scale"] else wide["x"]) + z
    n = norm(y, "next") if case["next"] else None
    out = dict(y=y.detach())
    if case["next"]:
        out["n"] = n.detach()
    if case["train"]:
        total = (y * wide["dy"]).sum()
        if case["next"]:
            total = total + (n * wide["dn"]).sum()
        for k, d in zip(leaves, torch.autograd.grad(total, [wide[k] for k in leaves])):
            out["d_" + k] = d
    return out
