"""Mixture-of-experts and block-scaled 8-bit operators, as timed cases.

Each case is one forward pass or one training step (forward, then backward)
through the public entry points, on resident device inputs.  ``own`` chooses
the framework's kernels (True) or the plain form in elementary 32-bit torch
operations (False).  ``exact`` computes the same outputs from the definitions
in 64 bits.

route       T tokens with k experts each are T k slots (slot t k + j), sorted by
            expert, stably; an expert outside 0 .. E - 1 drops its slot, and the
            dropped slots follow the last expert's.  pos[t, j] is the sorted row
            of a slot, offsets[e] expert e's first row, offsets[E] the first
            dropped one.
              dispatch  xs[pos[t, j]] = x[t]          (0 where dropped)
              combine   y[t] = sum_j w[t, j] ys[pos[t, j]]  (over those kept)
            and their gradients: dx[t] = sum_j dxs[pos[t, j]],
            dys[pos[t, j]] = w[t, j] dy[t], dw[t, j] = <dy[t], ys[pos[t, j]]>,
            both 0 where dropped
experts     the gated MLP of each token's experts, between dispatch and combine:
            ys_r = (act(xs_r Wg_e^T) * (xs_r Wu_e^T)) Wd_e^T for r's expert e,
            with the gradients of x, the weights w and every expert's matrices
f8_linear   y = act(x^ W^T + bias) with x^ and W in 8-bit floating point (e4m3):
            x^ is quantized in the call, a scale for each 128 features of a row;
            W comes quantized, a scale for each 128 x 128 block
f8_experts  the experts' layer on such weights; x and the hidden
            features h = act(g) u are quantized in the call

The quantization of a block: a = max(|v|, 2^-100) over it, scale a / 448, values
e4m3(v * (448 / a)) rounded to the nearest even, all in Float32.
"""
import math

import torch

own = False

BF16, F32 = "bf16", "f32"
_DT = {BF16: torch.bfloat16, F32: torch.float32}


def listed():
    return [
        # one decoding step of 32 sequences, 8 of 64 experts each: latency
        dict(name="route_decode", kind="route", tokens=32, topk=8, experts=64, dim=4096,
             dtype=BF16, drop=0.0, train=False),
        # a training batch of 8192 tokens, 8 of 64 experts each
        dict(name="route_train", kind="route", tokens=8192, topk=8, experts=64, dim=4096,
             dtype=BF16, drop=0.0, train=True),
        # a ragged Float32 batch of an odd width, some slots dropped
        dict(name="route_odd_f32", kind="route", tokens=1000, topk=3, experts=10, dim=1001,
             dtype=F32, drop=0.1, train=True),
        # decode: one token through 2 of 8 experts of 4096 -> 11008 -> 4096
        dict(name="experts_token", kind="experts", tokens=1, topk=2, experts=8, dim=4096,
             inner=11008, act="silu", drop=0.0, train=False),
        # prefill of 2048 tokens through 4 of 32 small experts
        dict(name="experts_prefill", kind="experts", tokens=2048, topk=4, experts=32, dim=2048,
             inner=1408, act="silu", drop=0.0, train=False),
        # a training step of 4096 tokens through 2 of 8 experts: the largest case
        dict(name="experts_train", kind="experts", tokens=4096, topk=2, experts=8, dim=4096,
             inner=5504, act="silu", drop=0.0, train=True),
        # a training step on a ragged batch, with slots over the experts' capacity dropped
        dict(name="experts_train_ragged", kind="experts", tokens=1000, topk=3, experts=16, dim=1040,
             inner=712, act="gelu", drop=0.05, train=True),
        # decode, one token: the up projection of a 4096 -> 11008 layer
        dict(name="f8_token", kind="f8_linear", rows=1, n=11008, k=4096, act="none", bias=False),
        # prefill of 2048 tokens through the same projection
        dict(name="f8_prefill", kind="f8_linear", rows=2048, n=11008, k=4096, act="none",
             bias=False),
        # a ragged batch, widths that end inside a block, with the whole epilogue
        dict(name="f8_ragged", kind="f8_linear", rows=1000, n=3000, k=1040, act="gelu", bias=True),
        # batched decode: 48 sequences through 2 of 8 experts
        dict(name="f8_experts_batch", kind="f8_experts", tokens=48, topk=2, experts=8, dim=4096,
             inner=11008, act="silu", drop=0.0),
        # prefill of 4096 tokens through 2 of 8 experts
        dict(name="f8_experts_prefill", kind="f8_experts", tokens=4096, topk=2, experts=8, dim=4096,
             inner=5504, act="silu", drop=0.0),
    ]


def draw(rng):
    def size(lo, hi, step=1):
        """Log-uniform multiples of step in [lo, hi]; half of the draws from 128 on
        are multiples of 128, as most layer widths are, and the rest are what comes."""
        v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        if v >= 128 and rng.random() < 0.5:
            v = v // 128 * 128
        return max(lo, min(hi, v // step * step))

    while True:
        kind = rng.choice(["route", "route", "experts", "experts", "f8_linear", "f8_linear",
                           "f8_experts"])
        if kind == "f8_linear":
            c = dict(kind=kind, rows=size(1, 4096), n=size(64, 11008), k=size(64, 11008, 16),
                     act=rng.choice(["none", "silu", "gelu", "relu"]), bias=rng.random() < 0.5)
            if c["rows"] * c["n"] * c["k"] <= 2048 * 11008 * 4096:
                return c
            continue
        topk = rng.randint(1, 8)
        experts = max(topk, size(2, 64 if kind != "route" else 256))
        drop = rng.choice([0.0, 0.0, 0.1])
        if kind == "route":
            c = dict(kind=kind, tokens=size(1, 16384), topk=topk, experts=experts,
                     dim=size(16, 8192), dtype=rng.choice([BF16, BF16, F32]), drop=drop,
                     train=rng.random() < 0.5)
            if c["tokens"] * topk * c["dim"] <= 8192 * 8 * 4096 // (1 if c["dtype"] == BF16 else 2):
                return c
            continue
        step = 8 if kind == "experts" else 16
        c = dict(kind=kind, tokens=size(1, 4096), topk=topk, experts=experts,
                 dim=size(64, 4096, step), inner=size(64, 11008, step),
                 act=rng.choice(["silu", "gelu", "relu"]), drop=drop)
        if kind == "experts":
            c["train"] = rng.random() < 0.5
        wide = c["dim"] * c["inner"]
        if c["tokens"] * topk * wide <= 8192 * 5504 * 4096 and experts * wide <= 8 * 5504 * 4096:
            return c


class _Gen:
    """Seeded device tensors: the same seed gives the same sequence."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(1000003 * int(seed) + 31)

    def normal(self, shape, dtype=torch.float32, std=1.0):
        return (torch.randn(shape, generator=self.g, device="cuda") * std).to(dtype)

    def uniform(self, shape):
        return torch.rand(shape, generator=self.g, device="cuda")


def _f8(v):
    return v.to(torch.float8_e4m3fn)


def _blocks_of(v, rows):
    """v [..., N, K] zero-padded to whole blocks of rows x 128, as [..., N/rows, rows, K/128, 128]."""
    n, k = v.shape[-2:]
    v = torch.nn.functional.pad(v, (0, -k % 128, 0, -n % rows))
    return v.reshape(*v.shape[:-2], v.shape[-2] // rows, rows, v.shape[-1] // 128, 128)


def _quantize(v, rows):
    """(values, scales, values as the numbers they stand for) of v [..., N, K] in Float32."""
    n, k = v.shape[-2:]
    b = _blocks_of(v.float(), rows)
    a = b.abs().amax(dim=(-3, -1), keepdim=True).clamp_min(2.0 ** -100)
    q = _f8(b * (448.0 / a))
    scale = a / 448.0
    cut = lambda t: t.reshape(*t.shape[:-4], t.shape[-4] * rows, -1)[..., :n, :k]  # noqa: E731
    return cut(q).contiguous(), scale[..., 0, :, 0].contiguous(), cut(q.float() * scale)


def _routing(g, case):
    """Each token's experts (int64, -1: dropped) and weights; some experts are busier."""
    t, k, e = case["tokens"], case["topk"], case["experts"]
    logits = g.normal((t, e)) + 0.5 * g.normal((e,))
    top, ids = torch.topk(logits, k, dim=1)
    if case["drop"]:
        ids = torch.where(g.uniform((t, k)) < case["drop"], -1, ids)
    return ids, torch.softmax(top, dim=1)


def prepare(case, seed):
    g, kind = _Gen(seed), case["kind"]
    s = dict(case=case)
    if kind == "f8_linear":
        m, n, k = case["rows"], case["n"], case["k"]
        s["x"] = g.normal((m, k), torch.bfloat16)
        s["w"], s["ws"], _ = _quantize(g.normal((n, k), std=k ** -0.5), 128)
        s["bias"] = g.normal((n,), std=0.1) if case["bias"] else None
        return s
    s["experts"], s["weights"] = _routing(g, case)
    t, k, d = case["tokens"], case["topk"], case["dim"]
    dt = _DT[case.get("dtype", BF16)]
    s["x"] = g.normal((t, d), dt)
    if kind == "route":
        s["ys"] = g.normal((t * k, d), dt)
        if case["train"]:
            s["dxs"], s["dy"] = g.normal((t * k, d), dt), g.normal((t, d), dt)
        return s
    e, i = case["experts"], case["inner"]
    for name, shape in (("gate", (e, i, d)), ("up", (e, i, d)), ("down", (e, d, i))):
        w = g.normal(shape, std=shape[2] ** -0.5)
        if kind == "experts":
            s[name] = w.to(dt)
        else:
            s[name], s[name + "_scale"], _ = _quantize(w, 128)
    if kind == "experts" and case["train"]:
        s["dy"] = g.normal((t, d), dt)
    return s


# ------------------------------------------------------------------ plain forms
def _sort_plain(ids, experts):
    """pos and offsets by counting: a slot's row is the number of slots of lower experts
    and of earlier slots of its own."""
    e = ids.reshape(-1)
    e = torch.where((e < 0) | (e >= experts), experts, e)
    one = (e[:, None] == torch.arange(experts + 1, device=e.device)).to(torch.int32)
    count = torch.cumsum(one, dim=0)
    first = torch.cumsum(count[-1], dim=0) - count[-1]
    pos = first[e] + count.gather(1, e[:, None])[:, 0] - 1
    return pos.to(torch.int32).reshape(ids.shape), first.to(torch.int32)


def _dispatch_plain(x, pos, kept):
    xs = torch.zeros((pos.numel(), x.shape[1]), device=x.device)
    for j in range(pos.shape[1]):
        xs[pos[:, j].long()] = x.float() * kept[:, j, None]
    return xs


def _gather_plain(ys, w, pos, kept):
    y = 0.0
    for j in range(pos.shape[1]):
        y = y + torch.where(kept[:, j, None], w[:, j, None] * ys[pos[:, j].long()].float(), 0.0)
    return y


def _combine_back_plain(dy, ys, w, pos, kept):
    dys = torch.zeros(ys.shape, device=ys.device)
    dw = torch.zeros_like(w)
    for j in range(pos.shape[1]):
        at = pos[:, j].long()
        dys[at] = torch.where(kept[:, j, None], w[:, j, None] * dy, 0.0)
        dw[:, j] = torch.where(kept[:, j], (dy * ys[at].float()).sum(dim=1), 0.0)
    return dys, dw


def _route_plain(s):
    case, dt, w = s["case"], s["x"].dtype, s["weights"]
    pos, offsets = _sort_plain(s["experts"], case["experts"])
    kept = pos < offsets[-1]
    out = dict(pos=pos, offsets=offsets, xs=_dispatch_plain(s["x"], pos, kept).to(dt),
               y=_gather_plain(s["ys"], w, pos, kept).to(dt))
    if case["train"]:
        out["dx"] = _gather_plain(s["dxs"], torch.ones_like(w), pos, kept).to(dt)
        dys, out["dw"] = _combine_back_plain(s["dy"].float(), s["ys"], w, pos, kept)
        out["dys"] = dys.to(dt)
    return out


def _act_plain(name, v):
    """act(v) and its derivative."""
    if name == "none":
        return v, torch.ones_like(v)
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


def _experts_plain(s):
    case, dt, w = s["case"], s["x"].dtype, s["weights"]
    pos, offsets = _sort_plain(s["experts"], case["experts"])
    kept = pos < offsets[-1]
    xs = _dispatch_plain(s["x"], pos, kept)
    ys, rows, keep = torch.zeros_like(xs), offsets.tolist(), []
    for e, (a, b) in enumerate(zip(rows[:-1], rows[1:])):
        if a == b:
            keep.append(None)
            continue
        x, wg, wu, wd = xs[a:b], s["gate"][e].float(), s["up"][e].float(), s["down"][e].float()
        g, u = x @ wg.t(), x @ wu.t()
        act, dact = _act_plain(case["act"], g)
        ys[a:b] = (act * u) @ wd.t()
        keep.append((x, wg, wu, wd, u, act, dact) if case["train"] else None)
    out = dict(y=_gather_plain(ys, w, pos, kept).to(dt))
    if not case["train"]:
        return out
    dys, out["dw"] = _combine_back_plain(s["dy"].float(), ys, w, pos, kept)
    dxs = torch.zeros_like(xs)
    for name in ("gate", "up", "down"):
        out["d" + name] = torch.zeros_like(s[name])
    for e, (a, b) in enumerate(zip(rows[:-1], rows[1:])):
        if keep[e] is None:
            continue
        x, wg, wu, wd, u, act, dact = keep[e]
        d = dys[a:b]
        dh = d @ wd
        dg, du = dh * u * dact, dh * act
        dxs[a:b] = dg @ wg + du @ wu
        out["dgate"][e], out["dup"][e] = (dg.t() @ x).to(dt), (du.t() @ x).to(dt)
        out["ddown"][e] = (d.t() @ (act * u)).to(dt)
    out["dx"] = _gather_plain(dxs, torch.ones_like(w), pos, kept).to(dt)
    return out


def _wide_scales(scale, n, k):
    """128 x 128 block scales for every element of an [n, k] matrix."""
    return scale.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]


def _f8_linear_plain(s):
    x = _quantize(s["x"], 1)[2]
    y = x @ (s["w"].float() * _wide_scales(s["ws"], *s["w"].shape)).t()
    if s["bias"] is not None:
        y = y + s["bias"]
    return dict(y=_act_plain(s["case"]["act"], y)[0].to(torch.bfloat16))


def _f8_experts_plain(s):
    case = s["case"]
    pos, offsets = _sort_plain(s["experts"], case["experts"])
    kept = pos < offsets[-1]
    xs = _dispatch_plain(_quantize(s["x"], 1)[2], pos, kept)
    ys, rows = torch.zeros_like(xs), offsets.tolist()
    for e, (a, b) in enumerate(zip(rows[:-1], rows[1:])):
        if a < b:
            wg, wu, wd = (s[n][e].float() * _wide_scales(s[n + "_scale"][e], *s[n][e].shape)
                          for n in ("gate", "up", "down"))
            h = _act_plain(case["act"], xs[a:b] @ wg.t())[0] * (xs[a:b] @ wu.t())
            ys[a:b] = _quantize(h, 1)[2] @ wd.t()
    return dict(y=_gather_plain(ys, s["weights"], pos, kept).to(torch.bfloat16))


# ------------------------------------------------------------------ the framework's
def _route_own(s):
    import momijo_amd as mj

    plan = mj.sort_experts(s["experts"], s["case"]["experts"])
    out = dict(pos=plan.pos, offsets=plan.offsets, xs=mj.dispatch(s["x"], plan),
               y=mj.combine(s["ys"], s["weights"], plan))
    if s["case"]["train"]:
        out["dx"] = mj.dispatch_backward(s["dxs"], plan)
        out["dys"], out["dw"] = mj.combine_backward(s["dy"], s["ys"], s["weights"], plan)
    return out


def _act_own(name):
    import momijo_amd as mj

    return {"none": mj.EPI_NONE, "silu": mj.EPI_SILU, "gelu": mj.EPI_GELU_TANH,
            "relu": mj.EPI_RELU}[name]


def _experts_own(s):
    import momijo_amd as mj

    layer = mj.ExpertsMLP(s["gate"], s["up"], s["down"], _act_own(s["case"]["act"]))
    if not s["case"]["train"]:
        return dict(y=layer.forward(s["x"], s["experts"], s["weights"]))
    y, saved = layer.forward_train(s["x"], s["experts"], s["weights"])
    g = layer.backward(s["dy"], saved)
    return dict(y=y, dx=g["x"], dw=g["weights"], dgate=g["gate"], dup=g["up"], ddown=g["down"])


def _f8_linear_own(s):
    import momijo_amd as mj

    layer = mj.F8Linear(s["w"], s["ws"], s["bias"], _act_own(s["case"]["act"]))
    return dict(y=layer.forward(s["x"]))


def _f8_experts_own(s):
    import momijo_amd as mj

    layer = mj.F8Experts(s["gate"], s["gate_scale"], s["up"], s["up_scale"], s["down"],
                         s["down_scale"], _act_own(s["case"]["act"]))
    return dict(y=layer.forward(s["x"], s["experts"], s["weights"]))


_PLAIN = dict(route=_route_plain, experts=_experts_plain, f8_linear=_f8_linear_plain,
              f8_experts=_f8_experts_plain)
_OWN = dict(route=_route_own, experts=_experts_own, f8_linear=_f8_linear_own,
            f8_experts=_f8_experts_own)


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["kind"]](state)


# ------------------------------------------------------------------ work and 64 bits
def _busy(case):
    """The experts that T tokens with k different ones each reach, if all are as likely."""
    e = case["experts"]
    return e * (1.0 - (1.0 - case["topk"] / e) ** case["tokens"])


def work(case):
    kind = case["kind"]
    if kind == "f8_linear":
        m, n, k = case["rows"], case["n"], case["k"]
        nbytes = 2 * m * k + n * k + 4 * math.ceil(n / 128) * math.ceil(k / 128) + 2 * m * n
        return dict(bytes=nbytes + (4 * n if case["bias"] else 0), flops=2 * m * n * k)
    t, k, d = case["tokens"], case["topk"], case["dim"]
    r = t * k
    if kind == "route":
        z = 2 if case["dtype"] == BF16 else 4
        rows, flops = 2 * t + 2 * r, 2 * r * d      # x, y; xs, ys
        nbytes = 8 * r + 4 * r + 4 * r              # ids, pos, weights
        if case["train"]:                           # dx, dy; dxs, dys
            rows, flops, nbytes = rows + 2 * t + 2 * r, flops + 4 * r * d, nbytes + 4 * r
        return dict(bytes=z * rows * d + nbytes + 4 * (case["experts"] + 1), flops=flops)
    i = case["inner"]
    kept = r * (1.0 - case["drop"])
    flops = 2 * kept * 3 * d * i
    if kind == "f8_experts":
        weights = 3 * _busy(case) * d * i
        return dict(bytes=int(weights + 4 * t * d + 12 * r), flops=int(flops))
    weights = 2 * 3 * _busy(case) * d * i
    nbytes = weights + 4 * t * d + 12 * r
    if case["train"]:  # dy read, dx written; the weights' gradients written, of idle experts too
        nbytes += 4 * t * d + 4 * r + 2 * 3 * case["experts"] * d * i
        flops *= 3
    return dict(bytes=int(nbytes), flops=int(flops))


def _e4m3_exact(v):
    """Float32 values up to 448 in magnitude, to the nearest e4m3 (ties to even), in 64 bits."""
    v = v.double()
    exponent = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6)))
    step = torch.exp2(exponent - 3)            # 3 bits after the leading one; 2^-9 below 2^-6
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def _rows_exact(x):
    """The values that a row's quantization stands for; scales and quotients are Float32 by
    definition."""
    parts = []
    for c in x.float().split(128, dim=1):
        a = c.abs().max(dim=1, keepdim=True).values.clamp_min(2.0 ** -100)
        parts.append(_e4m3_exact(c * (448.0 / a)) * (a / 448.0).double())
    return torch.cat(parts, dim=1)


def _matrix_exact(q, scale):
    n, k = q.shape
    rows = torch.arange(n, device=q.device) // 128
    cols = torch.arange(k, device=q.device) // 128
    return q.double() * scale.double()[rows][:, cols]


_ACT_EXACT = {"none": lambda v: v, "relu": torch.relu, "silu": torch.nn.functional.silu,
              "gelu": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}


def exact(case, seed):
    """The definitions in float64; gradients of the experts' layer by differentiating it."""
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "f8_linear":
        y = _rows_exact(s["x"]) @ _matrix_exact(s["w"], s["ws"]).t()
        if s["bias"] is not None:
            y = y + s["bias"].double()
        return dict(y=_ACT_EXACT[case["act"]](y))
    t, k, d, experts = case["tokens"], case["topk"], case["dim"], case["experts"]
    ids = s["experts"].reshape(-1)
    key = torch.where((ids >= 0) & (ids < experts), ids, experts)
    order = torch.sort(key, stable=True).indices           # sorted row -> slot
    counts = torch.bincount(key, minlength=experts + 1)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)[:-1]])
    kept = int(offsets[-1])
    slots = order[:kept]                                   # the rows of the experts
    token = slots // k
    w = s["weights"].double().reshape(-1)

    def back(values, scale):
        """Rows summed into their tokens."""
        v = values if scale is None else values * scale[:, None]
        return torch.zeros(t, d, dtype=torch.float64, device=v.device).index_add(0, token, v)

    if kind == "route":
        pos = torch.empty_like(order)
        pos[order] = torch.arange(t * k, device=order.device)
        whole = lambda v: torch.cat([v, v.new_zeros(t * k - kept, d)])  # noqa: E731
        out = dict(pos=pos.to(torch.int32).reshape(t, k), offsets=offsets.to(torch.int32),
                   xs=whole(s["x"].double()[token]), y=back(s["ys"][:kept].double(), w[slots]))
        if case["train"]:
            dy = s["dy"].double()[token]
            out["dx"] = back(s["dxs"][:kept].double(), None)
            out["dys"] = whole(dy * w[slots][:, None])
            dw = torch.zeros(t * k, dtype=torch.float64, device=w.device)
            dw[slots] = (dy * s["ys"][:kept].double()).sum(1)
            out["dw"] = dw.reshape(t, k)
        return out
    ends = offsets.tolist()
    if kind == "f8_experts":
        xs, ys = _rows_exact(s["x"])[token], []
        for e in range(experts):
            m = lambda n: _matrix_exact(s[n][e], s[n + "_scale"][e])  # noqa: E731
            v = xs[ends[e]:ends[e + 1]]
            if v.shape[0]:
                h = _ACT_EXACT[case["act"]](v @ m("gate").t()) * (v @ m("up").t())
                ys.append(_rows_exact(h) @ m("down").t())
        return dict(y=back(torch.cat(ys) if ys else xs, w[slots]))
    leaves = {n: s[n].double() for n in ("x", "weights", "gate", "up", "down")}
    for v in leaves.values():
        v.requires_grad_(case["train"])
    xs, ys = leaves["x"][token], []
    for e in range(experts):
        v = xs[ends[e]:ends[e + 1]]
        h = _ACT_EXACT[case["act"]](v @ leaves["gate"][e].t()) * (v @ leaves["up"][e].t())
        ys.append(h @ leaves["down"][e].t())
    y = back(torch.cat(ys), leaves["weights"].reshape(-1)[slots])
    out = dict(y=y.detach())
    if case["train"]:
        names = ("x", "weights", "gate", "up", "down")
        grads = torch.autograd.grad(y, [leaves[n] for n in names], s["dy"].double())
        out.update(zip(("dx", "dw", "dgate", "dup", "ddown"), grads))
    return out
