"""The operators of a transformer's feed-forward block, forward and backward.

``gated_mlp`` is the gated feed-forward layer, ``residual_norm`` the norms
before and after a block around its residual sum with gate and dropout, and
``dropout`` a dropout whose mask is drawn from a counter and never stored.
Each has a ``_train`` form that also returns what its ``_backward`` needs (the
dropout's backward needs its seed and counter only), and a class that keeps the
parameters.

Tensors are bfloat16 or Float32 on the current device; leading dimensions are
rows.  Operands of other strides are copied to contiguous ones first.  The
kernels run on the current stream, allocate through torch only and can be
captured into a HIP graph.
"""
from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple

import torch

from . import _lib
from .tensor import _ptr, _stream

_DTYPES = {torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}
_NORMS = {"rms": _lib.NORM_RMS, "layer": _lib.NORM_LAYER}
_MASK64 = (1 << 64) - 1


def _check_type(t: torch.Tensor, name: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{name} must be bfloat16 or float32, got {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on the GPU")
    return code


def _like(t: torch.Tensor, x: torch.Tensor, shape, name: str) -> torch.Tensor:
    """t as a contiguous tensor of x's type and device and the given shape."""
    if t.dtype is not x.dtype or t.device != x.device:
        raise TypeError(f"{name} must be {x.dtype} on {x.device}, got {t.dtype} on {t.device}")
    if t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _scratch(nbytes: int, device) -> torch.Tensor:
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


# ------------------------------------------------------------------ dropout
def _seed_args(seed, device):
    """(seed, state) of a call: an integer, or a device int64 tensor {seed, counter}."""
    if type(seed) is int:
        return seed & _MASK64, None
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 2 or seed.device != device or \
                not seed.is_contiguous():
            raise ValueError("a seed tensor is a contiguous int64 tensor {seed, counter} on the "
                             "operand's device")
        return 0, seed
    return int(seed) & _MASK64, None


def dropout(x: torch.Tensor, p: float, seed, counter: int = 0,
            out: torch.Tensor | None = None) -> torch.Tensor:
    """y = x / (1 - p) where the element is kept, else 0.

    The keep mask is a function of (seed, counter, flat element index) alone:
    another counter gives an independent mask, the same one the same mask.  p
    is rounded to a multiple of 2^-16 and the scale is exact for that.  ``seed``
    is an integer or a device int64 tensor {seed, counter}, whose counter is
    added (a captured graph draws a new mask when the tensor changes).
    ``out`` may be x."""
    code = _check_type(x, "x")
    if not x.is_contiguous():
        x = x.contiguous()
    if out is None:
        out = torch.empty_like(x)
    elif out.dtype != x.dtype or out.shape != x.shape or not out.is_contiguous() or \
            out.device != x.device:
        raise ValueError(f"out must be a contiguous {x.dtype} {list(x.shape)} tensor")
    s, state = _seed_args(seed, x.device)
    _lib.call("mj_dropout", code, x.data_ptr(), out.data_ptr(), x.numel(), p, s,
              int(counter) & _MASK64, _ptr(state), _stream())
    return out


def dropout_backward(dy: torch.Tensor, p: float, seed, counter: int = 0,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """The gradient of ``dropout``'s x: the same mask and scale on dy."""
    return dropout(dy, p, seed, counter, out)


class Dropout:
    """Dropout(p, seed): each training ``forward`` draws from the next counter;
    ``backward`` takes the counter that its forward returned.  ``seed`` is as in
    ``dropout``: a captured forward draws a new mask when a seed tensor changes."""

    def __init__(self, p: float, seed=0):
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"p must be in [0, 1], got {p}")
        self.p, self.counter = float(p), 0
        self.seed = seed if isinstance(seed, torch.Tensor) else int(seed)
        self.training = True

    def forward(self, x: torch.Tensor) -> tuple[torch.Tensor, int | None]:
        """(y, counter); in evaluation (x, None)."""
        if not self.training or self.p == 0.0:
            return x, None
        c = self.counter
        self.counter += 1
        return dropout(x, self.p, self.seed, c), c

    def backward(self, dy: torch.Tensor, counter: int | None) -> torch.Tensor:
        return dy if counter is None else dropout_backward(dy, self.p, self.seed, counter)


# ------------------------------------------------------------------ residual norm
class ResidualNormSaved(NamedTuple):
    """What residual_norm_backward needs: the operands, the arguments that the kernels
    take of them, and the rows' statistics."""
    x: torch.Tensor
    branch: torch.Tensor | None
    gate: torch.Tensor | None
    vectors: tuple        # scale, post_weight, post_bias, next_weight, next_bias
    args: tuple           # type, norm, pointers of the operands
    drop: tuple           # p, seed, counter, pointer of the state
    state: torch.Tensor | None
    stats: torch.Tensor


_VECTORS = ("scale", "post_weight", "post_bias", "next_weight", "next_bias")


def _vector(t, device, dim, name):
    if t is None:
        return None
    if t.dtype is not torch.float32 or t.numel() != dim or t.device != device:
        raise ValueError(f"{name} must be float32 with {dim} elements on {device}")
    return t if t.is_contiguous() else t.contiguous()


def _residual_norm(x, branch, gate, scale, post_weight, post_bias, next_weight, next_bias, norm,
                   eps, p, seed, counter, train):
    code = _check_type(x, "x")
    kind = _NORMS.get(norm)
    if kind is None:
        raise ValueError(f"norm must be 'rms' or 'layer', got {norm!r}")
    shape, device = x.shape, x.device
    if not shape:
        raise ValueError("x must have at least one dimension")
    if not x.is_contiguous():
        x = x.contiguous()
    dim = shape[-1]
    rows = x.numel() // dim if dim else 0
    if branch is not None:
        branch = _like(branch, x, shape, "branch")
    gate_rows = 0
    if gate is not None:
        if gate.dim() not in (1, 2) or gate.shape[-1] != dim:
            raise ValueError(f"gate must be [{dim}] or [groups, {dim}], got {list(gate.shape)}")
        gate = _like(gate, x, gate.shape, "gate")
        gate_rows = 1 if gate.dim() == 1 else gate.shape[0]
        if gate_rows == 0 and rows:  # (its pointer is null: no gate, to the call below)
            raise ValueError(f"0 gate rows for {rows} rows")
    scale = _vector(scale, device, dim, "scale")
    wp, bp = _vector(post_weight, device, dim, "post_weight"), _vector(post_bias, device, dim, "post_bias")
    wn, bn = _vector(next_weight, device, dim, "next_weight"), _vector(next_bias, device, dim, "next_bias")
    seed, state = _seed_args(seed, device)
    # without a branch and a scale, y is x itself
    y = x if branch is None and scale is None else torch.empty_like(x)
    n = None if wn is None else torch.empty_like(x)
    stats = torch.empty((4, rows), dtype=torch.float32, device=device) if train else None
    args = (code, kind, x.data_ptr(), _ptr(branch), _ptr(gate), gate_rows, _ptr(scale), _ptr(wp),
            _ptr(bp), _ptr(wn))
    drop = (p, seed, int(counter) & _MASK64, _ptr(state))
    _lib.call("mj_residual_norm", *args, _ptr(bn), eps, *drop, y.data_ptr(), _ptr(n), _ptr(stats),
              rows, dim, _stream())
    if not train:
        return y, n
    return y, n, ResidualNormSaved(x, branch, gate, (scale, wp, bp, wn, bn), args, drop, state, stats)


def residual_norm(x: torch.Tensor, branch: torch.Tensor | None = None, *,
                  gate: torch.Tensor | None = None, scale: torch.Tensor | None = None,
                  post_weight: torch.Tensor | None = None, post_bias: torch.Tensor | None = None,
                  next_weight: torch.Tensor | None = None, next_bias: torch.Tensor | None = None,
                  norm: str = "rms", eps: float = 1e-6, p: float = 0.0, seed=0, counter: int = 0):
    """(y, n): the norm after a block, its gate, dropout, the residual sum and
    the norm before the next block, in one pass over the rows of the last
    dimension:

        y = scale * x + dropout(gate * (norm(branch) * post_weight + post_bias))
        n = norm(y) * next_weight + next_bias

    A norm is applied where its weight is given (n is None without next_weight);
    gate and scale default to 1.  Without ``branch`` the call is the norm before
    the first block: y = scale * x.  ``gate`` is [dim] or [groups, dim] with
    consecutive rows of equal number in each group; x, branch and gate are of one
    type, the vectors Float32."""
    return _residual_norm(x, branch, gate, scale, post_weight, post_bias, next_weight, next_bias,
                          norm, eps, p, seed, counter, False)


def residual_norm_train(x: torch.Tensor, branch: torch.Tensor | None = None, *,
                        gate: torch.Tensor | None = None, scale: torch.Tensor | None = None,
                        post_weight: torch.Tensor | None = None,
                        post_bias: torch.Tensor | None = None,
                        next_weight: torch.Tensor | None = None,
                        next_bias: torch.Tensor | None = None, norm: str = "rms",
                        eps: float = 1e-6, p: float = 0.0, seed=0, counter: int = 0):
    """(y, n, saved): residual_norm and what its backward needs.  The operands are
    kept, not copied: they must not change before the backward."""
    return _residual_norm(x, branch, gate, scale, post_weight, post_bias, next_weight, next_bias,
                          norm, eps, p, seed, counter, True)


@functools.lru_cache(maxsize=1024)
def _norm_work(rows, dim, gate_rows):
    return _lib.load().mj_residual_norm_work_bytes(rows, dim, gate_rows)


def residual_norm_backward(dy: torch.Tensor | None, dn: torch.Tensor | None,
                           saved: ResidualNormSaved) -> dict[str, torch.Tensor]:
    """The gradients of residual_norm's operands, by their names, from the
    gradients of y and n (either may be None, for zero).  Those of x, branch and
    gate have their type, those of the vectors are Float32."""
    x, branch, gate, vectors, args, drop, _, stats = saved
    shape = x.shape
    dim, rows = shape[-1], stats.shape[1]
    if dy is not None:
        dy = _like(dy, x, shape, "dy")
    if dn is not None:
        if vectors[3] is None:
            raise ValueError("dn given, but the forward had no next norm")
        dn = _like(dn, x, shape, "dn")
    out = {"x": torch.empty_like(x)}
    if branch is not None:
        out["branch"] = torch.empty_like(x)
    if gate is not None:
        out["gate"] = torch.empty_like(gate)
    for name, v in zip(_VECTORS, vectors):
        if v is not None:
            out[name] = torch.empty_like(v)
    if rows == 0 or dim == 0 or (dy is None and dn is None):
        return {k: v.zero_() for k, v in out.items()}
    at = {k: v.data_ptr() for k, v in out.items()}
    if dn is None:  # nothing reaches the next norm
        for name in _VECTORS[3:]:
            if name in out:
                out[name].zero_()
                del at[name]
    nbytes = _norm_work(rows, dim, args[5])
    work = _scratch(nbytes, x.device)
    get = at.get
    _lib.call("mj_residual_norm_backward", *args, *drop, stats.data_ptr(), _ptr(dy), _ptr(dn),
              at["x"], get("branch"), get("gate"), get("scale"), get("post_weight"),
              get("post_bias"), get("next_weight"), get("next_bias"), rows, dim, work.data_ptr(),
              nbytes, _stream())
    return out


class ResidualNorm:
    """ResidualNorm(dim, norm, ...): the vectors of residual_norm as Float32
    parameters (weights 1, biases 0) with its options."""

    def __init__(self, dim: int, norm: str = "rms", *, post: bool = True, next: bool = True,
                 bias: bool = False, scale: bool = False, eps: float = 1e-6, p: float = 0.0,
                 seed: int = 0, device=None):
        device = device or torch.device("cuda", torch.cuda.current_device())
        ones = lambda on: torch.ones(dim, device=device) if on else None     # noqa: E731
        zeros = lambda on: torch.zeros(dim, device=device) if on else None   # noqa: E731
        self.dim, self.norm, self.eps, self.p, self.seed = dim, norm, eps, p, seed
        self.scale = ones(scale)
        self.post_weight, self.post_bias = ones(post), zeros(post and bias)
        self.next_weight, self.next_bias = ones(next), zeros(next and bias)
        self.counter = 0
        self.training = True

    def _kw(self, gate, p):
        return dict(gate=gate, scale=self.scale, post_weight=self.post_weight,
                    post_bias=self.post_bias, next_weight=self.next_weight,
                    next_bias=self.next_bias, norm=self.norm, eps=self.eps, p=p, seed=self.seed)

    def forward(self, x, branch, gate=None):
        """(y, n) without dropout."""
        return residual_norm(x, branch, **self._kw(gate, 0.0))

    def forward_train(self, x, branch, gate=None):
        """(y, n, saved); with dropout each call draws from the next counter."""
        c = self.counter
        if self.training and self.p > 0.0:
            self.counter += 1
        return residual_norm_train(x, branch, counter=c,
                                   **self._kw(gate, self.p if self.training else 0.0))

    backward = staticmethod(residual_norm_backward)


# ------------------------------------------------------------------ gated MLP
class GatedMLPSaved(NamedTuple):
    """What gated_mlp_backward needs: the operands, and one buffer with the fp32
    projections g and u, then h, then the zero-padded copies of operands whose widths
    are not multiples of 8 (bf16); ``ptrs`` is where the kernels read x, gate, up, down."""
    x: torch.Tensor
    gate: torch.Tensor
    up: torch.Tensor
    down: torch.Tensor
    buf: torch.Tensor
    ptrs: tuple
    act: int
    rows: torch.Size  # leading dimensions of x


# ctypes makes an array type anew, a cycle for the garbage collector, unless it is kept
_PTRS = [ctypes.c_void_p * n for n in range(5)]
_SIZES = [ctypes.c_int64 * (6 * n) for n in range(5)]


def _copy_rows(mats) -> None:
    """mats: (src pointer, dst pointer, rows, cols, src_ld, dst_rows, dst_cols, dst_ld)."""
    n = len(mats)
    sizes = [v for m in mats for v in m[2:]]
    _lib.call("mj_copy_rows_bf16", n, _PTRS[n](*[m[0] for m in mats]),
              _PTRS[n](*[m[1] for m in mats]), _SIZES[n](*sizes), _stream())


def _up16(n: int) -> int:
    return n + 15 & ~15


def _mlp_operands(x, gate, up, down):
    """x as [M, K] and the weights, checked and contiguous; K, I, H."""
    _check_type(x, "x")
    if x.dim() < 1 or gate.dim() != 2 or down.dim() != 2:
        raise ValueError("x must have a last dimension, and gate, up, down be 2-D")
    K, shape, (H, Iw) = x.shape[-1], gate.shape, down.shape
    if shape[1] != K or Iw != shape[0]:
        raise ValueError(f"x has {K} features, gate is {list(shape)}, down {list(down.shape)}")
    gate = _like(gate, x, shape, "gate")
    up = _like(up, x, shape, "up")
    down = _like(down, x, down.shape, "down")
    x2 = x if x.dim() == 2 else x.reshape(x.shape[:-1].numel(), K)
    if not x2.is_contiguous():
        x2 = x2.contiguous()
    return x2, gate, up, down, K, Iw, H


@functools.lru_cache(maxsize=1024)
def _mlp_work(M, K, I, H, backward, f32=False):
    lib = _lib.load()
    return (lib.mj_gated_mlp_f32_work_bytes if f32 else lib.mj_gated_mlp_work_bytes)(M, K, I, H, backward)


def _padded(mats, at):
    """Where the kernels read matrices (pointer, rows, cols, padded rows, padded cols):
    in place, or from ``at`` on for those whose widths or addresses they cannot take;
    and the copies that brings about, and their bytes."""
    ptrs, copies, used = [], [], 0
    for p, r, c, rp, cp in mats:
        if (r, c) == (rp, cp) and p % 16 == 0:
            ptrs.append(p)
        else:
            ptrs.append(at + used)
            copies.append((p, at + used, r, c, c, rp, cp, cp))
            used += _up16(2 * rp * cp)
    return tuple(ptrs), copies, used


def _gated_mlp(x, gate, up, down, act, train):
    x2, gate, up, down, K, I, H = _mlp_operands(x, gate, up, down)
    M, dev = x2.shape[0], x2.device
    y = x2.new_empty((M, H))
    ptrs = (x2.data_ptr(), gate.data_ptr(), up.data_ptr(), down.data_ptr())
    # one buffer: g, u [M, I] fp32 (kept for the backward; the fp32 form always writes
    # them), h, then in bf16 padded operands, a padded y and the workspace
    if x2.dtype == torch.float32:
        gu = _up16(4 * M * I)
        nbytes = _mlp_work(M, K, I, H, 0, True)
        buf = _scratch(3 * gu + (0 if train else nbytes), dev)
        more = _scratch(nbytes, dev) if train and nbytes else None
        g = buf.data_ptr()
        work = None if not nbytes else g + 3 * gu if more is None else more.data_ptr()
        _lib.call("mj_gated_mlp_f32", *ptrs, act, g + 2 * gu, g, g + gu, y.data_ptr(), M, K, I, H,
                  work, nbytes, _stream())
    else:
        Kp, Ip, Hp = K + 7 & ~7, I + 7 & ~7, H + 7 & ~7
        gu = _up16(4 * M * Ip) if train else 0
        hb = _up16(2 * M * Ip)
        mats = ((ptrs[0], M, K, M, Kp), (ptrs[1], I, K, Ip, Kp), (ptrs[2], I, K, Ip, Kp),
                (ptrs[3], H, I, Hp, Ip))
        pad = 0
        if Kp != K or Ip != I or Hp != H or any(p % 16 for p in ptrs):
            pad = _padded(mats, 0)[2]
        yb = 0 if Hp == H else _up16(2 * M * Hp)
        nbytes = _mlp_work(M, Kp, Ip, Hp, 0)
        # a training step keeps the buffer: what only this call needs goes into another
        buf = _scratch(2 * gu + hb + pad + (0 if train else yb + nbytes), dev)
        more = _scratch(yb + nbytes, dev) if train and yb + nbytes else None
        g = buf.data_ptr()
        h = g + 2 * gu
        if pad:
            ptrs, copies, _ = _padded(mats, h + hb)
            _copy_rows(copies)
        end = h + hb + pad if more is None else more.data_ptr()
        _lib.call("mj_gated_mlp_bf16", *ptrs, act, h, g if train else None,
                  g + gu if train else None, end if yb else y.data_ptr(), M, Kp, Ip, Hp,
                  end + yb if nbytes else None, nbytes, _stream())
        if yb:
            _copy_rows([(end, y.data_ptr(), M, H, Hp, M, H, H)])
    if x.dim() != 2:
        y = y.reshape(*x.shape[:-1], H)
    if not train:
        return y, None
    return y, GatedMLPSaved(x2, gate, up, down, buf, ptrs, act, x.shape[:-1])


def gated_mlp(x: torch.Tensor, gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor,
              act: int = _lib.EPI_SILU) -> torch.Tensor:
    """y = (act(x gate^T) * (x up^T)) down^T for x [..., K], gate and up [I, K],
    down [H, I], all bfloat16 or all Float32; act is EPI_NONE, EPI_RELU,
    EPI_GELU_TANH or EPI_SILU.  bfloat16 widths that are not multiples of 8 cost
    zero-padded copies of the operands."""
    return _gated_mlp(x, gate, up, down, act, False)[0]


def gated_mlp_train(x: torch.Tensor, gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor,
                    act: int = _lib.EPI_SILU):
    """(y, saved): gated_mlp and what its backward needs (h in x's type and the two
    projections in Float32).  The operands are kept, not copied: they must not
    change before the backward."""
    return _gated_mlp(x, gate, up, down, act, True)


def gated_mlp_backward(dy: torch.Tensor, saved: GatedMLPSaved):
    """(dx, dgate, dup, ddown) of gated_mlp from the gradient of y."""
    s = saved
    x, (M, K), (H, I) = s.x, s.x.shape, s.down.shape
    dy = _like(dy, x, s.rows + (H,), "dy")
    f32 = x.dtype == torch.float32
    dx, ddown = x.new_empty((M, K)), x.new_empty((H, I))
    # (fp32: side by side, for one launch)
    dgate, dup = x.new_empty((2, I, K)).unbind() if f32 else (x.new_empty((I, K)), x.new_empty((I, K)))
    out = dx, dgate, dup, ddown
    outs = tuple(t.data_ptr() for t in out)
    g = s.buf.data_ptr()
    if f32:
        gu = _up16(4 * M * I)
        nbytes = _mlp_work(M, K, I, H, 1, True)
        buf = _scratch(2 * gu + nbytes, x.device)  # dg, du, the workspace
        dg = buf.data_ptr()
        _lib.call("mj_gated_mlp_backward_f32", *s.ptrs, s.act, g + 2 * gu, g, g + gu, dy.data_ptr(),
                  dg, dg + gu, *outs, M, K, I, H, dg + 2 * gu if nbytes else None, nbytes, _stream())
    else:
        Kp, Ip, Hp = K + 7 & ~7, I + 7 & ~7, H + 7 & ~7
        gu, db = _up16(4 * M * Ip), _up16(2 * M * Ip)
        nbytes = _mlp_work(M, Kp, Ip, Hp, 1)
        mats = ((dy.data_ptr(), M, H, M, Hp),)
        pad = _padded(mats, 0)[2]
        grads = ((outs[0], M, K, M, Kp), (outs[1], I, K, Ip, Kp), (outs[2], I, K, Ip, Kp),
                 (outs[3], H, I, Hp, Ip))
        cut = (Kp, Ip, Hp) != (K, I, H)
        cutb = _padded(grads, 0)[2] if cut else 0
        buf = _scratch(2 * db + nbytes + pad + cutb, x.device)  # dg, du, the workspace, ..
        dg = buf.data_ptr()
        at = dg + 2 * db
        end = at + _up16(nbytes)
        (dyp,), copies, _ = _padded(mats, end)
        if copies:
            _copy_rows(copies)
        if cut:
            outs, back, _ = _padded(grads, end + pad)
        _lib.call("mj_gated_mlp_backward_bf16", *s.ptrs, s.act, g + 2 * gu, g, g + gu, dyp, dg,
                  dg + db, *outs, M, Kp, Ip, Hp, at if nbytes else None, nbytes, _stream())
        if cut:
            _copy_rows([(q, p, r, c, cp, r, c, c) for p, q, r, c, _, rp, cp, _ in back])
    if len(s.rows) != 1:
        dx = dx.reshape(*s.rows, K)
    return dx, dgate, dup, ddown


class GatedMLP:
    """GatedMLP(gate, up, down, act): gated_mlp with its weights."""

    def __init__(self, gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor,
                 act: int = _lib.EPI_SILU):
        if gate.dim() != 2 or up.shape != gate.shape or down.dim() != 2 or \
                down.shape[1] != gate.shape[0]:
            raise ValueError(f"gate {list(gate.shape)}, up {list(up.shape)} and down "
                             f"{list(down.shape)} do not fit each other")
        self.gate, self.up, self.down, self.act = gate, up, down, act

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return gated_mlp(x, self.gate, self.up, self.down, self.act)

    def forward_train(self, x: torch.Tensor):
        return gated_mlp_train(x, self.gate, self.up, self.down, self.act)

    backward = staticmethod(gated_mlp_backward)


__all__ = ["dropout", "dropout_backward", "Dropout", "residual_norm", "residual_norm_train",
           "residual_norm_backward", "ResidualNorm", "ResidualNormSaved", "gated_mlp",
           "gated_mlp_train", "gated_mlp_backward", "GatedMLP", "GatedMLPSaved"]
