"""Mixture of experts: tokens sorted by expert and back, and the experts' gated
feed-forward blocks over the sorted rows, forward and backward.

``sort_experts`` plans where each slot (token t, its j-th expert) goes;
``dispatch`` copies the tokens' rows there, ``combine`` sums the experts' rows
back with the tokens' weights, and each has its ``_backward``.  ``experts_mlp``
is ``gated_mlp`` of every row's own expert, and ``ExpertsMLP`` the layer from
tokens to tokens.  A slot whose expert is outside 0 .. E - 1 is dropped: it adds
nothing to its token.  How many rows an expert has stays on the device: no call
waits for it, and all can be captured into a HIP graph.

Tensors are on the current device; operands of other strides are copied to
contiguous ones first.  The kernels run on the current stream and allocate
through torch only.
"""
from __future__ import annotations

import functools
import operator
from typing import NamedTuple

import torch

from . import _lib
from .block import _DTYPES, _check_type, _like, _scratch, _up16
from .tensor import _ptr


# (A small call's time is the host's, so checks ask for numbers, not for torch.device objects:
# 0.3 us less a check, of 7 for a dispatch.)
def _check_device(t: torch.Tensor, name: str) -> None:
    index = t.get_device()
    if index < 0:
        raise ValueError(f"{name} must be on the GPU")
    if index != torch._C._cuda_getDevice():
        raise ValueError(f"{name} is on {t.device}, the current device is "
                         f"cuda:{torch._C._cuda_getDevice()}")


def _stream(t: torch.Tensor) -> int:
    """The current stream of the device of t, which _check_device has found to be the current
    one."""
    return torch._C._cuda_getCurrentRawStream(t.get_device())


class ExpertPlan:
    """Where the slots go, as ``sort_experts`` finds it.  pos int32 [tokens, topk]: a slot's row
    among those sorted by expert (in the order of the slots within an expert, dropped slots
    last); offsets int32 [experts + 1]: the experts' first rows, the last entry the first
    dropped slot's.  A plan of other entries gives meaningless rows, but no access outside the
    tensors.  A plan's tensors and sizes belong together and cannot be replaced."""

    __slots__ = ("_pos", "_offsets", "_tokens", "_topk", "_rows", "_experts", "_index")
    pos, offsets, tokens, topk, rows, experts, device = (
        property(operator.attrgetter(name))
        for name in ("_pos", "_offsets", "_tokens", "_topk", "_rows", "_experts", "_pos.device"))

    def __init__(self, pos: torch.Tensor, offsets: torch.Tensor):
        if pos.dim() != 2 or pos.dtype is not torch.int32 or not pos.is_contiguous() or \
                offsets.dim() != 1 or offsets.dtype is not torch.int32 or \
                not offsets.is_contiguous() or offsets.device != pos.device or not len(offsets):
            raise ValueError("pos must be a contiguous int32 [tokens, topk] tensor, offsets int32 "
                             "[experts + 1] on its device")
        self._set(pos, offsets, *pos.shape, offsets.shape[0] - 1, pos.get_device())

    def _set(self, pos, offsets, tokens, topk, experts, index):
        self._pos, self._offsets, self._experts, self._index = pos, offsets, experts, index
        self._tokens, self._topk, self._rows = tokens, topk, tokens * topk
        return self

    def __reduce__(self):
        return ExpertPlan, (self._pos, self._offsets)

    @property
    def _args(self):
        """The plan's part of a library call's arguments, with the addresses of now."""
        return self._pos.data_ptr(), self._offsets.data_ptr(), self._experts


def _contiguous(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous() else t.contiguous()


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """t as a contiguous tensor at a multiple of 16 bytes, as the tile kernels read it."""
    t = _contiguous(t)
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _rows_of(t: torch.Tensor, plan: ExpertPlan, rows: int, name: str):
    """(type code, t contiguous, its width) of a [rows, dim] operand on the plan's device."""
    code, index = _DTYPES.get(t.dtype), t.get_device()
    if code is None or t.dim() != 2 or index != plan._index:
        _check_type(t, name)
        _check_device(t, name)
        raise ValueError(f"{name} must be [{rows}, dim] on {plan.device}, got {list(t.shape)} on {t.device}")
    if index < 0 or index != torch._C._cuda_getDevice():
        _check_device(t, name)
    n, dim = t.shape
    if n != rows:
        raise ValueError(f"{name} must be [{rows}, dim], got {list(t.shape)}")
    return code, t if t.is_contiguous() else t.contiguous(), dim


def _weights(w: torch.Tensor, plan: ExpertPlan, name: str) -> torch.Tensor:
    if w.dtype is not torch.float32 or w.shape != plan._pos.shape or w.get_device() != plan._index:
        raise ValueError(f"{name} must be float32 {list(plan._pos.shape)} on {plan.device}, got "
                         f"{w.dtype} {list(w.shape)} on {w.device}")
    return w if w.is_contiguous() else w.contiguous()


@functools.lru_cache(maxsize=1024)
def _sort_work(slots, experts):
    return _lib.load().mj_sort_experts_work_bytes(slots, experts)


def sort_experts(experts: torch.Tensor, num_experts: int) -> ExpertPlan:
    """The plan for tokens whose experts are ``experts`` [tokens, topk], int32 or int64;
    an entry outside 0 .. num_experts - 1 is a dropped slot."""
    size = 8 if experts.dtype is torch.int64 else 4
    if size == 4 and experts.dtype is not torch.int32:
        raise TypeError(f"experts must be int32 or int64, got {experts.dtype}")
    if experts.dim() != 2:
        raise ValueError(f"experts must be [tokens, topk], got {list(experts.shape)}")
    _check_device(experts, "experts")
    ids = _contiguous(experts)
    T, k = ids.shape
    nbytes = _sort_work(T * k, num_experts)
    pos = ids.new_empty((T, k), dtype=torch.int32)
    offsets = ids.new_empty(max(num_experts, 0) + 1, dtype=torch.int32)
    work = _scratch(nbytes, ids.device) if nbytes else None
    index = ids.get_device()
    _lib.call("mj_sort_experts", ids.data_ptr(), size, T * k, num_experts, pos.data_ptr(),
              offsets.data_ptr(), _ptr(work), nbytes, torch._C._cuda_getCurrentRawStream(index))
    return object.__new__(ExpertPlan)._set(pos, offsets, T, k, num_experts, index)


def dispatch(x: torch.Tensor, plan: ExpertPlan, weights: torch.Tensor | None = None):
    """xs [tokens * topk, dim] with xs[pos[t, j]] = x[t], zeros for dropped slots; with
    ``weights`` [tokens, topk] (Float32) also their sorted form: (xs, ws)."""
    code, x, dim = _rows_of(x, plan, plan._tokens, "x")
    xs = x.new_empty((plan._rows, dim))
    if weights is None:
        _lib.call("mj_dispatch", code, x.data_ptr(), None, *plan._args, xs.data_ptr(), None,
                  plan._tokens, plan._topk, dim, _stream(xs))
        return xs
    weights = _weights(weights, plan, "weights")
    ws = weights.new_empty(plan._rows)
    _lib.call("mj_dispatch", code, x.data_ptr(), weights.data_ptr(), *plan._args, xs.data_ptr(),
              ws.data_ptr(), plan._tokens, plan._topk, dim, _stream(xs))
    return xs, ws


def combine(ys: torch.Tensor, weights: torch.Tensor | None, plan: ExpertPlan,
            dtype: torch.dtype | None = None) -> torch.Tensor:
    """y[t] = the sum over j of weights[t, j] ys[pos[t, j]], in Float32 and rounded once to
    ``dtype`` (ys's by default; Float32 rows can give bfloat16); weights None: ones.  Dropped
    slots are left out, whatever they hold."""
    code, ys, dim = _rows_of(ys, plan, plan._rows, "ys")
    if weights is not None:
        weights = _weights(weights, plan, "weights")
    if dtype is None or dtype is ys.dtype:
        to, y = code, ys.new_empty((plan._tokens, dim))
    elif ys.dtype is torch.float32 and dtype is torch.bfloat16:
        to, y = _lib.BF16, ys.new_empty((plan._tokens, dim), dtype=dtype)
    else:
        raise TypeError(f"{ys.dtype} rows cannot be combined to {dtype}")
    _lib.call("mj_combine", code, to, ys.data_ptr(), _ptr(weights), *plan._args, y.data_ptr(),
              plan._tokens, plan._topk, dim, _stream(ys))
    return y


def dispatch_backward(dxs: torch.Tensor, plan: ExpertPlan,
                      dtype: torch.dtype | None = None) -> torch.Tensor:
    """The gradient of ``dispatch``'s x: dx[t] = the sum over j of dxs[pos[t, j]], rounded as
    ``combine``'s."""
    return combine(dxs, None, plan, dtype)


def combine_backward(dy: torch.Tensor, ys: torch.Tensor, weights: torch.Tensor, plan: ExpertPlan):
    """(dys, dweights) of ``combine``: dys[pos[t, j]] = weights[t, j] dy[t] and dweights[t, j]
    = <dy[t], ys[pos[t, j]]>, both 0 for dropped slots.  dy is of ys's type, and so is dys."""
    code, dy, dim = _rows_of(dy, plan, plan._tokens, "dy")
    ys = _like(ys, dy, (plan._rows, dim), "ys")
    weights = _weights(weights, plan, "weights")
    dys, dw = torch.empty_like(ys), torch.empty_like(weights)
    _lib.call("mj_combine_backward", code, dy.data_ptr(), ys.data_ptr(), weights.data_ptr(),
              *plan._args, dys.data_ptr(), dw.data_ptr(), plan._tokens, plan._topk, dim, _stream(ys))
    return dys, dw


# ------------------------------------------------------------------ the experts' block
class ExpertsSaved(NamedTuple):
    """What experts_mlp_backward needs: the operands, and one buffer with the fp32
    projections g and u, then h."""
    xs: torch.Tensor
    plan: ExpertPlan
    weights: torch.Tensor | None  # sorted, [rows]
    gate: torch.Tensor
    up: torch.Tensor
    down: torch.Tensor
    buf: torch.Tensor
    act: int


def _matrices(xs, plan, gate, up, down):
    E = plan._experts
    if xs.dtype is not torch.bfloat16:
        raise TypeError(f"the experts' block takes bfloat16 rows, got {xs.dtype}")
    if gate.dim() != 3 or down.dim() != 3 or gate.shape[0] != E or down.shape[0] != E or \
            gate.shape[2] != xs.shape[1] or down.shape[2] != gate.shape[1]:
        raise ValueError(f"gate {list(gate.shape)} and down {list(down.shape)} do not fit rows of "
                         f"{xs.shape[1]} features and {E} experts")
    return [_aligned(_like(t, xs, shape, name)) for t, shape, name in
            ((gate, gate.shape, "gate"), (up, gate.shape, "up"), (down, down.shape, "down"))]


def _experts_mlp(xs, plan, gate, up, down, act, weights, train):
    xs = _aligned(_rows_of(xs, plan, plan._rows, "xs")[1])
    gate, up, down = _matrices(xs, plan, gate, up, down)
    if weights is not None:
        if weights.dtype is not torch.float32 or weights.shape != (plan._rows,) or \
                weights.device != xs.device:
            raise ValueError(f"weights must be float32 [{plan._rows}] on {xs.device}")
        weights = _contiguous(weights)
    R, K = xs.shape
    I, H = gate.shape[1], down.shape[1]
    ys = torch.empty((R, H), dtype=torch.float32, device=xs.device)
    gu = _up16(4 * R * I) if train else 0
    buf = _scratch(2 * gu + _up16(2 * R * I), xs.device)
    g = buf.data_ptr()
    _lib.call("mj_experts_mlp_bf16", xs.data_ptr(), plan._offsets.data_ptr(), plan._experts,
              gate.data_ptr(), up.data_ptr(), down.data_ptr(), act, _ptr(weights), g + 2 * gu,
              g if train else None, g + gu if train else None, ys.data_ptr(), R, K, I, H, _stream(xs))
    return ys, ExpertsSaved(xs, plan, weights, gate, up, down, buf, act) if train else None


def experts_mlp(xs: torch.Tensor, plan: ExpertPlan, gate: torch.Tensor, up: torch.Tensor,
                down: torch.Tensor, act: int = _lib.EPI_SILU,
                weights: torch.Tensor | None = None) -> torch.Tensor:
    """ys [rows, H] in Float32: ``gated_mlp`` of each sorted row with its expert's matrices,
    gate and up [E, I, K], down [E, H, I], all bfloat16 with widths in multiples of 8.
    ``weights`` [rows] (sorted, as ``dispatch`` gives them) multiply h, and so ys.  Rows of
    dropped slots are zeros."""
    return _experts_mlp(xs, plan, gate, up, down, act, weights, False)[0]


def experts_mlp_train(xs: torch.Tensor, plan: ExpertPlan, gate: torch.Tensor, up: torch.Tensor,
                      down: torch.Tensor, act: int = _lib.EPI_SILU,
                      weights: torch.Tensor | None = None):
    """(ys, saved): experts_mlp and what its backward needs (h in bfloat16, the two
    projections in Float32).  The operands are kept, not copied: they must not change before
    the backward."""
    return _experts_mlp(xs, plan, gate, up, down, act, weights, True)


def experts_mlp_backward(dys: torch.Tensor, saved: ExpertsSaved):
    """(dxs, dgate, dup, ddown, dweights) of experts_mlp from dys, bfloat16; dxs and dweights
    are Float32.  An expert without rows gets zeros, and so do dxs's rows of dropped slots;
    dweights [tokens, topk] is the gradient of the unsorted weights, or None without weights.
    dys's rows of dropped slots are not read."""
    s = saved
    xs, plan, dev = s.xs, s.plan, s.xs.device
    _check_device(xs, "xs")
    (R, K), (E, I, _), H = xs.shape, s.gate.shape, s.down.shape[1]
    dys = _aligned(_like(dys, xs, (R, H), "dys"))
    out = [torch.empty(xs.shape, dtype=torch.float32, device=dev)]
    out += [torch.empty_like(t) for t in (s.gate, s.up, s.down)]
    dw, dots = None, 0
    if s.weights is not None:
        dw = torch.empty(plan._pos.shape, dtype=torch.float32, device=dev)
        dots = 4 * _lib.load().mj_experts_mlp_dots(R, E, K, I, H)
    gu, db = _up16(4 * R * I), _up16(2 * R * I)
    work = _scratch(2 * db + dots, dev)  # dg, du, the parts of dweights
    g, dg = s.buf.data_ptr(), work.data_ptr()
    _lib.call("mj_experts_mlp_backward_bf16", xs.data_ptr(), plan._offsets.data_ptr(), E,
              s.gate.data_ptr(), s.up.data_ptr(), s.down.data_ptr(), s.act, _ptr(s.weights),
              g + 2 * gu, g, g + gu, dys.data_ptr(), dg, dg + db, *[t.data_ptr() for t in out],
              plan._pos.data_ptr(), R if dw is not None else 0, dg + 2 * db if dots else None,
              _ptr(dw), R, K, I, H, _stream(xs))
    return (*out, dw)


class ExpertsMLP:
    """ExpertsMLP(gate, up, down, act): the layer of E gated blocks, gate and up [E, I, K],
    down [E, H, I], bfloat16:

        y[t] = the sum over j of weights[t, j] mlp_e(x[t]) for e = experts[t, j]

    experts [tokens, topk] are int32 or int64 (outside 0 .. E - 1: dropped), weights Float32 of
    the same shape, x [tokens, K]."""

    def __init__(self, gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor,
                 act: int = _lib.EPI_SILU):
        if gate.dim() != 3 or up.shape != gate.shape or down.dim() != 3 or \
                down.shape[0] != gate.shape[0] or down.shape[2] != gate.shape[1]:
            raise ValueError(f"gate {list(gate.shape)}, up {list(up.shape)} and down "
                             f"{list(down.shape)} do not fit each other")
        self.gate, self.up, self.down, self.act = gate, up, down, act

    def _sorted(self, x, experts, weights):
        plan = sort_experts(experts, self.gate.shape[0])
        return plan, *dispatch(x, plan, weights)

    def forward(self, x: torch.Tensor, experts: torch.Tensor, weights: torch.Tensor) -> torch.Tensor:
        plan, xs, ws = self._sorted(x, experts, weights)
        ys = experts_mlp(xs, plan, self.gate, self.up, self.down, self.act, ws)
        return combine(ys, None, plan, x.dtype)

    def forward_train(self, x: torch.Tensor, experts: torch.Tensor, weights: torch.Tensor):
        """(y, saved)"""
        plan, xs, ws = self._sorted(x, experts, weights)
        ys, saved = experts_mlp_train(xs, plan, self.gate, self.up, self.down, self.act, ws)
        return combine(ys, None, plan, x.dtype), saved

    @staticmethod
    def backward(dy: torch.Tensor, saved: ExpertsSaved) -> dict[str, torch.Tensor]:
        """The gradients of x, weights, gate, up and down, by their names."""
        dys = dispatch(dy, saved.plan)
        dxs, dgate, dup, ddown, dw = experts_mlp_backward(dys, saved)
        return dict(x=dispatch_backward(dxs, saved.plan, dy.dtype), weights=dw, gate=dgate, up=dup, down=ddown)


__all__ = ["ExpertPlan", "sort_experts", "dispatch", "dispatch_backward", "combine",
           "combine_backward", "experts_mlp", "experts_mlp_train", "experts_mlp_backward",
           "ExpertsMLP", "ExpertsSaved"]
