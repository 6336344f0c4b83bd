"""Inference in 8-bit floating point with block scales: a Linear and a mixture of
experts whose weights are e4m3 with a scale for each 128 x 128 block and whose
activations are quantized at call time, a scale for each 128 features of a row.

A block of largest magnitude m is quantized with a = max(m, 2^-100): scale
a * (1 / 448), values e4m3(v * (448 * (1 / a))) to the nearest even, each operation
rounded to Float32.  Products of a block
are summed on the matrix cores, multiplied by the product of their two scales and added
up in Float32; blocks whose largest magnitudes multiply to less than 2^-108 or to 2^145
and more leave Float32's range there.

Values are torch.float8_e4m3fn.  Scales of rows lie block by block, Float32
[ceil(K / 128), rows]; those of a matrix are [ceil(N / 128), ceil(K / 128)].  K is a
multiple of 16; N is any (for the experts' gate and up a multiple of 16).
"""
from __future__ import annotations

import functools

import torch

from . import _lib
from .block import _check_type, _scratch
from .experts import (ExpertPlan, _aligned, _check_device, _contiguous, _rows_of, _stream, combine,
                      sort_experts)
from .tensor import _ptr

_F8 = torch.float8_e4m3fn


def _blocks(k: int) -> int:
    return (k + 127) // 128


def quantize_rows_fp8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(q [rows, K], scales [ceil(K / 128), rows]) of x [rows, K], bfloat16 or Float32."""
    code = _check_type(x, "x")
    _check_device(x, "x")
    if x.dim() != 2:
        raise ValueError(f"x must be [rows, K], got {list(x.shape)}")
    x = _aligned(x)
    M, K = x.shape
    q = torch.empty((M, K), dtype=_F8, device=x.device)
    scales = torch.empty((_blocks(K), M), dtype=torch.float32, device=x.device)
    _lib.call("mj_quantize_rows_f8", code, x.data_ptr(), q.data_ptr(), scales.data_ptr(), M, K,
              _stream(x))
    return q, scales


def quantize_blocks_fp8(W: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(q, scales) of a matrix W [N, K] or of matrices [E, N, K], bfloat16 or Float32:
    q of W's shape, scales [.., ceil(N / 128), ceil(K / 128)]."""
    code = _check_type(W, "W")
    _check_device(W, "W")
    if W.dim() not in (2, 3):
        raise ValueError(f"W must be [N, K] or [E, N, K], got {list(W.shape)}")
    W = _aligned(W)
    mats, (N, K) = W.shape[0] if W.dim() == 3 else 1, W.shape[-2:]
    q = torch.empty(W.shape, dtype=_F8, device=W.device)
    scales = torch.empty((*W.shape[:-2], _blocks(N), _blocks(K)), dtype=torch.float32, device=W.device)
    _lib.call("mj_quantize_blocks_f8", code, W.data_ptr(), q.data_ptr(), scales.data_ptr(), mats, N, K,
              _stream(W))
    return q, scales


def _matrix(q, scales, dims, name):
    """A quantized matrix (dims 2) or the experts' (3), checked and contiguous."""
    if q.dtype is not _F8 or q.dim() != dims:
        raise ValueError(f"{name} must be a {dims}-D float8_e4m3fn tensor, got {q.dtype} {list(q.shape)}")
    want = (*q.shape[:-2], _blocks(q.shape[-2]), _blocks(q.shape[-1]))
    if scales.dtype is not torch.float32 or scales.shape != want or scales.device != q.device:
        raise ValueError(f"{name}'s scales must be float32 {list(want)} on {q.device}, got "
                         f"{scales.dtype} {list(scales.shape)} on {scales.device}")
    return _aligned(q), _contiguous(scales)


def _rows(q, scales, K, name):
    if q.dtype is not _F8 or q.dim() != 2 or q.shape[1] != K:
        raise ValueError(f"{name} must be float8_e4m3fn [rows, {K}], got {q.dtype} {list(q.shape)}")
    want = (_blocks(K), q.shape[0])
    if scales.dtype is not torch.float32 or scales.shape != want or scales.device != q.device:
        raise ValueError(f"{name}'s scales must be float32 {list(want)} on {q.device}, got "
                         f"{scales.dtype} {list(scales.shape)} on {scales.device}")
    _check_device(q, name)
    return _aligned(q), _contiguous(scales)


@functools.lru_cache(maxsize=1024)
def _work(name, *sizes):
    return getattr(_lib.load(), name)(*sizes)


def _bias(bias, N, device):
    if bias is None:
        return None
    if bias.numel() != N or bias.device != device:
        raise ValueError(f"bias must have {N} elements on {device}")
    return _contiguous(bias.float().reshape(-1))


def gemm_fp8_nt(q: torch.Tensor, scales: torch.Tensor, Wq: torch.Tensor, Wscales: torch.Tensor,
                bias: torch.Tensor | None = None, act: int = _lib.EPI_NONE) -> torch.Tensor:
    """y = act(x W^T + bias) in bfloat16 from quantized rows and a quantized matrix; act is
    EPI_NONE, EPI_RELU, EPI_GELU_TANH or EPI_SILU."""
    Wq, Wscales = _matrix(Wq, Wscales, 2, "W")
    N, K = Wq.shape
    q, scales = _rows(q, scales, K, "x")
    if Wq.device != q.device:
        raise ValueError(f"W is on {Wq.device}, x on {q.device}")
    bias = _bias(bias, N, q.device)
    M = q.shape[0]
    y = torch.empty((M, N), dtype=torch.bfloat16, device=q.device)
    nbytes = _work("mj_gemm_f8_work_bytes", M, N, K)
    work = _scratch(nbytes, q.device) if nbytes else None
    _lib.call("mj_gemm_f8", q.data_ptr(), scales.data_ptr(), Wq.data_ptr(), Wscales.data_ptr(),
              _ptr(bias), act, y.data_ptr(), M, N, K, _ptr(work), nbytes, _stream(q))
    return y


class F8Linear:
    """F8Linear(q, scales, bias, act): y = act(x W^T + bias) in bfloat16 for x [..., K],
    bfloat16 or Float32, quantized in the call; q [N, K] float8_e4m3fn with its block scales.
    q, scales and bias can be replaced by others of their shapes on the same device."""

    def __init__(self, q: torch.Tensor, scales: torch.Tensor, bias: torch.Tensor | None = None,
                 act: int = _lib.EPI_NONE):
        self.q, self.scales = _matrix(q, scales, 2, "q")
        self.out_features, self.in_features = self.q.shape
        self.bias = _bias(bias, self.out_features, self.q.device)
        self.act = act

    def __setattr__(self, name, value):
        held = self.__dict__
        if name in held:  # (a forward goes by the constructor's checks and sizes)
            if name in ("in_features", "out_features"):
                raise AttributeError(f"{name} is q's")
            if name in ("q", "scales") and value.shape != held[name].shape:
                raise ValueError(f"{name} must be {list(held[name].shape)}, got {list(value.shape)}")
            if name == "q":
                value, _ = _matrix(value, self.scales, 2, name)
            elif name == "scales":
                _, value = _matrix(self.q, value, 2, "q")
            elif name == "bias":
                value = _bias(value, self.out_features, self.q.device)
        held[name] = value

    @classmethod
    def from_float(cls, W: torch.Tensor, bias: torch.Tensor | None = None,
                   act: int = _lib.EPI_NONE) -> "F8Linear":
        return cls(*quantize_blocks_fp8(W), bias, act)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        code = _check_type(x, "x")
        _check_device(x, "x")
        K, N, shape = self.in_features, self.out_features, x.shape
        if not shape or shape[-1] != K or x.device != self.q.device:
            raise ValueError(f"x must be [..., {K}] on {self.q.device}, got {list(shape)} on {x.device}")
        x = _aligned(x)
        M = shape[0] if len(shape) == 2 else shape[:-1].numel()
        y = x.new_empty((*shape[:-1], N), dtype=torch.bfloat16)
        nbytes = _work("mj_linear_f8_work_bytes", M, N, K)
        work = _scratch(nbytes, x.device) if nbytes else None
        _lib.call("mj_linear_f8", code, x.data_ptr(), self.q.data_ptr(), self.scales.data_ptr(),
                  _ptr(self.bias), self.act, y.data_ptr(), M, N, K, _ptr(work), nbytes, _stream(x))
        return y


# ------------------------------------------------------------------ experts
def dispatch_fp8(x: torch.Tensor, plan: ExpertPlan) -> tuple[torch.Tensor, torch.Tensor]:
    """(q [rows, K], scales [ceil(K / 128), rows]): each token's row quantized once and copied
    to its slots' sorted rows; zeros for dropped slots."""
    code, x, K = _rows_of(x, plan, plan._tokens, "x")
    x = _aligned(x)
    q = torch.empty((plan._rows, K), dtype=_F8, device=x.device)
    scales = torch.empty((_blocks(K), plan._rows), dtype=torch.float32, device=x.device)
    _lib.call("mj_dispatch_f8", code, x.data_ptr(), *plan._args, q.data_ptr(), scales.data_ptr(),
              plan._tokens, plan._topk, K, _stream(x))
    return q, scales


def _expert_operands(q, scales, plan, Wq, Wscales, name):
    Wq, Wscales = _matrix(Wq, Wscales, 3, name)
    q, scales = _rows(q, scales, Wq.shape[2], "x")
    if q.get_device() != plan._index or q.shape[0] != plan._rows or Wq.shape[0] != plan._experts or Wq.device != q.device:
        raise ValueError(f"{plan._rows} rows and {plan._experts} experts planned, got {q.shape[0]} rows "
                         f"and {Wq.shape[0]} matrices on {Wq.device}")
    return q, scales, Wq, Wscales


def experts_gemm_fp8(q: torch.Tensor, scales: torch.Tensor, plan: ExpertPlan, Wq: torch.Tensor,
                     Wscales: torch.Tensor) -> torch.Tensor:
    """y [rows, N] in Float32: each sorted row times its expert's matrix of Wq [E, N, K];
    zeros for dropped slots."""
    q, scales, Wq, Wscales = _expert_operands(q, scales, plan, Wq, Wscales, "W")
    (R, K), (E, N, _) = q.shape, Wq.shape
    y = torch.empty((R, N), dtype=torch.float32, device=q.device)
    _lib.call("mj_experts_gemm_f8", q.data_ptr(), scales.data_ptr(), plan._offsets.data_ptr(), E,
              Wq.data_ptr(), Wscales.data_ptr(), y.data_ptr(), R, N, K, _stream(q))
    return y


def experts_gate_fp8(q: torch.Tensor, scales: torch.Tensor, plan: ExpertPlan, gate: torch.Tensor,
                     gate_scales: torch.Tensor, up: torch.Tensor, up_scales: torch.Tensor,
                     act: int = _lib.EPI_SILU) -> tuple[torch.Tensor, torch.Tensor]:
    """(hq [rows, I], scales): h = act(x gate^T) (x up^T) of each sorted row with its expert's
    matrices, quantized from Float32 as the next product's rows."""
    q, scales, gate, gate_scales = _expert_operands(q, scales, plan, gate, gate_scales, "gate")
    up, up_scales = _matrix(up, up_scales, 3, "up")
    if up.shape != gate.shape or up.device != gate.device:
        raise ValueError(f"gate is {list(gate.shape)} on {gate.device}, up {list(up.shape)} on {up.device}")
    (R, K), (E, I, _) = q.shape, gate.shape
    hq = torch.empty((R, I), dtype=_F8, device=q.device)
    hs = torch.empty((_blocks(I), R), dtype=torch.float32, device=q.device)
    nbytes = _work("mj_experts_gate_f8_work_bytes", R, E, I, K)
    work = _scratch(nbytes, q.device) if nbytes else None
    _lib.call("mj_experts_gate_f8", q.data_ptr(), scales.data_ptr(), plan._offsets.data_ptr(), E,
              gate.data_ptr(), gate_scales.data_ptr(), up.data_ptr(), up_scales.data_ptr(), act,
              hq.data_ptr(), hs.data_ptr(), R, I, K, _ptr(work), nbytes, _stream(q))
    return hq, hs


class F8Experts:
    """F8Experts(gate, gate_scales, up, up_scales, down, down_scales, act): ``ExpertsMLP`` for
    inference on 8-bit weights, gate and up [E, I, K], down [E, H, I] with their block
    scales.  x and the hidden features are quantized in the call."""

    def __init__(self, gate: torch.Tensor, gate_scales: torch.Tensor, up: torch.Tensor,
                 up_scales: torch.Tensor, down: torch.Tensor, down_scales: torch.Tensor,
                 act: int = _lib.EPI_SILU):
        self.gate, self.gate_scales = _matrix(gate, gate_scales, 3, "gate")
        self.up, self.up_scales = _matrix(up, up_scales, 3, "up")
        self.down, self.down_scales = _matrix(down, down_scales, 3, "down")
        if self.up.shape != self.gate.shape or self.down.shape[0] != self.gate.shape[0] or \
                self.down.shape[2] != self.gate.shape[1]:
            raise ValueError(f"gate {list(gate.shape)}, up {list(up.shape)} and down "
                             f"{list(down.shape)} do not fit each other")
        self.act = act

    @classmethod
    def from_float(cls, gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor,
                   act: int = _lib.EPI_SILU) -> "F8Experts":
        return cls(*quantize_blocks_fp8(gate), *quantize_blocks_fp8(up), *quantize_blocks_fp8(down), act)

    def forward(self, x: torch.Tensor, experts: torch.Tensor, weights: torch.Tensor) -> torch.Tensor:
        """y[t] = the sum over j of weights[t, j] mlp_e(x[t]) for e = experts[t, j], in
        bfloat16; x [tokens, K] bfloat16 or Float32, experts and weights as ``ExpertsMLP``'s."""
        plan = sort_experts(experts, self.gate.shape[0])
        q, s = dispatch_fp8(x, plan)
        hq, hs = experts_gate_fp8(q, s, plan, self.gate, self.gate_scales, self.up, self.up_scales,
                                  self.act)
        return combine(experts_gemm_fp8(hq, hs, plan, self.down, self.down_scales), weights, plan,
                       torch.bfloat16)


__all__ = ["quantize_rows_fp8", "quantize_blocks_fp8", "gemm_fp8_nt", "F8Linear", "dispatch_fp8",
           "experts_gemm_fp8", "experts_gate_fp8", "F8Experts"]
