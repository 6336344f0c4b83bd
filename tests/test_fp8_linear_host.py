"""Host checks of what an F8Linear holds: a replaced weight, scale or bias goes through the constructor's checks,
since a forward goes by its sizes."""
import pytest
import torch

import momijo_amd as mj

F8 = torch.float8_e4m3fn


def _linear(bias=None):
    return mj.F8Linear(torch.zeros(200, 272).to(F8), torch.ones(2, 3), bias)


def _off(t):
    """t at an address that is no multiple of 16 bytes."""
    flat = torch.empty(t.numel() + 1, dtype=torch.uint8)[1:].view(t.dtype)
    return flat.view(t.shape).copy_(t)


@pytest.mark.parametrize("name,value", [
    ("q", torch.zeros(72, 272).to(F8)), ("q", torch.zeros(199, 272).to(F8)), ("q", torch.zeros(200, 256).to(F8)),
    ("q", torch.zeros(200, 272)), ("scales", torch.ones(2, 2)), ("scales", torch.ones(1, 3)),
    ("scales", torch.ones(2, 3, dtype=torch.float64)), ("bias", torch.ones(199)), ("in_features", 4096),
    ("out_features", 4096)])
@pytest.mark.parametrize("bias", [None, torch.ones(200)])
def test_what_does_not_fit_is_refused(name, value, bias):
    lin = _linear(bias)
    old = getattr(lin, name)
    with pytest.raises((AttributeError, ValueError)):
        setattr(lin, name, value)
    assert getattr(lin, name) is old


def test_others_of_their_shapes():
    lin = _linear()
    q = torch.randn(272, 200).to(F8).t()          # strides that the kernels do not take
    lin.q, lin.scales = q, torch.full((3, 2), 2.0).t()
    lin.bias, lin.act = torch.ones(200, dtype=torch.bfloat16), mj.EPI_SILU
    assert lin.q.is_contiguous() and torch.equal(lin.q.float(), q.float())
    assert lin.scales.is_contiguous() and bool((lin.scales == 2).all())
    assert lin.bias.dtype is torch.float32 and lin.act == mj.EPI_SILU
    lin.q = _off(q.contiguous())
    assert lin.q.data_ptr() % 16 == 0 and torch.equal(lin.q.float(), q.float())
    lin.bias = None
    assert lin.bias is None and (lin.in_features, lin.out_features) == (272, 200)
