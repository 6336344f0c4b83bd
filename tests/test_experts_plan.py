"""Host checks of the experts' plan as an object: what a library call is given are always the plan's own
tensors and the sizes that belong to them."""
import copy
import pickle

import pytest
import torch

import momijo_amd as mj


def _plan(tokens=4, topk=2, experts=3):
    return mj.ExpertPlan(torch.arange(tokens * topk, dtype=torch.int32).reshape(tokens, topk),
                         torch.full((experts + 1,), tokens * topk, dtype=torch.int32))


def _given(plan):
    return plan._args == (plan.pos.data_ptr(), plan.offsets.data_ptr(), plan.experts)


@pytest.mark.parametrize("name,value", [
    ("pos", torch.zeros(4, 2, dtype=torch.int32)), ("offsets", torch.zeros(4, dtype=torch.int32)), ("tokens", 400),
    ("topk", 200), ("rows", 800), ("experts", 300), ("device", torch.device("cuda", 0))])
def test_nothing_of_a_plan_is_replaced(name, value):
    plan = _plan()
    old = getattr(plan, name)
    with pytest.raises(AttributeError):
        setattr(plan, name, value)
    with pytest.raises(AttributeError):
        delattr(plan, name)
    assert getattr(plan, name) is old or getattr(plan, name) == old
    assert _given(plan)


@pytest.mark.parametrize("again", [copy.copy, copy.deepcopy, lambda p: pickle.loads(pickle.dumps(p))])
def test_a_copied_plan_has_its_own_tensors(again):
    plan = _plan()
    twin = again(plan)
    assert _given(plan) and _given(twin)
    assert torch.equal(twin.pos, plan.pos) and torch.equal(twin.offsets, plan.offsets)
    assert (twin.tokens, twin.topk, twin.rows, twin.experts) == (4, 2, 8, 3) and twin.device == plan.device
    assert twin._index == twin.pos.get_device()


def test_a_plan_loaded_to_another_device(tmp_path):
    """The device of a plan's tensors is the one that its rows are checked against."""
    plan = _plan()
    plan._index = 0  # as of a plan made on the GPU
    torch.save(plan, tmp_path / "plan")
    twin = torch.load(tmp_path / "plan", map_location="cpu", weights_only=False)
    assert twin._index == -1 and _given(twin)


def test_a_plan_follows_its_tensors():
    """Tensors that grew in place lie elsewhere."""
    plan = _plan()
    plan.pos.resize_(1 << 12, 2)
    plan.offsets.resize_(1 << 12)
    assert _given(plan)
