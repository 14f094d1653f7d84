"""Operands of the delta rule's calls that the documentation allows, and the same answer the first time as later."""
import pytest
import torch

from test_gpu_delta import definition, inputs, name, near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_step_operands_need_no_alignment(dtype):
    """q, k and v that start anywhere and whose rows lie anywhere: the step reads them value by value."""
    from recommenders.hip.delta import delta_rule_step
    x, n = inputs(3, 1, 2, 4, 40, 24, dtype)
    x = {m: t[:, 0] for m, t in x.items()}
    for m, width in (("q", 2 * 40), ("k", 2 * 40), ("v", 4 * 24)):
        room = torch.full((3, width + 7), float("nan"), device="cuda", dtype=dtype)
        room[:, 3:3 + width] = x[m].flatten(1)
        x[m] = room[:, 3:3 + width].unflatten(1, x[m].shape[1:])
        assert x[m].data_ptr() % 16
    state = n(3, 4, 40, 24)
    want = definition({m: t[:, None] for m, t in x.items()}, 0.5, None, state.clone())
    o = delta_rule_step(**x, state=state, scale=0.5)
    near(o, want[0][:, 0], name("o", o))
    near(state, want[1], "state")
