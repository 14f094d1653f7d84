"""What a backward call reads again has to be what the forward call read."""
import pytest
import torch

import test_gpu_delta
import test_gpu_linear_ce

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", ["W", "bias"])
def test_linear_ce_refuses_weights_with_other_memory(which):
    """tensor.data = other, or a storage that was let go, does not count as a write in place."""
    from recommenders.hip.linear_ce import linear_ce, linear_ce_backward
    h, W, b, t, n = test_gpu_linear_ce.inputs(20, 100, 32, torch.bfloat16, True, 0.1)
    dloss = torch.ones(20, device="cuda")
    loss, saved = linear_ce(h, W, t, bias=b, save=True)
    want = linear_ce_backward(saved, dloss)
    x = {"W": W, "bias": b}[which]
    kept = x.data
    x.data = kept.clone() + 1
    with pytest.raises(RuntimeError, match="other memory"):
        linear_ce_backward(saved, dloss)
    x.data = kept[:50]
    with pytest.raises(RuntimeError, match="other memory"):
        linear_ce_backward(saved, dloss)
    x.data = kept
    for a, e in zip(linear_ce_backward(saved, dloss), want):
        assert torch.equal(a, e)


@pytest.mark.parametrize("which", ["q", "k", "v", "g", "beta", "state", "lens"])
def test_delta_refuses_operands_with_other_memory(which):
    from recommenders.hip.delta import delta_rule, delta_rule_backward
    x, n = test_gpu_delta.inputs(2, 40, 1, 2, 16, 24, torch.float32)
    x |= {"state": n(2, 2, 16, 24), "lens": torch.tensor([40, 7], device="cuda")}
    o, final, saved = delta_rule(**x, save=True)
    do = n(*o.shape)
    want = delta_rule_backward(saved, do)
    kept = x[which].data
    x[which].data = kept.clone()
    with pytest.raises(RuntimeError, match="other memory"):
        delta_rule_backward(saved, do)
    x[which].data = kept
    for a, e in zip(delta_rule_backward(saved, do), want):
        assert torch.equal(a, e)
