"""What a forward call leaves for the backward call is used on another stream, and let go while that stream is still busy:
the forward's stream must not get its memory back before."""
import pytest
import torch

import test_gpu_delta
import test_gpu_linear_ce

pytestmark = pytest.mark.gpu


def busy():
    a = torch.randn(4096, 4096, device="cuda")
    for _ in range(40):
        a = torch.tanh(a @ a)
    return a


def on_two_streams(forward, backward):
    """forward() -> saved on a side stream, backward(saved) on this one behind other work; the side stream then takes and fills
    memory of the sizes that were let go."""
    want = [t.clone() for t in backward(forward()) if t is not None]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            saved = forward()
        torch.cuda.current_stream().wait_stream(side)
        held = busy()
        sizes = [t.numel() * t.element_size() for t in vars(saved).values() if isinstance(t, torch.Tensor) and t.is_cuda]
        got = [t for t in backward(saved) if t is not None]
        del saved
        with torch.cuda.stream(side):
            taken = [torch.full((n,), 255, dtype=torch.uint8, device="cuda") for n in sizes for _ in range(2)]
        torch.cuda.synchronize()
        for a, e in zip(got, want):
            assert torch.equal(a, e)
        del taken, held


def test_linear_ce():
    from recommenders.hip.linear_ce import linear_ce, linear_ce_backward
    h, W, b, t, n = test_gpu_linear_ce.inputs(3000, 5000, 128, torch.bfloat16, True, 0.1)
    dloss = torch.rand(3000, device="cuda")
    on_two_streams(lambda: linear_ce(h, W, t, bias=b, save=True)[1], lambda saved: linear_ce_backward(saved, dloss))


@pytest.mark.parametrize("B,T", [(200, 50), (2, 2000)])
def test_delta(B, T):
    from recommenders.hip.delta import delta_rule, delta_rule_backward
    x, n = test_gpu_delta.inputs(B, T, 1, 2, 64, 64, torch.float32)
    do = n(B, T, 2, 64)
    on_two_streams(lambda: delta_rule(**x, save=True)[2], lambda saved: delta_rule_backward(saved, do))


def test_backward_captured_behind_an_eager_forward():
    """The captured backward call runs on the capture's stream; what the forward call left is held by the program."""
    from recommenders.hip.delta import delta_rule, delta_rule_backward
    from recommenders.hip.linear_ce import linear_ce, linear_ce_backward
    h, W, b, t, n = test_gpu_linear_ce.inputs(300, 2000, 64, torch.bfloat16, True, 0.1)
    x, m = test_gpu_delta.inputs(3, 90, 1, 2, 32, 32, torch.float32)
    g, do = torch.rand(300, device="cuda"), m(3, 90, 2, 32)
    kept, saved = linear_ce(h, W, t, bias=b, save=True)[1], delta_rule(**x, save=True)[2]

    def both():
        return [*linear_ce_backward(kept, g), *delta_rule_backward(saved, do)[:5]]
    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for _ in range(3):
        g.copy_(torch.rand(300, device="cuda"))
        do.copy_(m(3, 90, 2, 32))
        graph.replay()
        eager = both()
        torch.cuda.synchronize()
        for a, e in zip(held, eager):
            assert torch.equal(a, e)
    del kept, saved
    torch.cuda.synchronize()
