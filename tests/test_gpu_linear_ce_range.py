"""Linear cross entropy with items masked by large finite biases, and with
logits far from zero.

A masked item has probability 0 in fp32 and in 64 bits alike, so losses and
gradients are those of the other items, with the tolerances of
test_gpu_linear_ce.  Where all logits are of size c, neighbouring fp32 values
are 2^-23·c apart; the biases lie 2^-10·c apart, so one item has all of the
probability in either precision, and the loss, a difference of two logits that
are each rounded at most four times (the product's two halves, the bias, the
difference), is within 8·2^-24·c.
"""
import pytest
import torch

from test_gpu_linear_ce import check, inputs

pytestmark = pytest.mark.gpu
TYPES = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])


@pytest.mark.parametrize("N,V,D", [(64, 10001, 32), (130, 3001, 200)])
@pytest.mark.parametrize("low", [-1e9, -2e9, -1e10, -1e12, -1e20, -1e30, -1e38])
@pytest.mark.parametrize("where", ["first halves", "whole runs"])
@TYPES
def test_large_finite_masks(N, V, D, low, where, dtype):
    """Half of every 64 items (the first ones of any piece of the vocabulary among them), or all of the first two thirds."""
    from recommenders.hip.linear_ce import linear_ce, linear_ce_backward
    h, W, b, t, n = inputs(N, V, D, dtype, True, 0.1)
    item = torch.arange(V, device="cuda")
    off = item % 64 < 32 if where == "first halves" else item < V * 2 // 3
    keep = (~off).nonzero()[:, 0]
    t = torch.where(t < 0, t, keep[t.clamp(min=0) % len(keep)])
    b[off] = low
    loss, saved = linear_ce(h, W, t, bias=b, save=True)
    dloss = torch.rand(N, device="cuda") / N
    dh, dW, db = linear_ce_backward(saved, dloss)
    assert (dW[off] == 0).all() and (db[off] == 0).all()
    place = torch.zeros(V, dtype=torch.long, device="cuda")
    place[keep] = torch.arange(len(keep), device="cuda")
    check(h, W[keep], b[keep], torch.where(t < 0, t, place[t.clamp(min=0)]), loss, dloss, (dh, dW[keep], db[keep]))
    assert torch.equal(linear_ce(h, W, t, bias=b), loss)


@pytest.mark.parametrize("c", [-1e5, 1e5, -1e7, 1e7, -1e9, 1e9, -1e20, 1e20, -1e30, 1e30, -1e38])
@TYPES
def test_all_logits_far_from_zero(c, dtype):
    from recommenders.hip.linear_ce import linear_ce, linear_ce_backward
    h, W, b, t, n = inputs(70, 700, 64, dtype, True, 0.1)
    g = torch.Generator().manual_seed(5)
    j = torch.randperm(700, generator=g).cuda()
    b = (c * (1 + j.double() * 2.0 ** -10)).float()
    t[::3] = b.argmax()                       # rows that the model predicts, and others
    loss, saved = linear_ce(h, W, t, bias=b, save=True)
    dloss = torch.rand(70, device="cuda") + 0.5
    grads = linear_ce_backward(saved, dloss)
    z = h.double() @ W.double().t() + b.double()
    ok = t >= 0
    want = torch.where(ok, z.logsumexp(1) - z.gather(1, t.clamp(min=0)[:, None])[:, 0], 0.0)
    assert ((loss.double() - want).abs() <= 8 * 2.0 ** -24 * 1.7 * abs(c)).all()
    check(h, W, b, t, want.float(), dloss, grads)
