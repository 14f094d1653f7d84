"""The target's share of the linear cross entropy's loss and gradients: rows
that the model predicts well, and rows of unlike weights.

A probability is the exponential of a difference of fp32 sums of size
s = max Σ|h||W| + |b|: relative error e = 2·16·2^-24·s (7.6e-5 for s = 40),
taken as 1e-4·max(1, s / 40) with the sums that follow.  The odds against the
target, q = Σ_{v ≠ t} p_v / p_t, carry that relative error too, so the loss
log(1 + q) and the target's share 1 − p_t are within e of themselves,
however small they are.  The other items' probabilities are rounded to the
inputs' type (u = finfo.eps / 2) for the gradient products, the target's
share is not, and each output is rounded once.
"""
import pytest
import torch

from test_gpu_linear_ce import check, inputs

pytestmark = pytest.mark.gpu
TYPES = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])


def exact(h, W, b, t, g):
    """Loss, gradients, and what bounds their errors, in 64 bits; 1 − p_t from the other items' probabilities."""
    h, W, g = h.double(), W.double(), g.double()
    z = h @ W.t() + (0 if b is None else b.double())
    s = (h.abs() @ W.abs().t() + (0 if b is None else b.double().abs())).max().item()
    p = z.softmax(1)
    others = p.scatter(1, t[:, None], 0.0)
    rest = others.sum(1)
    loss = -torch.log1p(-rest)
    loss = torch.where(rest > 0.5, z.logsumexp(1) - z.gather(1, t[:, None])[:, 0], loss)
    hit = torch.zeros_like(p).scatter_(1, t[:, None], 1.0) * (g * rest)[:, None]
    dz = g[:, None] * others - hit
    return dict(s=s, rest=rest, loss=loss, dz=dz, others=(g[:, None] * others).abs(), hit=hit.abs(), dh=dz @ W, dW=dz.t() @ h, db=dz.sum(0))


def close(h, W, b, t, g, loss, dh=None, dW=None, db=None):
    x = exact(h, W, b, t, g)
    e, u = 1e-4 * max(1.0, x["s"] / 40), torch.finfo(h.dtype).eps / 2
    assert ((loss.double() - x["loss"]).abs() <= e * x["loss"] + 2.0 ** -140).all()
    small = 2.0 ** -24 if h.dtype == torch.float16 else 2.0 ** -110
    for got, ref, terms, share in ((dh, x["dh"], x["others"] @ W.double().abs(), x["hit"] @ W.double().abs()),
                                   (dW, x["dW"], x["others"].t() @ h.double().abs(), x["hit"].t() @ h.double().abs())):
        if got is None:
            continue
        room = u * ref.abs() + (u + e) * terms + e * share + small
        off = (got.double() - ref).abs()
        assert (off <= room).all(), (off / room).max()
    if db is not None:
        assert ((db.double() - x["db"]).abs() <= 2 * e * (x["others"].sum(0) + x["hit"].sum(0)) + 1e-30).all()


@pytest.mark.parametrize("D,bias", [(64, True), (128, False), (200, True)])
@TYPES
def test_loss_and_dh_of_rows_that_are_predicted_well(D, bias, dtype):
    """Hidden rows along their targets' weights, p_t from a tenth to 1 − 1e-9."""
    from recommenders.hip.linear_ce import linear_ce, linear_ce_backward
    h, W, b, t, n = inputs(300, 4001, D, dtype, bias, 0.0)
    t = torch.randint(0, 4001, (300,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    along = W[t].float()
    h = (along / along.square().sum(1, keepdim=True) * torch.linspace(6, 30, 300, device="cuda")[:, None] + 0.05 * n(300, D)).to(dtype)
    loss, saved = linear_ce(h, W, t, bias=b, save=True)
    g = torch.full((300,), 1 / 300, device="cuda")
    x = exact(h, W, b, t, g)
    assert x["rest"].min() < 1e-7 and x["rest"].max() > 0.5
    close(h, W, b, t, g, loss, linear_ce_backward(saved, g)[0])


@pytest.mark.parametrize("weights", ["clicks and purchases", "uniform", "spread", "signed"])
@pytest.mark.parametrize("bias", [False, True])
@TYPES
def test_rows_of_unlike_weights(weights, bias, dtype):
    from recommenders.hip.linear_ce import linear_ce, linear_ce_backward
    h, W, b, t, n = inputs(900, 4001, 64, dtype, bias, 0.0)
    g = torch.Generator(device="cuda").manual_seed(4)
    t = torch.randperm(4001, generator=g, device="cuda")[:900]
    t[:200] = t[0]                            # one popular item, hit many times in a chunk of rows
    r = torch.rand(900, generator=g, device="cuda")
    dloss = {"clicks and purchases": torch.where(r < 0.8, 0.2, 1.0), "uniform": r + 0.01, "spread": torch.exp(-6 * r),
             "signed": r - 0.5}[weights] / 900
    loss, saved = linear_ce(h, W, t, bias=b, save=True)
    close(h, W, b, t, dloss, loss, *linear_ce_backward(saved, dloss))


@TYPES
def test_a_popular_item_in_every_chunk(dtype):
    """Most rows have the same target: its share is a long sum."""
    from recommenders.hip.linear_ce import linear_ce, linear_ce_backward
    h, W, b, t, n = inputs(3000, 500, 40, dtype, True, 0.0)
    t[torch.rand(3000, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) < 0.8] = 33
    dloss = torch.full((3000,), 0.3 / 3000, device="cuda")
    loss, saved = linear_ce(h, W, t, bias=b, save=True)
    close(h, W, b, t, dloss, loss, *linear_ce_backward(saved, dloss))


@TYPES
def test_masked_targets_and_rows_with_nothing_else(dtype):
    """A masked target: the loss is as large as its bias says and its gradients are those of probability 0.  Items that are all
    masked but one: that one's rows lose nothing and leave no gradient."""
    from recommenders.hip.linear_ce import linear_ce, linear_ce_backward
    h, W, b, t, n = inputs(70, 300, 32, dtype, True, 0.0)
    b[7] = -1e9
    t[4] = 7
    loss, saved = linear_ce(h, W, t, bias=b, save=True)
    assert abs(loss[4].item() - 1e9) <= 64 and (loss[:4] < 100).all()
    dh, dW, db = linear_ce_backward(saved, torch.ones(70, device="cuda"))
    z = h.double() @ W.double().t() + b.double()
    check(h, W, b, t, (z.logsumexp(1) - z.gather(1, t[:, None])[:, 0]).float(), torch.ones(70, device="cuda"), (dh, dW, db))
    assert abs(db[7].item() + (t == 7).sum().item()) <= 1e-3
    b[:] = -float("inf")
    b[7], t[:] = 0.5, 7
    loss, saved = linear_ce(h, W, t, bias=b, save=True)
    dh, dW, db = linear_ce_backward(saved, torch.ones(70, device="cuda"))
    assert (loss == 0).all() and (dh == 0).all() and (dW == 0).all() and (db == 0).all()
