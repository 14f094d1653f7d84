"""Linear cross entropy over vocabularies whose backward pass takes whole rounds
of 256 blocks of 256 items (65 536 and more) and a remainder that is split
over the rows: every item's dW and db, in pieces of the vocabulary, against
64 bits.  Tolerances as in test_gpu_linear_ce_targets.
"""
import pytest
import torch

from test_gpu_linear_ce import inputs

pytestmark = pytest.mark.gpu
PIECE = 8192


def compare(h, W, b, t, g, loss, dh, dW, db):
    V, u = W.shape[0], torch.finfo(h.dtype).eps / 2
    ok, hd, weight = t >= 0, h.double(), torch.where(t >= 0, g.double(), 0.0)
    pieces = [slice(lo, min(V, lo + PIECE)) for lo in range(0, V, PIECE)]

    def logits(w):
        return hd @ W[w].double().t() + (0 if b is None else b[w].double())

    lse = torch.full((len(t),), -float("inf"), dtype=torch.float64, device="cuda")
    s = 0.0
    for w in pieces:
        lse = torch.logaddexp(lse, logits(w).logsumexp(1))
        s = max(s, (hd.abs() @ W[w].double().abs().t() + (0 if b is None else b[w].double().abs())).max().item())
    e = 1e-4 * max(1.0, s / 40)
    own = W[t.clamp(min=0)].double()
    z = (hd * own).sum(1) + (0 if b is None else b[t.clamp(min=0)].double())
    rest = -torch.expm1(z - lse)
    want = torch.where(ok, lse - z, 0.0)
    # lse - z of 64-bit sums is off by 1e-13 itself
    assert ((loss.double() - want).abs() <= e * want + 1e-12).all()
    small = 2.0 ** -24 if h.dtype == torch.float16 else 2.0 ** -110
    ref_h = -(weight * rest)[:, None] * own
    terms_h, share_h = torch.zeros_like(ref_h), ref_h.abs()
    for w in pieces:
        p = (logits(w) - lse[:, None]).exp() * weight.abs()[:, None]
        mine = ok & (t >= w.start) & (t < w.stop)
        at = (t - w.start).clamp(0, p.shape[1] - 1)[:, None]
        p = p.scatter(1, at, torch.where(mine[:, None], 0.0, p.gather(1, at)))
        hit = torch.zeros_like(p).scatter_(1, at, torch.where(mine, weight * rest, 0.0)[:, None])
        signed = p * weight.sign()[:, None]
        ref_h += signed @ W[w].double()
        terms_h += p @ W[w].double().abs()
        ref = (signed - hit).t() @ hd
        room = u * ref.abs() + (u + e) * (p.t() @ hd.abs()) + e * (hit.abs().t() @ hd.abs()) + small
        off = (dW[w].double() - ref).abs()
        assert (off <= room).all(), (w, (off / room).max())
        if b is not None:
            want_b = (signed - hit).sum(0)
            assert ((db[w].double() - want_b).abs() <= 2 * e * (p.sum(0) + hit.abs().sum(0)) + 1e-30).all(), w
    assert ((dh.double() - ref_h).abs() <= u * ref_h.abs() + (u + e) * terms_h + e * share_h + small).all()
    assert (db is None) == (b is None)


# (N, V, D): a remainder of none, one and a few blocks; one chunk of rows (nothing to split) and several
@pytest.mark.parametrize("N,V,D", [(300, 65536, 32), (700, 65537, 8), (200, 66001, 24), (60, 66001, 32), (64, 65536, 16),
                                   (500, 131073, 8), (333, 70001, 136)])
@pytest.mark.parametrize("bias", [False, True])
def test_whole_rounds_and_the_remainder(N, V, D, bias):
    from recommenders.hip.linear_ce import linear_ce, linear_ce_backward
    dtype = torch.float16 if N % 2 else torch.bfloat16
    h, W, b, t, n = inputs(N, V, D, dtype, bias, 0.2)
    t[:10] = torch.tensor([0, 255, 256, V - 1, V - 2, V // 256 * 256 - 1, 65535, 65279, 65280, 31], device="cuda")
    loss, saved = linear_ce(h, W, t, bias=b, save=True)
    g = torch.rand(N, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)) / N
    compare(h, W, b, t, g, loss, *linear_ce_backward(saved, g))


@pytest.mark.parametrize("N,V,D", [(2600, 65537, 64), (2600, 65600, 128), (2600, 65537, 200), (17001, 65537, 16)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_popular_items(N, V, D, dtype):
    """Most rows' targets among a few neighbouring items, more than a wave lists at once, others spread over the vocabulary,
    rows of unlike weights, some of them negative."""
    from recommenders.hip.linear_ce import linear_ce, linear_ce_backward
    h, W, b, t, n = inputs(N, V, D, dtype, D % 128 == 0 or D == 16, 0.1)
    g = torch.Generator(device="cuda").manual_seed(7)
    r = torch.rand(N, generator=g, device="cuda")
    hot = torch.randint(0, 40, (N,), generator=g, device="cuda")
    t = torch.where(r < 0.6, 1000 + hot % 5, torch.where(r < 0.7, 1032 + hot, torch.where(r < 0.75, 65530 + hot % 7, t)))
    dloss = torch.where(torch.rand(N, generator=g, device="cuda") < 0.8, 0.2, 1.0) / N
    dloss[::17] *= -0.3
    loss, saved = linear_ce(h, W, t, bias=b, save=True)
    grads = linear_ce_backward(saved, dloss)
    compare(h, W, b, t, dloss, loss, *grads)
    for x, y in zip(grads, linear_ce_backward(saved, dloss)):
        assert x is None or torch.equal(x, y)


@pytest.mark.parametrize("N,V,D", [(1500, 65537, 64), (2500, 3001, 136)])
def test_captured_and_replayed(N, V, D):
    """More rows than one workgroup lists, whole rounds or splits, a popular item that changes between replays."""
    from recommenders.hip.linear_ce import linear_ce, linear_ce_backward
    h, W, b, t, n = inputs(N, V, D, torch.bfloat16, True, 0.3)
    g = torch.rand(N, device="cuda")

    def whole():
        loss, saved = linear_ce(h, W, t, bias=b, save=True)
        return (loss, *linear_ce_backward(saved, g))
    whole()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = whole()
    for k in range(4):
        h.copy_(n(N, D))
        t.copy_(torch.randint(-V // 2 if k else 0, V, (N,), device="cuda"))
        t[: N * k // 4] = 17 + 900 * k
        b[100:200] = -1e9 if k % 2 else 0.0
        graph.replay()
        eager = whole()
        torch.cuda.synchronize()
        for x, y in zip(held, eager):
            assert torch.equal(x, y)
    compare(h, W, b, t, g, *held)
