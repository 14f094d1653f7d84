"""Linear cross entropy (csrc/linear_ce.hip) against its definition in 64 bits.

Tolerances.  Logits are exact products summed in fp32 over at most 256
columns: with e = 2^-24 and |z| sums of size s = Σ|h||W| <= 40 here, lse and
the loss are off by at most about 16·e·s + e·|lse| < 5e-5; db, sums of fp32
probabilities with relative error 2·5e-5, by 2e-4 of Σ_r |g_r| p (plus
the same of the target's share).  dh and dW: a probability is rounded to the
type (half a step, u = 2^-8 / 2^-11·½ … finfo.eps / 2) before a product, so
each is within u + 1e-4 of Σ |terms|, and the output's own rounding adds u of the
value.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu


def inputs(N, V, D, dtype, bias, ignored, seed=0, scale=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    h, W = n(N, D).to(dtype), (n(V, D) * scale / D ** 0.5).to(dtype)
    b = n(V) * 0.5 if bias else None
    t = torch.randint(0, V, (N,), generator=g, device="cuda")
    t[torch.rand(N, generator=g, device="cuda") < 0.3] = V // 3      # one popular item
    t[torch.rand(N, generator=g, device="cuda") < ignored] = -100
    return h, W, b, t, n


def check(h, W, b, t, loss, dloss=None, grads=None, s=40.0):
    # a probability is the exponential of a difference of sums of size s: relative error 2·16·e·s, 7.6e-5 for s = 40
    far = max(1.0, s / 40)
    z = h.double() @ W.double().t()
    if b is not None:
        z = z + b.double()
    ok = t >= 0
    lse = z.logsumexp(1)
    want = torch.where(ok, lse - z.gather(1, t.clamp(min=0)[:, None])[:, 0], 0.0)
    assert loss.dtype == torch.float32
    assert ((loss.double() - want).abs() <= 5e-5 * (1 + 0.05 * want.abs())).all()
    assert (loss[~ok] == 0).all()
    if grads is None:
        return
    dh, dW, db = grads
    g = torch.where(ok, dloss.double(), 0.0)[:, None]
    p = (z - lse[:, None]).exp()
    hit = torch.zeros_like(p)
    hit[torch.arange(len(t), device="cuda")[ok], t[ok]] = 1
    dz, size = g * (p - hit), g.abs() * (p + hit)
    u = torch.finfo(h.dtype).eps / 2
    for got, ref, terms in ((dh, dz @ W.double(), size @ W.double().abs()),
                            (dW, dz.t() @ h.double(), size.t() @ h.double().abs())):
        assert got.dtype == h.dtype and got.shape == ref.shape
        # fp16's smallest value; probabilities below fp32's (and bf16's) smallest normal number, 2^-126, are zero: at
        # most 2^-126 · |operand| lost in each of at most 2^12 terms, operands below 2^4
        tiny = 2.0 ** -24 if h.dtype == torch.float16 else 2.0 ** -110
        assert ((got.double() - ref).abs() <= (u + 1e-4 * far) * terms + u * ref.abs() + tiny).all()
    assert (dh[~ok] == 0).all()
    if b is None:
        assert db is None
    else:
        assert db.dtype == torch.float32
        assert ((db.double() - dz.sum(0)).abs() <= 2e-4 * far * size.sum(0) + 1e-30).all()


CASES = [(1, 1, 8, True, 0.0), (1, 7, 16, False, 0.0), (5, 64, 24, True, 0.0), (64, 65, 32, True, 0.4),
         (63, 1000, 64, False, 0.0), (130, 777, 72, True, 0.2), (384, 3001, 128, True, 0.0), (385, 129, 120, False, 0.5),
         (1000, 5003, 136, True, 0.1), (513, 4099, 256, True, 0.3), (700, 130, 200, False, 0.9), (64, 40001, 128, True, 0.0),
         (4099, 515, 64, True, 0.5), (3000, 20000, 40, False, 0.0), (600, 9001, 248, True, 1.0)]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_loss_and_gradients(case, dtype):
    from recommenders.hip.linear_ce import linear_ce, linear_ce_backward
    N, V, D, bias, ignored = case
    h, W, b, t, n = inputs(N, V, D, dtype, bias, ignored)
    loss, saved = linear_ce(h, W, t, bias=b, save=True)
    dloss = n(N) / N
    grads = linear_ce_backward(saved, dloss)
    check(h, W, b, t, loss, dloss, grads)
    assert torch.equal(linear_ce(h, W, t, bias=b), loss)
    for x, y in zip(grads, linear_ce_backward(saved, dloss)):
        assert x is None or torch.equal(x, y)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_strides(dtype):
    from recommenders.hip.linear_ce import linear_ce, linear_ce_backward
    h, W, b, t, n = inputs(200, 999, 64, dtype, True, 0.2)
    hs = torch.full((200, 3, 64), float("nan"), device="cuda", dtype=dtype)
    Ws = torch.full((999, 96), float("nan"), device="cuda", dtype=dtype)
    hs[:, 1], Ws[:, 16:80] = h, W
    ts, ds = torch.stack([t, t * 0 + 5], 1)[:, 0], torch.rand(400, device="cuda")[::2]
    loss, saved = linear_ce(hs[:, 1], Ws[:, 16:80], ts, bias=b, save=True)
    plain, saved2 = linear_ce(h, W, t, bias=b, save=True)
    assert torch.equal(loss, plain)
    for x, y in zip(linear_ce_backward(saved, ds), linear_ce_backward(saved2, ds.contiguous())):
        assert torch.equal(x, y)


def test_ignored_rows_are_not_read():
    from recommenders.hip.linear_ce import linear_ce, linear_ce_backward
    h, W, b, t, n = inputs(300, 500, 64, torch.bfloat16, True, 0.5)
    dloss = torch.rand(300, device="cuda")
    loss, saved = linear_ce(h, W, t, bias=b, save=True)
    grads = linear_ce_backward(saved, dloss)
    h2, d2 = h.clone(), dloss.clone()
    h2[t < 0], d2[t < 0] = float("nan"), float("inf")
    loss2, saved = linear_ce(h2, W, t, bias=b, save=True)
    assert torch.equal(loss, loss2)
    for x, y in zip(grads, linear_ce_backward(saved, d2)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("scale", [1e-3, 30.0])
def test_flat_and_peaked_rows(scale):
    """Nearly equal logits, and logits hundreds apart that grow along the vocabulary, so the running reference keeps moving."""
    from recommenders.hip.linear_ce import linear_ce, linear_ce_backward
    h, W, b, t, n = inputs(90, 3000, 64, torch.bfloat16, True, 0.0)
    b = torch.linspace(0, 10 * scale, 3000, device="cuda")
    loss, saved = linear_ce(h, W, t, bias=b, save=True)
    dloss = torch.rand(90, device="cuda") + 0.5
    grads = linear_ce_backward(saved, dloss)
    z = h.double() @ W.double().t() + b.double()
    want = z.logsumexp(1) - z.gather(1, t[:, None])[:, 0]
    assert ((loss.double() - want).abs() <= 1e-4 * (1 + z.abs().amax(1) * 0.01)).all()
    sums = (h.double().abs() @ W.double().abs().t() + b.double()).max().item()
    check(h, W, b, t, want.float(), dloss, grads, s=sums)


def test_masked_items():
    """Bias −inf and the lowest fp32 value take items out: no gradient, others as without them."""
    from recommenders.hip.linear_ce import linear_ce, linear_ce_backward
    h, W, b, t, n = inputs(70, 400, 32, torch.bfloat16, True, 0.0)
    t = t % 100
    off = torch.zeros(400, dtype=torch.bool, device="cuda")
    off[100:200], off[250:] = True, True
    b[100:200], b[250:] = -float("inf"), torch.finfo(torch.float32).min
    loss, saved = linear_ce(h, W, t, bias=b, save=True)
    dloss = torch.rand(70, device="cuda")
    dh, dW, db = linear_ce_backward(saved, dloss)
    assert (dW[off] == 0).all() and (db[off] == 0).all()
    keep = (~off).nonzero()[:, 0]
    where = torch.zeros(400, dtype=torch.long, device="cuda")
    where[keep] = torch.arange(len(keep), device="cuda")
    check(h, W[keep], b[keep], where[t], loss, dloss, (dh, dW[keep], db[keep]))


def test_targets_that_are_no_items():
    from recommenders.hip.linear_ce import linear_ce, linear_ce_backward
    h, W, b, t, n = inputs(70, 100, 32, torch.bfloat16, False, 0.0)
    t[5], t[6] = 100, 1 << 40
    loss, saved = linear_ce(h, W, t, save=True)
    assert loss[5].isnan() and loss[6].isnan() and loss.isnan().sum() == 2
    dh, dW, _ = linear_ce_backward(saved, torch.ones(70, device="cuda"))
    assert dh[5].isnan().all() and dh.isnan().any(1).sum() == 2 and dW.isnan().all()


def test_fp16_small_weights():
    """Upstream gradients far below fp16's range leave dW with fp16's own precision."""
    from recommenders.hip.linear_ce import linear_ce, linear_ce_backward
    h, W, b, t, n = inputs(256, 2000, 64, torch.float16, True, 0.0)
    loss, saved = linear_ce(h, W, t, bias=b, save=True)
    one = linear_ce_backward(saved, torch.full((256,), 1.0, device="cuda"))
    tiny = linear_ce_backward(saved, torch.full((256,), 2.0 ** -40, device="cuda"))
    assert torch.equal(one[2], tiny[2] * 2.0 ** 40)
    assert (tiny[1] == 0).all()
    big = linear_ce_backward(saved, torch.full((256,), 2.0 ** -8, device="cuda"))
    assert torch.equal(big[2] * 2.0 ** 8, one[2])


def test_gradient_by_differences():
    """db against central differences of the summed loss (truncation below 1e-5 at step 0.05, fp32 sums 2e-5 / step)."""
    from recommenders.hip.linear_ce import linear_ce, linear_ce_backward
    h, W, b, t, n = inputs(40, 300, 64, torch.bfloat16, True, 0.2)
    _, saved = linear_ce(h, W, t, bias=b, save=True)
    db = linear_ce_backward(saved, torch.ones(40, device="cuda"))[2]
    for v in (0, 100, 299):
        f = []
        for sign in (1, -1):
            c = b.clone()
            c[v] += sign * 0.05
            f.append(linear_ce(h, W, t, bias=c).double().sum().item())
        assert abs((f[0] - f[1]) / 0.1 - db[v].item()) <= 2e-3 * max(1.0, abs(db[v].item()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_captured_and_replayed(dtype):
    from recommenders.hip.linear_ce import linear_ce, linear_ce_backward
    h, W, b, t, n = inputs(200, 5000, 64, dtype, True, 0.3)
    dloss = torch.rand(200, device="cuda")

    def whole():
        loss, saved = linear_ce(h, W, t, bias=b, save=True)
        return (loss, *linear_ce_backward(saved, dloss))
    whole()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = whole()
    for k in range(3):
        h.copy_(n(200, 64))
        t.copy_(torch.randint(-2000 * k, 5000, (200,), device="cuda"))
        graph.replay()
        eager = whole()
        torch.cuda.synchronize()
        for x, y in zip(held, eager):
            assert torch.equal(x, y)


def test_changed_weights_are_refused_and_no_rows():
    from recommenders.hip.linear_ce import linear_ce, linear_ce_backward
    h, W, b, t, n = inputs(4, 10, 8, torch.bfloat16, True, 0.0)
    _, saved = linear_ce(h, W, t, bias=b, save=True)
    W.zero_()
    with pytest.raises(RuntimeError, match="in place"):
        linear_ce_backward(saved, torch.ones(4, device="cuda"))
    loss, saved = linear_ce(h[:0], W, t[:0], bias=b, save=True)
    dh, dW, db = linear_ce_backward(saved, torch.ones(0, device="cuda"))
    assert loss.shape == (0,) and dh.shape == (0, 8) and (dW == 0).all() and (db == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("bias", [False, True])
def test_targets_share_is_not_rounded_twice(dtype, bias):
    """A mean's weight g is the same for all rows and most of a target item's gradient.  Scaled by the largest weight it
    enters as 2^13 (p − 1), and what rounding that moves is at most p (the nearest value kept is −1) and at most u.  Beside it
    the other items' probabilities carry u, every sum 1e-4 and the output's rounding u, once."""
    from recommenders.hip.linear_ce import linear_ce, linear_ce_backward
    h, W, b, t, n = inputs(700, 4001, 64, dtype, bias, 0.0)
    t = torch.randperm(4001, device="cuda")[:700]
    dloss = torch.full((700,), 1.00389 / 512, device="cuda")   # 257 / 256: halfway between bf16 values
    loss, saved = linear_ce(h, W, t, bias=b, save=True)
    dh, dW, db = linear_ce_backward(saved, dloss)
    z = h.double() @ W.double().t() + (0 if b is None else b.double())
    hit = torch.zeros_like(z).scatter_(1, t[:, None], 1.0)
    p, g, u = z.softmax(1), dloss.double()[:, None], torch.finfo(dtype).eps / 2
    ref = (g * (p - hit)).t() @ h.double()
    a = h.double().abs()
    room = u * ref.abs() + (u + 1e-4) * ((g * p).t() @ a) + ((1e-4 + p.clamp(max=u)) * g * hit).t() @ a + 2.0 ** -24
    assert ((dW.double() - ref).abs() <= room).all()
