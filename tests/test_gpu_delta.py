"""Gated delta rule (csrc/delta.hip) against its definition stepped in 64 bits,
gradients by differentiating that; one gradient against differences too.

Tolerances.  Everything inside is fp32 or better: three bf16 planes drop terms
below 2^-24 of a product, so each of the chained products (at most 6: K·S,
T·X, P·U and their merges) adds at most about (depth 128 + 6 plane sums)·2^-24
relative to the sizes of its terms, which for unit keys and these decays are
within ten of the result's root mean square: 10·6·134·2^-24 = 5e-4 in the worst
case and its square root's share, about 4e-5, where roundings do not line up.
Outputs have to be within 4e-5 of the largest value (plus half a rounding
step of a bf16 output, 2^-8 of the value): a wrong row, head, mask or
chunk is off by the values' own size.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu


def inputs(B, T, Hk, Hv, Dk, Dv, dtype, seed=0, slow=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    unit = lambda x: x / x.norm(dim=-1, keepdim=True)  # noqa: E731
    x = dict(q=unit(n(B, T, Hk, Dk)).to(dtype), k=unit(n(B, T, Hk, Dk)).to(dtype), v=n(B, T, Hv, Dv).to(dtype),
             g=-torch.rand(B, T, Hv, generator=g, device="cuda") * (0.02 if slow else 1.0),
             beta=torch.sigmoid(n(B, T, Hv)))
    return x, n


def definition(x, scale, lens, state, do=None, dstate=None):
    """o, final and the gradients, one position after the other, in 64 bits."""
    names = ["q", "k", "v", "g", "beta"]
    y = {n: x[n].double() for n in names}
    B, T, Hk, Dk = y["q"].shape
    Hv, Dv = y["v"].shape[2:]
    S = torch.zeros(B, Hv, Dk, Dv, dtype=torch.float64, device="cuda") if state is None else state.double()
    y["S"] = S
    y = {n: t.detach().clone().requires_grad_(do is not None) for n, t in y.items()}
    S, out = y["S"], []
    at = lens if lens is not None else torch.full((B,), T, device="cuda")
    for t in range(T):
        on = (t < at)[:, None]
        q, k = (y[n][:, t].repeat_interleave(Hv // Hk, 1) for n in ("q", "k"))
        q, k, v = (torch.where(on[..., None], z, 0.0) for z in (q, k, y["v"][:, t]))
        a = torch.where(on, y["g"][:, t], 0.0).exp()[..., None, None]
        b = torch.where(on, y["beta"][:, t], 0.0)[..., None]
        S = S * a
        u = b * (v - torch.matmul(k[..., None, :], S)[..., 0, :])
        S = S + k[..., None] * u[..., None, :]
        out.append(scale * torch.matmul(q[..., None, :], S)[..., 0, :])
    o = torch.stack(out, 1)
    if do is None:
        return o, S
    loss = (o * torch.where((torch.arange(T, device="cuda")[None] < at[:, None])[..., None, None], do.double(), 0.0)).sum()
    if dstate is not None:
        loss = loss + (S * dstate.double()).sum()
    grads = torch.autograd.grad(loss, [y[n] for n in names + ["S"]])
    return (o.detach(), S.detach()) + grads


def near(got, want, what):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), what
    room = 4e-5 * want.abs().max() + 1e-30
    if what.endswith("bf16"):
        room = room + 2.0 ** -8 * want.abs()
    off = (got - want).abs() - room
    assert (off <= 0).all(), f"{what}: {(got - want).abs().max():.3g} off, largest value {want.abs().max():.3g}"


def name(n, t):
    return n + (" bf16" if t.dtype == torch.bfloat16 else "")


CASES = [
    # B, T, Hk, Hv, Dk, Dv, lens, state
    (1, 1, 1, 1, 8, 8, None, False),
    (3, 5, 1, 1, 16, 24, [5, 1, 0], True),
    (2, 15, 2, 2, 32, 32, None, True),
    (2, 16, 1, 2, 64, 16, [16, 9], False),
    (4, 50, 2, 2, 64, 64, [50, 33, 17, 0], False),
    (3, 64, 1, 3, 40, 72, [64, 63, 48], True),
    (2, 65, 2, 4, 128, 128, [65, 64], True),
    (2, 130, 1, 1, 104, 120, None, False),
    (3, 193, 2, 2, 24, 40, [193, 128, 70], True),
    (1, 700, 1, 2, 64, 128, None, True),
    (300, 33, 1, 1, 64, 64, list(range(33)) * 9 + [3, 33, 0], False),
    (900, 50, 1, 2, 64, 64, [1 + 50 * i // 900 for i in range(900)], False),
    (2, 1100, 2, 2, 128, 96, [1100, 517], True),
    (1, 1500, 1, 1, 40, 24, None, True),
    (2, 900, 1, 2, 104, 72, [411, 900], True),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:6])))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_forward_and_backward(case, dtype):
    from recommenders.hip.delta import delta_rule, delta_rule_backward
    B, T, Hk, Hv, Dk, Dv, lens, with_state = case
    x, n = inputs(B, T, Hk, Hv, Dk, Dv, dtype)
    lens = None if lens is None else torch.tensor(lens, device="cuda")
    state = n(B, Hv, Dk, Dv) * 0.5 if with_state else None
    do, dstate = n(B, T, Hv, Dv).to(dtype), n(B, Hv, Dk, Dv) if with_state else None
    want = definition(x, 0.3, lens, state, do, dstate)
    if lens is not None:   # what lies behind a length is never read
        behind = torch.arange(T, device="cuda")[None] >= lens[:, None]
        for t in (*x.values(), do):
            t[behind] = float("nan")
    o, final, saved = delta_rule(**x, scale=0.3, lens=lens, state=state, save=True)
    near(o, want[0], name("o", o))
    near(final, want[1], "state")
    again, last = delta_rule(**x, scale=0.3, lens=lens, state=state)
    assert torch.equal(again, o) and torch.equal(last, final)
    got = delta_rule_backward(saved, do, dstate)
    for what, a, b in zip(("dq", "dk", "dv", "dg", "dbeta"), got, want[2:]):
        near(a, b, name(what, a))
    if with_state:
        near(got[5], want[7], "dstate")
    else:
        assert got[5] is None
    for a, b in zip(got, delta_rule_backward(saved, do, dstate)):
        assert a is None or torch.equal(a, b)


def test_strides():
    """Heads cut out of one projection, time-major rows, scalars of any stride: the same bits as contiguous copies."""
    from recommenders.hip.delta import delta_rule, delta_rule_backward
    B, T, H, D = 3, 70, 2, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    one = (torch.randn(T, B, 3 * H * D, generator=g, device="cuda") * 0.2).bfloat16().transpose(0, 1)
    q, k, v = (one[..., i * H * D:(i + 1) * H * D].unflatten(-1, (H, D)) for i in range(3))
    two = torch.rand(B, 2 * H, T, generator=g, device="cuda").transpose(1, 2)
    gg, beta = -two[..., 0::2], two[..., 1::2]
    do = torch.randn(B, H, T, D, generator=g, device="cuda").bfloat16().transpose(1, 2)
    o, s, saved = delta_rule(q, k, v, gg, beta, save=True)
    grads = delta_rule_backward(saved, do)
    c = [t.contiguous() for t in (q, k, v, gg, beta)]
    o2, s2, saved2 = delta_rule(*c, save=True)
    assert torch.equal(o, o2) and torch.equal(s, s2)
    for a, b in zip(grads[:5], delta_rule_backward(saved2, do.contiguous())[:5]):
        assert torch.equal(a, b)


def test_in_parts_equals_whole():
    """A long row in two calls, then token by token, the state handed on."""
    from recommenders.hip.delta import delta_rule, delta_rule_step
    x, _ = inputs(2, 150, 1, 2, 64, 48, torch.float32, slow=True)
    o, final = delta_rule(**x)
    part = lambda a, b: {n: t[:, a:b] for n, t in x.items()}  # noqa: E731
    o1, s = delta_rule(**part(0, 87))
    o2, s = delta_rule(**part(87, 140), state=s)
    outs = [o1, o2]
    for t in range(140, 150):
        outs.append(delta_rule_step(**{n: y[:, t] for n, y in x.items()}, state=s)[:, None])
    near(torch.cat(outs, 1), o, "o")
    near(s, final, "state")


@pytest.mark.parametrize("B,Hk,Hv,Dk,Dv", [(1, 1, 1, 8, 8), (5, 2, 4, 64, 40), (3, 1, 3, 128, 128), (70, 2, 2, 24, 72)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_step(B, Hk, Hv, Dk, Dv, dtype):
    from recommenders.hip.delta import delta_rule_step
    x, n = inputs(B, 1, Hk, Hv, Dk, Dv, dtype)
    pool = n(2 * B, Hv, Dk, Dv)
    held = pool.clone()
    want = definition(x, 0.5, None, held[::2])
    o = delta_rule_step(**{n_: t[:, 0] for n_, t in x.items()}, state=pool[::2], scale=0.5)
    near(o, want[0][:, 0], name("o", o))
    near(pool[::2], want[1], "state")
    assert torch.equal(pool[1::2], held[1::2])


def test_resets_and_extreme_decays():
    """g = −inf forgets everything before; very small and very large decays stay finite and right."""
    from recommenders.hip.delta import delta_rule, delta_rule_backward, delta_rule_step
    x, n = inputs(2, 140, 1, 1, 32, 32, torch.float32)
    x["g"][:, 20] = -float("inf")
    x["g"][:, 90:95] = -300.0
    x["g"][:, 100:110] = 0.0
    o, final, saved = delta_rule(**x, save=True)
    safe = dict(x, g=x["g"].clamp(min=-700))
    do = n(2, 140, 1, 32)
    want = definition(safe, 32 ** -0.5, None, None, do)
    near(o, want[0], "o")
    near(final, want[1], "state")
    for what, a, b in zip(("dq", "dk", "dv", "dg", "dbeta"), delta_rule_backward(saved, do), want[2:]):
        near(a, b, what)
    tail, s = delta_rule(**{n_: t[:, 20:] for n_, t in x.items()})
    near(tail, o[:, 20:], "o behind a reset")
    state = torch.full((2, 1, 32, 32), float("inf"), device="cuda")
    step = delta_rule_step(**{n_: t[:, 20] for n_, t in x.items()}, state=state)
    near(step, o[:, 20], "o of a reset step")


def test_repeated_keys():
    """The same key at every position, written at full strength: the triangular system is as far from diagonal as it gets."""
    from recommenders.hip.delta import delta_rule, delta_rule_backward
    x, n = inputs(2, 128, 1, 1, 64, 32, torch.float32)
    x["k"] = x["k"][:, :1].expand(-1, 128, -1, -1).contiguous()
    x["beta"] = torch.full_like(x["beta"], 0.999)
    x["g"] = torch.zeros_like(x["g"])
    do = n(2, 128, 1, 32)
    want = definition(x, 0.125, None, None, do)
    o, final, saved = delta_rule(**x, scale=0.125, save=True)
    near(o, want[0], "o")
    grads = delta_rule_backward(saved, do)
    for what, a, b in zip(("dq", "dk", "dv", "dg", "dbeta"), grads, want[2:]):
        if what != "dg":
            near(a, b, what)
    # dg cancels here: every write replaces the last one whole, so a decay hardly matters (values below 1e-3), while the
    # terms dA_ij A_ij = −(dX_i · U_j) A_ij it sums are of size 1.  A term carries at most 16 roundings of 2^-24 (dX and
    # U 4 each for their chains of products, their planes 3, the contraction 2, k·k 2, the product with it 1), and dg is a
    # sum of a chunk's terms, so 16 · 2^-24 · sum |terms| bounds its error.  U_t = beta (v_t − Sᵀk), and Sᵀk is u_0 + .. + u_{t-1}.
    u, total = [], torch.zeros(2, 1, 32, dtype=torch.float64, device="cuda")
    for t in range(128):
        u.append(0.999 * (x["v"][:, t].double() - total))
        total = total + u[-1]
    u, dx = torch.stack(u, 1)[:, :, 0], want[4][:, :, 0].double() / 0.999
    for lo in (0, 64):
        terms = torch.matmul(dx[:, lo:lo + 64], u[:, lo:lo + 64].transpose(1, 2).contiguous()).tril(-1).abs().sum((1, 2))
        off = (grads[3] - want[5]).abs()[:, lo:lo + 64, 0].amax(1)
        assert (off <= 16 * 2.0 ** -24 * terms).all()


def test_gradient_by_differences():
    """dg of one position against central differences of the forward pass itself: with step e the truncation is e²·|f'''|/6
    (below 1e-4 of these values) and fp32 sums leave about 1e-6 / e."""
    from recommenders.hip.delta import delta_rule, delta_rule_backward
    x, n = inputs(1, 80, 1, 1, 32, 32, torch.float32)
    do = n(1, 80, 1, 32)
    _, _, saved = delta_rule(**x, save=True)
    dg, dbeta = delta_rule_backward(saved, do)[3:5]
    for name_, grad in (("g", dg), ("beta", dbeta)):
        for t in (0, 37, 70):
            e, f = 0.02, []
            for sign in (1, -1):
                y = dict(x, **{name_: x[name_].clone()})
                y[name_][0, t, 0] += sign * e
                f.append((delta_rule(**y)[0].double() * do.double()).sum().item())
            want = (f[0] - f[1]) / (2 * e)
            assert abs(grad[0, t, 0].item() - want) <= 2e-3 * max(1.0, abs(want))


def test_captured_and_replayed():
    from recommenders.hip.delta import delta_rule, delta_rule_backward, delta_rule_step
    x, n = inputs(3, 100, 1, 2, 64, 64, torch.bfloat16)
    lens = torch.tensor([100, 64, 0], device="cuda")
    do = n(3, 100, 2, 64).bfloat16()
    state = n(3, 2, 64, 64)

    def whole():
        o, s, saved = delta_rule(**x, lens=lens, state=state, save=True)
        last = s.clone()
        step = delta_rule_step(**{n_: t[:, 0] for n_, t in x.items()}, state=last)
        return (o, s, step, last, *delta_rule_backward(saved, do))
    whole()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = whole()
    for k in range(3):
        x["v"].copy_(n(*x["v"].shape))
        lens.copy_(torch.tensor([99 - k, k, 70], device="cuda"))
        graph.replay()
        eager = whole()
        torch.cuda.synchronize()
        for a, b in zip(held, eager):
            assert torch.equal(a, b)


def test_changed_operand_is_refused():
    from recommenders.hip.delta import delta_rule, delta_rule_backward
    x, n = inputs(1, 4, 1, 1, 8, 8, torch.float32)
    o, s, saved = delta_rule(**x, save=True)
    x["k"].zero_()
    with pytest.raises(RuntimeError, match="in place"):
        delta_rule_backward(saved, o)


def test_no_positions():
    from recommenders.hip.delta import delta_rule, delta_rule_backward
    x, n = inputs(2, 0, 1, 1, 8, 8, torch.float32)
    state = n(2, 1, 8, 8)
    o, s, saved = delta_rule(**x, state=state, save=True)
    assert o.shape == (2, 0, 1, 8) and torch.equal(s, state)
    grads = delta_rule_backward(saved, o, state)
    assert torch.equal(grads[5], state)
