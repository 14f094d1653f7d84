"""The delta rule, the linear cross entropy and the 4-bit scores together, as a
program uses them: a training step over padded sessions with a next-item loss
at every position, and serving (a prefill of histories, then one click after the
other, scored against the packed table).  Each operator's results are
checked against 64 bits on what the operator before it handed over, with the
tolerances derived beside the operators' own tests, so that nothing is lost or
exchanged on the way.
"""
import pytest
import torch

from test_gpu_delta import definition, near
from test_gpu_linear_ce import check as check_ce
from test_gpu_q4 import check as check_q4

pytestmark = pytest.mark.gpu

HK, HV, DK, DV, V = 2, 4, 32, 16, 3001


def model(seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    D = HV * DV
    weights = {"E": n(V, D), "q": n(D, HK * DK) / 8, "k": n(D, HK * DK) / 8, "v": n(D, HV * DV) / 8, "g": n(D, HV) / 8,
               "beta": n(D, HV) / 8}
    return weights, (n(V, D) / 4).bfloat16(), n(V) / 4, g


def project(w, x):
    lead = x.shape[:-1]
    unit = lambda t: t / t.norm(dim=-1, keepdim=True)  # noqa: E731
    return (unit((x @ w["q"]).view(*lead, HK, DK)), unit((x @ w["k"]).view(*lead, HK, DK)), (x @ w["v"]).view(*lead, HV, DV),
            -torch.nn.functional.softplus(x @ w["g"]), torch.sigmoid(x @ w["beta"]))


def test_training_step():
    from recommenders.hip.delta import delta_rule, delta_rule_backward
    from recommenders.hip.linear_ce import linear_ce, linear_ce_backward
    w, W, b, g = model()
    w = {n: t.requires_grad_() for n, t in w.items()}
    B, T = 9, 70
    lens = torch.tensor([70, 0, 1, 33, 64, 2, 69, 32, 5], device="cuda")
    items = torch.randint(0, V, (B, T + 1), generator=g, device="cuda")
    on = torch.arange(T, device="cuda")[None] < lens[:, None]
    target = torch.where(on, items[:, 1:], -1).flatten()
    x = w["E"][items[:, :-1]]
    qkvgb = project(w, x)
    held = [t.detach() for t in qkvgb]
    o, final, saved = delta_rule(*held, lens=lens, save=True)
    h = o.flatten(2).flatten(0, 1).bfloat16()
    loss, kept = linear_ce(h, W, target, bias=b, save=True)
    dloss = on.flatten().float() / on.sum()
    dh, dW, db = linear_ce_backward(kept, dloss)
    check_ce(h, W, b, target, loss, dloss, (dh, dW, db))
    do = dh.float().view(B, T, HV, DV)
    grads = delta_rule_backward(saved, do)
    names = ["q", "k", "v", "g", "beta"]
    want = definition(dict(zip(names, held)), DK ** -0.5, lens, None, do)
    near(o, want[0], "o")
    near(final, want[1], "final")
    for n, a, e in zip(names, grads, want[2:]):
        near(a, e, "d" + n)
    # the embedding's gradient: nothing comes from behind a session's end
    torch.autograd.backward(qkvgb, list(grads[:5]))
    used = torch.zeros(V, dtype=torch.bool, device="cuda")
    used[items[:, :-1][on]] = True
    assert torch.isfinite(w["E"].grad).all() and (w["E"].grad[~used] == 0).all()
    assert (w["E"].grad[used].abs().amax(1) > 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_serving(dtype):
    """Histories of unlike lengths prefilled in one call, then six clicks, each one replay of a captured step and scoring;
    the state and every score are those of the eager calls, and those of the whole sequence at once in 64 bits."""
    from recommenders.hip.delta import delta_rule, delta_rule_step
    from recommenders.hip.q4 import q4_pack, q4_scores
    w, W, b, g = model(1)
    codes, scales = q4_pack(W, 32)
    B, T, clicks = 5, 100, 6
    lens = torch.tensor([100, 0, 1, 37, 64], device="cuda")
    x = w["E"][torch.randint(0, V, (B, T + clicks), generator=g, device="cuda")]
    whole = [t.to(dtype) if i < 3 else t for i, t in enumerate(project(w, x))]
    _, state = delta_rule(*[t[:, :T] for t in whole], lens=lens)
    held, out = [t[:, 0].clone() for t in whole], torch.empty(B, V, device="cuda")
    live = state.clone()

    def click(s):
        o = delta_rule_step(*held, s)
        return o, q4_scores(o.flatten(1), codes, scales, bias=b, out=out)

    click(live.clone())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, y = click(live)
    live.copy_(state)
    for c in range(clicks):
        for t, a in zip(held, whole):
            t.copy_(a[:, T + c])
        graph.replay()
        seen, served = o.clone(), y.clone()
        o2, y2 = click(state)
        torch.cuda.synchronize()
        assert torch.equal(seen, o2) and torch.equal(served, y2) and torch.equal(live, state)
        check_q4(served, seen.flatten(1), codes, scales, b, 32)
        # the same from the start: each history with its clicks put behind its end
        for r in range(B):
            n = int(lens[r])
            row = {m: torch.cat([a[r:r + 1, :n], a[r:r + 1, T:T + c + 1]], 1)
                   for m, a in zip(["q", "k", "v", "g", "beta"], whole)}
            at, final = definition(row, DK ** -0.5, None, None)
            near(seen[r], at[0, -1], "o" + (" bf16" if dtype == torch.bfloat16 else ""))
            near(state[r], final[0], "state")


def test_a_step_in_place_is_a_change():
    """A state that a training call still needs and that a step has written since."""
    from recommenders.hip.delta import delta_rule, delta_rule_backward, delta_rule_step
    w, W, b, g = model(2)
    x = w["E"][torch.randint(0, V, (2, 9), generator=g, device="cuda")]
    q, k, v, a, beta = project(w, x)
    state = torch.zeros(2, HV, DK, DV, device="cuda")
    o, final, saved = delta_rule(q, k, v, a, beta, state=state, save=True)
    delta_rule_step(q[:, 0], k[:, 0], v[:, 0], a[:, 0], beta[:, 0], state)
    with pytest.raises(RuntimeError, match="in place"):
        delta_rule_backward(saved, o)


def test_two_streams_at_once():
    """Two training steps and two scorings side by side, each on a stream of its own: nothing is shared between calls."""
    from recommenders.hip.delta import delta_rule, delta_rule_backward
    from recommenders.hip.linear_ce import linear_ce, linear_ce_backward
    from recommenders.hip.q4 import q4_pack, q4_scores
    w, W, b, g = model(3)
    codes, scales = q4_pack(W, 64)
    cases = []
    for B, T in ((40, 90), (3, 1000)):
        items = torch.randint(0, V, (B, T), generator=g, device="cuda")
        cases.append(([t.contiguous() for t in project(w, w["E"][items])], items.flatten()))

    def step(x, target):
        o, s, saved = delta_rule(*x, save=True)
        h = o.flatten(2).flatten(0, 1).bfloat16()
        loss, kept = linear_ce(h, W, target, bias=b, save=True)
        grads = linear_ce_backward(kept, torch.full_like(loss, 1 / len(loss)))
        back = delta_rule_backward(saved, grads[0].float().view(o.shape))
        return [o, s, loss, *grads, *back[:5], q4_scores(h[:7], codes, scales, bias=b)]

    want = [step(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(3):
        got = []
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        for s, c in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(step(*c))
        torch.cuda.synchronize()
        for a, e in zip(got, want):
            for y, z in zip(a, e):
                assert torch.equal(y, z)
