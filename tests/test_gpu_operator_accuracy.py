"""The operators at the accuracy that their fp32 results claim, which the tolerances of the other tests (worst cases, masks,
sizes) do not show.

4-bit scores.  A code enters as 16 + c and the offset 24 is taken off, both exactly.  (1) One-hot x: a single product s·(c − 8),
exact.  (2) x = 1 + 2^-10 + r·2^-23 with |r| < 128 needs all three of its planes, 1, 2^-10 and r·2^-23, and codes whose c − 8 sum
to zero in each group leave only the last one's: y = 2^-23·Σ s Σ r (c − 8).  Sums of the first plane are whole numbers
below 2^12, exact; those of the others start and stay below 24·G·2^-9, so each of at most 2·G + 4 roundings in a group is at most
2^-25 of twice that, and the K / G scaled additions add half a step of the result each.

Delta rule, fp32.  Sums of fp32 terms round independently: a product of depth d runs through d / 32 + 3 accumulations of three
to six plane products, whose roundings leave about 2^-24·sqrt((128 / 32 + 3)·6) / sqrt(3) = 4·2^-24 of its root mean square, and at
most six products follow one another: sqrt(6)·4·2^-24 < 10·2^-24.  The root mean square of an output's error is below
2^-20 of the output's.  With one plane fewer (16 bits a factor, 2^-18.8 a product) it is not.  dg is a difference of sums of pairs
(row sums less column sums), which cancel to a part of their size: 2^-18.
"""
import pytest
import torch

from test_gpu_delta import definition, inputs
from test_gpu_q4 import dequant, table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N,K,G", [(1001, 64, 32), (333, 192, 64), (70001, 128, 128), (65600, 256, 32), (257, 1024, 64)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_q4_every_code(N, K, G, dtype):
    from recommenders.hip.q4 import q4_scores
    codes, scales, g = table(N, K, G)
    y = q4_scores(torch.eye(K, device="cuda", dtype=dtype), codes, scales)
    assert torch.equal(y.double(), dequant(codes, scales).t())


@pytest.mark.parametrize("M,N,K,G", [(1, 1003, 128, 32), (5, 70001, 128, 64), (17, 515, 512, 128), (2, 66000, 256, 32)])
def test_q4_all_bits_of_x(M, N, K, G):
    from recommenders.hip.q4 import q4_scores
    g = torch.Generator(device="cuda").manual_seed(3)
    half = torch.randint(1, 16, (N, K // G, G // 2), generator=g, device="cuda")
    c = torch.cat([half, 16 - half], 2)                       # c − 8 and its negative
    c = c.gather(2, torch.rand(N, K // G, G, generator=g, device="cuda").argsort(2)).reshape(N, K)
    codes = (c[:, 0::2] | (c[:, 1::2] << 4)).to(torch.uint8)
    scales = (torch.rand(N, K // G, generator=g, device="cuda") + 0.5).bfloat16()
    r = torch.randint(-127, 128, (M, K), generator=g, device="cuda").double()
    x = 1 + 2.0 ** -10 + r * 2.0 ** -23
    assert torch.equal(x.float().double(), x)
    y = q4_scores(x.float(), codes, scales).double()
    w = dequant(codes, scales)
    ref = 2.0 ** -23 * (r @ w.t())
    s = scales.double().sum(1)
    room = (2 * G + 4) * 2.0 ** -25 * 2 * 24 * G * 2.0 ** -9 * s + (K // G) * 2.0 ** -24 * 2.0 ** -23 * (r.abs() @ w.abs().t())
    assert ((y - ref).abs() <= room).all()
    # and the room does not hide the last plane: without it the result is 0, off by |ref|
    assert (room < ref.abs()).double().mean() > 0.5


@pytest.mark.parametrize("case", [(64, 50, 2, 2, 64, 64, False), (3, 200, 1, 2, 128, 128, True), (2, 1100, 1, 1, 96, 48, True),
                                  (20, 32, 1, 1, 32, 128, True)], ids=str)
def test_delta_fp32(case):
    from recommenders.hip.delta import delta_rule, delta_rule_backward, delta_rule_step
    B, T, Hk, Hv, Dk, Dv, with_state = case
    x, n = inputs(B, T, Hk, Hv, Dk, Dv, torch.float32, seed=5)
    state = n(B, Hv, Dk, Dv) * 0.5 if with_state else None
    do, dstate = n(B, T, Hv, Dv), n(B, Hv, Dk, Dv) if with_state else None
    want = definition(x, Dk ** -0.5, None, state, do, dstate)
    o, final, saved = delta_rule(**x, state=state, save=True)
    got = (o, final, *delta_rule_backward(saved, do, dstate))

    def off(a, e):
        return ((a.double() - e).square().mean().sqrt() / e.square().mean().sqrt()).item()
    for what, a, e in zip(("o", "state", "dq", "dk", "dv", "dg", "dbeta", "dstate"), got, want):
        if a is not None:
            assert off(a, e) <= (2.0 ** -18 if what == "dg" else 2.0 ** -20), (what, off(a, e))
    if with_state:
        held = state.clone()
        first = {m: t[:, 0] for m, t in x.items()}
        o1 = delta_rule_step(**first, state=held)
        w1 = definition({m: t[:, :1] for m, t in x.items()}, Dk ** -0.5, None, state)
        assert off(o1, w1[0][:, 0]) <= 2.0 ** -20 and off(held, w1[1]) <= 2.0 ** -20
