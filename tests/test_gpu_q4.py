"""Scores from a 4-bit item table (csrc/q4.hip) against 64-bit products of the
same codes.

Tolerance: a code enters the matrix products as 16 + c and the offset 24 is
taken off again, so the running sums of a group of G products are at most
31·Σ|x| and every fp32 rounding (G products, three planes of x, K / G scaled
additions) is at most 2^-24 of that: |error| <= 2^-24·(3·G + K / G + 4)·31·Σ_k |x_k| s_k, a bound no input
exceeds; a wrong code, scale or row is off by far more.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu


def dequant(codes, scales):
    c = torch.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1).double() - 8
    return c * scales.double().repeat_interleave(c.shape[1] // scales.shape[1], 1)


def table(N, K, G, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 256, (N, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = (torch.rand(N, K // G, generator=g, device="cuda") * 0.1 + 0.01).bfloat16()
    return codes, scales, g


def check(y, x, codes, scales, bias, G):
    K = x.shape[1]
    ref = x.double() @ dequant(codes, scales).t()
    if bias is not None:
        ref = ref + bias.double()
    s = scales.double().repeat_interleave(G, 1)
    room = 2.0 ** -24 * ((3 * G + K // G + 4) * 31 * (x.double().abs() @ s.t()) + 2 * ref.abs()) + 1e-30
    assert y.dtype == torch.float32 and y.shape == ref.shape
    assert ((y.double() - ref).abs() <= room).all()


@pytest.mark.parametrize("M,N,K,G", [(1, 1, 32, 32), (1, 15, 64, 64), (3, 17, 128, 128), (16, 1000, 96, 32),
                                     (17, 33, 192, 64), (5, 4099, 1024, 32), (2, 70001, 256, 128), (40, 515, 640, 128),
                                     (1, 300001, 128, 32), (16, 299, 1024, 64),
                                     (17, 66001, 192, 64), (3, 80003, 96, 32), (1, 70000, 32, 32), (18, 65553, 512, 128)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scores(M, N, K, G, dtype):
    from recommenders.hip.q4 import q4_scores
    codes, scales, g = table(N, K, G)
    x = torch.randn(M, K, generator=g, device="cuda").to(dtype)
    bias = torch.randn(N, generator=g, device="cuda") if N % 2 else None
    check(q4_scores(x, codes, scales, bias), x, codes, scales, bias, G)


def test_wide_range_of_x():
    """fp32 x of very different sizes enters with all its bits."""
    from recommenders.hip.q4 import q4_scores
    codes, scales, g = table(501, 128, 32)
    x = torch.randn(4, 128, generator=g, device="cuda") * torch.logspace(-12, 12, 128, device="cuda")
    check(q4_scores(x, codes, scales), x, codes, scales, None, 32)


def test_strided_rows_and_untouched_gaps():
    from recommenders.hip.q4 import q4_scores
    codes, scales, g = table(1003, 64, 32)
    x = torch.randn(6, 100, generator=g, device="cuda")[::2, 3:67]
    out = torch.full((3, 1111), 7.0, device="cuda")
    y = q4_scores(x, codes, scales, out=out[:, 5:1008])
    assert y.data_ptr() == out[:, 5:].data_ptr()
    check(y, x, codes, scales, None, 32)
    assert (out[:, :5] == 7).all() and (out[:, 1008:] == 7).all()


def test_no_rows_or_items():
    from recommenders.hip.q4 import q4_pack, q4_scores
    codes, scales, g = table(10, 64, 32)
    assert q4_scores(torch.empty(0, 64, device="cuda"), codes, scales).shape == (0, 10)
    c, s = q4_pack(torch.empty(0, 64, device="cuda"))
    assert q4_scores(torch.randn(2, 64, device="cuda"), c, s).shape == (2, 0)


@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_pack(G, dtype):
    """codes and scales are the documented formula's, and a weight moves by half a scale step (and the scale's rounding)."""
    from recommenders.hip.q4 import q4_pack
    g = torch.Generator(device="cuda").manual_seed(3)
    W = (torch.randn(1001, 2 * G + 5, generator=g, device="cuda") * 0.05).to(dtype)[:, 5:]
    W[7] = 0
    codes, scales = q4_pack(W, G)
    blocks = W.float().unflatten(1, (2, G))
    s = (blocks.abs().amax(-1) / 7).bfloat16()
    assert torch.equal(scales, s)
    c = ((blocks / torch.where(s > 0, s, 1).float()[..., None]).round() + 8).clamp(0, 15).to(torch.uint8).flatten(1)
    assert torch.equal(codes, c[:, 0::2] | (c[:, 1::2] << 4))
    off = (dequant(codes, scales) - W.double()).abs()
    # half a step, and max|w| itself may lie 2^-8 beyond 7 scale steps where the scale was rounded down
    assert (off <= (0.5 + 7 * 2.0 ** -8) * s.double().repeat_interleave(G, 1)).all()


def test_captured_and_on_another_stream():
    from recommenders.hip.q4 import q4_scores
    codes, scales, g = table(2003, 128, 32)
    x = torch.randn(2, 128, generator=g, device="cuda")
    want = q4_scores(x, codes, scales)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(q4_scores(x, codes, scales), want)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    held = x.clone()
    with torch.cuda.graph(graph):
        y = q4_scores(held, codes, scales)
    for k in range(3):
        held.copy_(torch.randn(2, 128, generator=g, device="cuda"))
        graph.replay()
        eager = q4_scores(held, codes, scales)
        torch.cuda.synchronize()
        assert torch.equal(y, eager)


def test_scores_of_a_trained_head():
    """The model's output layer packed once: scores of its own hidden rows rank as the dequantised table's do."""
    from recommenders.hip.q4 import q4_pack, q4_scores
    from recommenders.models.GRU4Rec.model import GRU4Rec_trainer
    t = GRU4Rec_trainer(hidden_dim=64, embedding_dim=64, gru_layers=1, train_pad_embed=True, use_packed_seq=True,
                        learning_rate=0.01, item_num=500, state_size=10, action_dim=500, device="cuda")
    sd = t.gru_model.state_dict()
    W, b = sd["output.weight"].cuda(), sd["output.bias"].cuda()
    codes, scales = q4_pack(W, 32)
    h = torch.tanh(torch.randn(3, 64, device="cuda"))
    check(q4_scores(h, codes, scales, b), h, codes, scales, b, 32)


def test_rows_that_overlap_are_refused():
    """A row repeated by a stride of 0 is not K apart from itself: refused, not read as if it were."""
    from recommenders.hip.q4 import q4_pack, q4_scores
    codes, scales, g = table(20, 64, 32)
    x = torch.randn(1, 64, generator=g, device="cuda")
    for bad in (x.expand(5, 64), torch.as_strided(x, (2, 32), (16, 1))):
        with pytest.raises(ValueError, match="overlap"):
            q4_scores(bad, *q4_pack(torch.randn(9, bad.shape[1], device="cuda")))
        with pytest.raises(ValueError, match="overlap"):
            q4_pack(bad)
