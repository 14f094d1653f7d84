"""Scores from a 4-bit table for x at the ends of fp32's range: infinities, NaN
and values whose products with the codes pass 2^128 before the scale brings
them back.  The definition is Σ_k x·w with w = scale·(code − 8), an exact fp32
value; a row is compared in 64 bits, with the bound of test_gpu_q4 and the same
rounding 2^-24·(K + 2)·Σ|x w| of a plain fp32 sum beside it.
"""
import pytest
import torch

from test_gpu_q4 import dequant, table

pytestmark = pytest.mark.gpu


def special(K, dtype):
    """Rows by name; the first and the last are ordinary."""
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(10, K, generator=g, device="cuda")
    x[1, 5] = float("inf")
    x[2, K - 1] = -float("inf")
    x[3, 0] = float("nan")
    x[4] *= 1e36
    x[5, 7] = torch.finfo(dtype).max
    x[6] *= 2.0 ** 100
    x[7, 3], x[7, 4] = float("inf"), -float("inf")
    x[8] *= 2.0 ** 95
    return x.to(dtype)


@pytest.mark.parametrize("N,K,G", [(333, 64, 32), (500, 192, 64), (257, 1024, 128), (66001, 128, 32), (65601, 256, 128)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_rows_at_the_ends_of_the_range(N, K, G, dtype):
    from recommenders.hip.q4 import q4_scores
    codes, scales, g = table(N, K, G)
    bias = torch.randn(N, generator=g, device="cuda")
    x = special(K, dtype)
    x = torch.cat([x, x.flip(0)], 0)          # 20 rows: past the first 16
    y = q4_scores(x, codes, scales, bias)
    w = dequant(codes, scales)
    s = scales.double().repeat_interleave(G, 1)
    for m in range(20):
        ref = (x[m].double() * w).sum(1) + bias.double()
        terms = (x[m].double() * w).abs().sum(1)
        room = 2.0 ** -24 * (((3 * G + K // G + 4) * 31 * (x[m].double().abs() * s).sum(1)) + (K + 2) * terms + 2 * ref.abs())
        finite = torch.isfinite(x[m]).all()
        got = y[m].double()
        if finite:
            inside = ref.abs() + room < torch.finfo(torch.float32).max
            assert torch.isfinite(got[inside]).all() and ((got - ref).abs() <= room)[inside].all(), m
        else:
            assert torch.equal(got.isnan(), ref.isnan()), m
            assert torch.equal(got[~ref.isnan()], ref[~ref.isnan()]), m


def test_one_row_and_a_graph():
    """One session, an infinity among its values that comes and goes between replays."""
    from recommenders.hip.q4 import q4_scores
    codes, scales, g = table(1003, 64, 32)
    x = torch.randn(1, 64, generator=g, device="cuda")
    q4_scores(x, codes, scales)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = q4_scores(x, codes, scales)
    w = dequant(codes, scales)
    for k, value in enumerate((1.0, float("inf"), 2.0, -float("inf"), 3e38)):
        x[0, 7] = value
        graph.replay()
        eager = q4_scores(x, codes, scales)
        torch.cuda.synchronize()
        assert torch.equal(y.nan_to_num(7.0, 1e30, -1e30), eager.nan_to_num(7.0, 1e30, -1e30))
        if abs(value) == float("inf"):
            assert torch.equal(y[0].isnan(), w[:, 7] == 0)
            assert torch.equal(y[0].isinf(), w[:, 7] != 0)
        else:
            assert torch.isfinite(y).all()
