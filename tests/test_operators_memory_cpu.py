"""An output that shares memory with an operand is told from one that lies beside it."""
import itertools

import pytest
import torch


def bytes_of(t):
    at = set()
    for index in itertools.product(*map(range, t.shape)):
        first = t.data_ptr() + sum(i * s for i, s in zip(index, t.stride())) * t.element_size()
        at.update(range(first, first + t.element_size()))
    return at


def test_against_every_byte():
    from recommenders.hip.operands import shares_memory
    room = torch.zeros(600)
    small = room.view(torch.bfloat16)
    outs = [torch.as_strided(room, (m, n), (ld, 1), at) for m, n, ld, at in
            ((1, 7, 7, 100), (3, 7, 7, 100), (3, 7, 20, 100), (4, 18, 20, 95), (1, 50, 1, 60))]
    others = [torch.as_strided(room, (m, n), (ld, 1), at) for m, n, ld, at in
              ((1, 5, 5, 107), (3, 5, 20, 107), (3, 13, 20, 107), (3, 14, 20, 107), (3, 14, 20, 106), (2, 5, 20, 87), (5, 2, 20, 73),
               (2, 5, 20, 200), (5, 2, 20, 113), (5, 2, 20, 33))]
    others += [room[98:100], room[99:101], room[121:122], room[0:600], room[160:180], small[199:200], small[200:201], room[:0]]
    for out in outs:
        for t in others:
            meet = bool(bytes_of(out) & bytes_of(t))
            same_rows = t.dim() == 2 and t.shape[0] > 1 and out.shape[0] > 1 and t.stride(0) == out.stride(0)
            if meet:
                assert shares_memory(t, out)
            elif same_rows or out.shape[0] == 1 and (t.dim() == 1 or t.shape[0] == 1) or t.numel() == 0:
                assert not shares_memory(t, out), (out.shape, out.stride(), t.shape, t.stride())
    assert not shares_memory(None, outs[0])


def test_different_storages():
    from recommenders.hip.operands import shares_memory
    assert not shares_memory(torch.zeros(5, 4), torch.zeros(3, 9))


@pytest.mark.gpu
def test_q4_refuses_an_output_over_its_operands():
    from recommenders.hip.q4 import q4_scores
    g = torch.Generator(device="cuda").manual_seed(0)
    codes = torch.randint(0, 256, (50, 32), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.rand(50, 2, generator=g, device="cuda").bfloat16()
    room = torch.randn(3, 114, generator=g, device="cuda")
    x = room[:, 50:]
    want = q4_scores(x.clone(), codes, scales)
    with pytest.raises(ValueError, match="x"):
        q4_scores(x, codes, scales, out=room[:, 1:51])
    with pytest.raises(ValueError, match="bias"):
        q4_scores(x, codes, scales, bias=room[0, :50], out=room[:, :50])
    assert torch.equal(q4_scores(x, codes, scales, out=room[:, :50]), want)   # beside it is fine
