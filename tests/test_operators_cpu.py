"""Operator modules (q4, linear_ce, delta): refusals, checked on the CPU."""
import pytest
import torch


def test_q4_refuses_before_the_device():
    from recommenders.hip.q4 import q4_pack, q4_scores
    W = torch.randn(10, 64)
    with pytest.raises(ValueError, match="HIP device"):
        q4_pack(W)
    with pytest.raises(ValueError, match="type"):
        q4_pack(W.double())
    with pytest.raises(ValueError, match="shape"):
        q4_pack(W[0])
    with pytest.raises(ValueError, match="HIP device"):
        q4_scores(W, torch.zeros(5, 32, dtype=torch.uint8), torch.zeros(5, 2, dtype=torch.bfloat16))


def test_q4_c_entry_refuses_more_rows_than_a_grid():
    from recommenders.hip import load_library
    one = 4096
    assert load_library().rg_q4_scores(one, 0, 64, one, one, None, 65535 * 16 + 1, 5, 64, 32, one, 5, None) == -3


def test_q4_c_entry_refusals():
    from recommenders.hip import load_library
    lib = load_library()
    one = 4096  # an aligned address that is never read: every call below is refused first
    assert lib.rg_q4_pack(one, 0, 64, 0, 64, 32, one, one, None) == -3
    assert lib.rg_q4_pack(one, 0, 64, 5, 64, 16, one, one, None) == -3
    assert lib.rg_q4_pack(one, 0, 63, 5, 64, 32, one, one, None) == -1
    assert lib.rg_q4_pack(one, 2, 64, 5, 64, 32, one, one, None) == -1
    assert lib.rg_q4_scores(one, 0, 64, one, one, None, 1, 5, 48, 32, one, 5, None) == -3
    assert lib.rg_q4_scores(one, 0, 2048, one, one, None, 1, 5, 2048, 32, one, 5, None) == -3
    assert lib.rg_q4_scores(one, 0, 64, one, one, None, 0, 5, 64, 32, one, 5, None) == -3
    assert lib.rg_q4_scores(one, 0, 64, one + 4, one, None, 1, 5, 64, 32, one, 5, None) == -1
    assert lib.rg_q4_scores(one, 0, 64, one, one, None, 1, 5, 64, 32, one, 4, None) == -1
    assert lib.rg_q4_scores(one, 2, 64, one, one, None, 1, 5, 64, 32, one, 5, None) == -1


def test_delta_refuses_before_the_device():
    from recommenders.hip.delta import delta_rule, delta_rule_backward, delta_rule_step
    x = torch.randn(2, 5, 1, 16)
    g = torch.zeros(2, 5, 1)
    with pytest.raises(ValueError, match="HIP device"):
        delta_rule(x, x, x, g, g)
    with pytest.raises(ValueError, match="type"):
        delta_rule(x.half(), x, x, g, g)
    with pytest.raises(ValueError, match="HIP device"):
        delta_rule_step(x[:, 0], x[:, 0], x[:, 0], g[:, 0], g[:, 0], torch.zeros(2, 1, 16, 16))
    with pytest.raises(ValueError, match="saved"):
        delta_rule_backward(None, x)


def test_delta_c_entry_refusals():
    import ctypes as C
    from recommenders.hip import load_library
    lib = load_library()
    p, s = 4096, (C.c_int64 * 18)(*[64] * 18)   # an aligned address that is never read: each call is refused first

    def fwd(type=0, B=1, T=5, Hk=1, Hv=1, Dk=16, Dv=16, q=p, o=p, strides=s, U=None, S0=None, trans=None, local=None):
        return lib.rg_delta_fwd(q, p, p, p, p, strides, None, None, type, B, T, Hk, Hv, Dk, Dv, 1.0, o, p, U, S0, trans, local, None)
    assert fwd(type=2) == -1 and fwd(o=None) == -1 and fwd(q=None) == -1 and fwd(strides=None) == -1
    assert fwd(B=0) == -3 and fwd(T=0) == -3 and fwd(Hk=2, Hv=3) == -3
    assert fwd(Dk=12) == -3 and fwd(Dk=136) == -3 and fwd(Dv=0) == -3 and fwd(T=65536 * 32) == -3
    assert fwd(q=p + 4) == -1 and fwd(strides=(C.c_int64 * 18)(*[63] * 18)) == -1
    assert fwd(T=33, U=p) == -1                 # the chunk states' room is missing
    assert lib.rg_delta_segments(1, 4000, 1, 16, 16) > 1 and fwd(T=4000) == -1 and fwd(T=4000, trans=p) == -1   # the segments' room is missing

    def bwd(do=p, dX=p, T=5, dS=None, state0=None):
        return lib.rg_delta_bwd(p, p, p, p, p, do, s, None, state0, None, p, None, None, 0, 1, T, 1, 1, 16, 16, 1.0, dX, dS, None, p, p, p,
                                p, p, None, None)
    assert bwd(do=None) == -1 and bwd(dX=None) == -1 and bwd(T=65) == -1 and bwd(state0=p + 4) == -1

    def step(stride=256, state=p, B=2):
        return lib.rg_delta_step(p, p, p, p, p, s, 0, B, 1, 1, 16, 16, 1.0, state, stride, p, None)
    assert step(stride=255) == -1 and step(stride=252) == -1 and step(state=p + 4) == -1 and step(B=0) == -3
    assert fwd(B=1 << 24) == -3   # 256 threads for each would pass a grid's 2^32
    assert lib.rg_delta_chunk_floats(2, 32, 3, 8, 8) == 0 and lib.rg_delta_chunk_floats(2, 33, 3, 8, 16) == 2 * 3 * 8 * 16


def test_linear_ce_refuses_before_the_device():
    from recommenders.hip.linear_ce import linear_ce, linear_ce_backward
    h, W, t = torch.randn(4, 16).bfloat16(), torch.randn(9, 16).bfloat16(), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="HIP device"):
        linear_ce(h, W, t)
    with pytest.raises(ValueError, match="type"):
        linear_ce(h.float(), W, t)
    with pytest.raises(ValueError, match="saved"):
        linear_ce_backward(None, t)


def test_linear_ce_c_entry_refusals():
    from recommenders.hip import load_library
    lib = load_library()
    p = 4096   # an aligned address that is never read: every call below is refused first

    def fwd(h=p, ldh=16, W=p, ldw=16, t=p, type=1, N=4, V=9, D=16, work=p, saved=p, loss=p):
        return lib.rg_linear_ce_fwd(h, ldh, W, ldw, None, t, 1, type, N, V, D, 1, work, saved, loss, None)
    assert fwd(type=0) == -1 and fwd(h=None) == -1 and fwd(h=p + 8) == -1 and fwd(ldh=15) == -1 and fwd(ldw=20) == -1
    assert fwd(ldw=1 << 23) == -1 and fwd(t=None) == -1 and fwd(work=p + 4) == -1 and fwd(loss=None) == -1
    assert fwd(N=0) == -3 and fwd(V=0) == -3 and fwd(D=12) == -3 and fwd(D=264, ldh=264, ldw=264) == -3
    assert fwd(N=(1 << 24) + 1) == -3

    def bwd(W=p, g=p, dh=p, dW=p, db=None, D=16):
        return lib.rg_linear_ce_bwd(W, 16, None, g, 1, 1, 4, 9, D, p, p, dh, dW, db, None)
    assert bwd(W=None) == -1 and bwd(g=None) == -1 and bwd(dh=None) == -1 and bwd(dW=p + 2) == -1 and bwd(db=p) == -1
    assert bwd(D=0) == -3


@pytest.mark.parametrize("N,V,D", [(1, 1, 8), (64, 10001, 32), (4096, 1000001, 128), (13111, 78341, 256), (8192, 5000001, 256),
                                   (1 << 24, 100, 64)])
def test_linear_ce_partial_results_stay_small(N, V, D):
    """Splits are bounded: partial sums of a pass take at most 2^28 values beyond one set of results."""
    from recommenders.hip import load_library
    lib = load_library()
    for k in (1, 2):
        assert 0 < lib.rg_linear_ce_work_floats(N, V, D, k) <= (1 << 28) + 4 * (N + 512) * 256 + 4 * V * (D + 1) + 4 * 512 * N
