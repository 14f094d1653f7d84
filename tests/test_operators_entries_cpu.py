"""More refusals of the delta rule's C entries: each call is refused before anything is launched or read."""
import ctypes as C

P = 4096   # an aligned address that is never read


def strides(**rows):
    flat = []
    for n in ("q", "k", "v", "g", "beta", "do"):
        flat += rows.get(n, (64, 64, 64))
    return (C.c_int64 * 18)(*flat)


def backward(s, q=P, v=P, dq=P, dk=P, B=1, T=5, Hk=1, Hv=1, Dk=16, Dv=16, S0=None, dS=None):
    from recommenders.hip import load_library
    return load_library().rg_delta_bwd(q, P, v, P, P, P, s, None, None, None, P, S0, None, 0, B, T, Hk, Hv, Dk, Dv, 1.0, P, dS, None,
                                       dq, dk, P, P, P, None, None)


def test_backward_refuses_misaligned_values():
    """The backward kernel reads v, and writes dq and dk, in pieces of 16 bytes."""
    assert backward(strides(), v=P + 4) == -1
    assert backward(strides(v=(64, 66, 64))) == -1
    assert backward(strides(), dq=P + 8) == -1 and backward(strides(), dk=P + 4) == -1


def test_more_heads_than_a_buffer_reaches():
    """Outputs are contiguous, so their positions lie Hv·Dv apart, and 32 of them in bytes have to stay below 2 GB; inputs with
    heads before positions may pass their own check."""
    import pytest
    from recommenders.hip import load_library
    from recommenders.hip.delta import _sizes
    heads = 1 << 17   # of width 64: 2^23 values

    def forward(T, Hk, Hv, Dk, Dv):
        return load_library().rg_delta_fwd(P, P, P, P, P, strides(), None, None, 0, 1, T, Hk, Hv, Dk, Dv, 1.0, P, P, None, None, P, P, None)
    for T in (1, 5, 40):
        assert forward(T, 1, heads, 64, 64) == -3 and forward(T, heads, heads, 64, 8) == -3
        assert backward(strides(), T=T, Hv=heads, Dk=64, Dv=64, S0=P, dS=P) == -3
        for shape in ((1, heads, 64, 64), (heads, heads, 64, 8)):
            with pytest.raises(ValueError, match="2\\^23"):
                _sizes(1, T, *shape, 2)
    _sizes(1, 40, 1, heads - 1, 64, 64, 2)
    _sizes(1, 1, 1, heads, 64, 64, 1)
