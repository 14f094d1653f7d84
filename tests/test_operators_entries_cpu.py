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
