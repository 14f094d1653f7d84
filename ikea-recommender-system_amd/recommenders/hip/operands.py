"""Argument checks shared by the operator modules (delta, linear_ce, q4):
they raise before anything is launched, ValueError for shapes, types, strides
and devices."""
from __future__ import annotations

import torch

from . import load_library

# element types as the C ABI numbers them
TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def fail(name, what):
    raise ValueError(f"{name}: {what}")


def tensor(name, t, shape, dtypes, device=None, align=1):
    """A device tensor of `shape` (None: any size) and one of `dtypes`; its last
    dimension contiguous and, with align > 1, every row starting at a multiple of
    `align` bytes.  Dimensions of one element may have any stride."""
    if not isinstance(t, torch.Tensor):
        fail(name, f"a tensor is expected, got {type(t).__name__}")
    if t.dim() != len(shape) or any(s is not None and s != n for s, n in zip(shape, t.shape)):
        want = tuple("any" if s is None else s for s in shape)
        fail(name, f"shape {want} is expected, got {tuple(t.shape)}")
    if t.dtype not in dtypes:
        fail(name, f"type {' or '.join(str(d) for d in dtypes)} is expected, got {t.dtype}")
    if t.device.type != "cuda":
        fail(name, f"a tensor on an MI355X (HIP device) is expected, got {t.device}")
    if device is not None and t.device != device:
        fail(name, f"on {t.device}, the other operands are on {device}")
    if t.dim() and t.shape[-1] > 1 and t.stride(-1) != 1:
        fail(name, f"the last dimension has stride {t.stride(-1)}: it has to be contiguous")
    if align > 1 and t.numel():
        es = t.element_size()
        if t.data_ptr() % align or any(st * es % align for n, st in zip(t.shape[:-1], t.stride()[:-1]) if n > 1):
            fail(name, f"rows have to start at multiples of {align} bytes, strides are {t.stride()}")
    return t


def whole(name, t, shape, dtypes, device=None):
    """tensor() that is contiguous as a whole."""
    tensor(name, t, shape, dtypes, device)
    if not t.is_contiguous():
        fail(name, f"has to be contiguous, strides are {t.stride()}")
    return t


def stride(t, dim):
    """Stride of `dim` in elements, 0 where the dimension has one element."""
    return 0 if t.shape[dim] == 1 else t.stride(dim)


class launch:
    """The device of `t` made current for the calls inside; the stream they use."""

    def __init__(self, t):
        load_library()
        self._guard = torch.cuda.device(t.device)
        self._device = t.device

    def __enter__(self):
        self._guard.__enter__()
        return torch.cuda.current_stream(self._device).cuda_stream

    def __exit__(self, *exc):
        return self._guard.__exit__(*exc)
