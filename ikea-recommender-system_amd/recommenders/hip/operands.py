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


def shares_memory(t, rows):
    """Whether the bytes of a tensor lie among `rows` (dimensions 0 and 1; rows of contiguous values, the rows apart): for an
    output that is written while t is still read."""
    if t is None or not t.numel() or not rows.numel():
        return False
    size, step = rows.element_size(), rows.stride(0) * rows.element_size()
    first, width = rows.data_ptr(), rows.shape[1] * size
    last = first + (rows.shape[0] - 1) * step + width
    each = t.element_size()
    # t as rows of its own: its first dimension, if any, and what a row spans
    n = t.shape[0] if t.dim() > 1 else 1
    lead = t.stride(0) * each if t.dim() > 1 else 0
    span = (sum((s - 1) * st for s, st in zip(t.shape[-1:], t.stride()[-1:])) + 1) * each
    lo, hi = t.data_ptr(), t.data_ptr() + (n - 1) * lead + span
    if hi <= first or last <= lo:
        return False
    if n > 1 and rows.shape[0] > 1 and lead == step:   # columns of one matrix: do they meet?
        off = (lo - first) % step
        return off < width or off + span > step
    return True


def layout(t):
    """What the checks of a tensor argument look at, apart from its address: calls with known layouts skip them."""
    return (t.shape, t.stride(), t.dtype, t.device) if isinstance(t, torch.Tensor) else None if t is None else type(t)


def version(t):
    """Changes with every write in place (None: not known, as for inference tensors)."""
    return None if t is None or t.is_inference() else t._version


def held(t):
    """What a backward pass that reads an operand again compares: its version, and where and how it lies."""
    return None if t is None else (version(t), t.data_ptr(), t.stride(), t.shape)


def wrote(t):
    """After a kernel wrote a caller's tensor in place: counted as a write, so that a backward pass that still needs the
    old values says so."""
    if not t.is_inference():
        torch._C._increment_version([t])


def stream(device):
    """The current stream of a device, as run() uses it."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def keep(device, since, *buffers):
    """Buffers that a call on stream `since` left are read on the current stream: if that is another one, their memory is not
    given away before it has passed."""
    if stream(device) != since:
        now = torch.cuda.current_stream(device)
        for t in buffers:
            if t is not None:
                t.record_stream(now)


class Plans(dict):
    """Checked argument layouts -> what a call needs of them.  Bounded: a program has few layouts; one that keeps making
    new ones starts over now and then."""

    def put(self, key, plan):
        if len(self) >= 512:
            self.clear()
        self[key] = plan
        return plan


def entry(name):
    """The C function of an entry point; use run() to call it."""
    return getattr(load_library(), name)


def run(fn, device, *args):
    """Launch on `device`'s current stream, with `device` current (it usually is already)."""
    index = device.index
    if index == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc < 0:
        raise RuntimeError(f"{fn.__name__} failed with status {rc}")
