"""Linear cross entropy over a large item vocabulary (csrc/linear_ce.hip): the
output layer and its loss in one operator, logits never kept, for bf16 / fp16
activations of every position of a batch.

    loss, saved = linear_ce(h, W, target, bias=b, save=True)      # (N,) fp32
    dh, dW, db = linear_ce_backward(saved, dloss)                 # dloss (N,) fp32: d total / d loss

h (N, D), W (V, D), both bf16 or both fp16; bias (V) fp32; target (N) int64.
Rows with a negative target are ignored: loss 0, gradient 0, no work.  A
target >= V gives NaN in the row's loss and in the gradients.  D is a multiple
of 8 up to 256, rows start at multiples of 16 bytes, N up to 2^24, V up to
2^31 − 4112.  Sums, the log-sum-exp and gradients are accumulated in fp32 and
rounded once on output (probabilities are rounded to the inputs' type for the
gradient products, the target's share is not).
At least one logit of a row has to lie above −2e38.  dh, dW have their
inputs' type, db is fp32 (None without a bias).  Nothing synchronises with the
host; calls can be captured in a graph.  Plain tensors in and out: no autograd
graph is built, whatever requires a gradient.
"""
from __future__ import annotations

import torch

from . import call, ptr
from .operands import TYPES, Plans, entry, fail, held, keep, layout, run, stream, stride, tensor, whole

_HALF = (torch.bfloat16, torch.float16)
_I64 = (torch.int64,)


class Saved:
    """What the backward pass needs of a forward call; W and bias are not copied and have to keep their values."""

    def __init__(self, plan, W, bias, buffer):
        self.plan, self.W, self.bias, self.buffer = plan, W, bias, buffer
        self.held, self.stream = (held(W), held(bias)), stream(plan.device)


_plans, _plans_back = Plans(), Plans()

N_MAX, V_MAX = 1 << 24, 0x7ffffff0 - 4096   # what the C entry takes: it counts in 32 bits


def _sizes(N, V, D):
    if D == 0 or D % 8 or D > 256:
        fail("h", f"a width that is a multiple of 8 up to 256 is expected, got {D}")
    if V == 0:
        fail("W", "has no rows")
    if V > V_MAX:
        fail("W", f"at most {V_MAX} rows are expected, got {V}")
    if N > N_MAX:
        fail("h", f"at most 2^24 rows are expected, got {N}")


class _Plan:
    def __init__(self, h, W, target, bias):
        tensor("h", h, (None, None), _HALF, align=16)
        self.N, self.D = N, D = h.shape
        tensor("W", W, (None, D), (h.dtype,), h.device, align=16)
        self.V = V = W.shape[0]
        _sizes(N, V, D)
        for name, t in (("h", h), ("W", W)):
            if t.shape[0] > 1 and not D <= t.stride(0) < 1 << 23:
                fail(name, f"rows overlap or lie too far apart: stride {t.stride(0)}")
        if not isinstance(target, torch.Tensor) or target.dim() != 1:
            fail("target", "a tensor of shape (N,) is expected")
        tensor("target", target[:, None], (N, 1), _I64, h.device)
        if bias is not None:
            whole("bias", bias, (V,), (torch.float32,), h.device)
        self.device, self.dtype, self.type = h.device, h.dtype, TYPES[h.dtype]
        self.ldh, self.ldw, self.st = stride(h, 0) or D, stride(W, 0) or D, stride(target, 0)
        if N:
            self.forward, self.backward = entry("rg_linear_ce_fwd"), entry("rg_linear_ce_bwd")
            self.saved = call("rg_linear_ce_saved_bytes", N, V, D)
            self.work = [call("rg_linear_ce_work_floats", N, V, D, k) for k in range(3)]


def _aligned(**tensors):
    for name, t in tensors.items():
        if t.data_ptr() & 15:
            fail(name, "has to start at a multiple of 16 bytes")


def linear_ce(h, W, target, bias=None, save=False):
    """Losses (N,) fp32 and, with save=True, what linear_ce_backward() takes (the forward then also sums dh)."""
    key = (layout(h), layout(W), layout(target), layout(bias)) if isinstance(h, torch.Tensor) else None
    p = _plans.get(key) or _plans.put(key, _Plan(h, W, target, bias))
    loss = torch.empty(p.N, dtype=torch.float32, device=p.device)
    buffer = None
    if p.N:
        if (h.data_ptr() | W.data_ptr()) & 15:
            _aligned(h=h, W=W)
        save = bool(save)
        buffer = torch.empty(p.saved, dtype=torch.uint8, device=p.device)
        work = torch.empty(p.work[save], dtype=torch.float32, device=p.device)
        run(p.forward, p.device, h.data_ptr(), p.ldh, W.data_ptr(), p.ldw, ptr(bias), target.data_ptr(), p.st, p.type, p.N,
            p.V, p.D, save, work.data_ptr(), buffer.data_ptr(), loss.data_ptr())
    return (loss, Saved(p, W, bias, buffer)) if save else loss


def linear_ce_backward(saved, dloss):
    """dh (N, D), dW (V, D), db (V) or None of sum(loss·dloss).  Can be called again with another dloss."""
    if not isinstance(saved, Saved):
        fail("saved", "what linear_ce(..., save=True) returned is expected")
    p, W, bias = saved.plan, saved.W, saved.bias
    if (held(W), held(bias)) != saved.held:
        raise RuntimeError("linear_ce_backward: W or bias was changed in place or given other memory since the forward call")
    key = (p.N, layout(dloss), p.device) if isinstance(dloss, torch.Tensor) else None
    step = _plans_back.get(key)
    if step is None:
        if not isinstance(dloss, torch.Tensor) or dloss.dim() != 1:
            fail("dloss", "a tensor of shape (N,) is expected")
        tensor("dloss", dloss[:, None], (p.N, 1), (torch.float32,), p.device)
        step = _plans_back.put(key, (stride(dloss, 0),))
    dh = torch.empty(p.N, p.D, dtype=p.dtype, device=p.device)
    dW = torch.empty(p.V, p.D, dtype=p.dtype, device=p.device)
    db = None if bias is None else torch.empty(p.V, dtype=torch.float32, device=p.device)
    if p.N == 0:
        dW.zero_()
        if db is not None:
            db.zero_()
    else:
        keep(p.device, saved.stream, saved.buffer)
        work = torch.empty(p.work[2], dtype=torch.float32, device=p.device)
        run(p.backward, p.device, W.data_ptr(), p.ldw, ptr(bias), dloss.data_ptr(), *step, p.type, p.N, p.V, p.D,
            saved.buffer.data_ptr(), work.data_ptr(), dh.data_ptr(), dW.data_ptr(), ptr(db))
    return dh, dW, db
