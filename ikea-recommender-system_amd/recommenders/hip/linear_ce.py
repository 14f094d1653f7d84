"""Linear cross entropy over a large item vocabulary (csrc/linear_ce.hip): the
output layer and its loss in one operator, logits never kept, for bf16 / fp16
activations of every position of a batch.

    loss, saved = linear_ce(h, W, target, bias=b, save=True)      # (N,) fp32
    dh, dW, db = linear_ce_backward(saved, dloss)                 # dloss (N,) fp32: d total / d loss

h (N, D), W (V, D), both bf16 or both fp16; bias (V) fp32; target (N) int64.
Rows with a negative target are ignored: loss 0, gradient 0, no work.  A
target >= V gives NaN in the row's loss and in the gradients.  D is a multiple
of 8 up to 256, rows start at multiples of 16 bytes, N up to 2^24.  Sums, the
log-sum-exp and gradients are accumulated in fp32 and rounded once on output
(probabilities are rounded to the inputs' type for the gradient products).
At least one logit of a row has to lie above −2e38.  dh, dW have their
inputs' type, db is fp32 (None without a bias).  Nothing synchronises with the
host; calls can be captured in a graph.
"""
from __future__ import annotations

import torch

from . import call, ptr
from .operands import TYPES, fail, launch, stride, tensor, whole

_HALF = (torch.bfloat16, torch.float16)
_I64 = (torch.int64,)


class Saved:
    """What the backward pass needs of a forward call; W and bias are not copied and have to keep their values."""

    def __init__(self, h, W, bias, buffer):
        self.shape, self.W, self.bias, self.buffer = h.shape, W, bias, buffer
        self.versions = (W._version, None if bias is None else bias._version)


def linear_ce(h, W, target, bias=None, save=False):
    """Losses (N,) fp32 and, with save=True, what linear_ce_backward() takes (the forward then also sums dh)."""
    tensor("h", h, (None, None), _HALF, align=16)
    N, D = h.shape
    tensor("W", W, (None, D), (h.dtype,), h.device, align=16)
    V = W.shape[0]
    if D == 0 or D % 8 or D > 256:
        fail("h", f"a width that is a multiple of 8 up to 256 is expected, got {D}")
    if V == 0:
        fail("W", "has no rows")
    if N > 1 << 24:
        fail("h", f"at most 2^24 rows are expected, got {N}")
    for name, t in (("h", h), ("W", W)):
        if t.shape[0] > 1 and not D <= t.stride(0) < 1 << 23:
            fail(name, f"rows overlap or lie too far apart: stride {t.stride(0)}")
    if not isinstance(target, torch.Tensor) or target.dim() != 1:
        fail("target", "a tensor of shape (N,) is expected")
    tensor("target", target[:, None], (N, 1), _I64, h.device)
    if bias is not None:
        whole("bias", bias, (V,), (torch.float32,), h.device)
    loss = torch.empty(N, dtype=torch.float32, device=h.device)
    buffer = None
    if N:
        with launch(h) as st:
            buffer = torch.empty(call("rg_linear_ce_saved_bytes", N, V, D), dtype=torch.uint8, device=h.device)
            work = torch.empty(call("rg_linear_ce_work_floats", N, V, D, int(save)), dtype=torch.float32, device=h.device)
            call("rg_linear_ce_fwd", ptr(h), stride(h, 0) or D, ptr(W), stride(W, 0) or D, ptr(bias), ptr(target),
                 stride(target, 0), TYPES[h.dtype], N, V, D, int(save), ptr(work), ptr(buffer), ptr(loss), st)
    return (loss, Saved(h, W, bias, buffer)) if save else loss


def linear_ce_backward(saved, dloss):
    """dh (N, D), dW (V, D), db (V) or None of sum(loss·dloss).  Can be called again with another dloss."""
    if not isinstance(saved, Saved):
        fail("saved", "what linear_ce(..., save=True) returned is expected")
    W, bias, (N, D) = saved.W, saved.bias, saved.shape
    if (W._version, None if bias is None else bias._version) != saved.versions:
        raise RuntimeError("linear_ce_backward: W or bias was changed in place since the forward call")
    V = W.shape[0]
    if not isinstance(dloss, torch.Tensor) or dloss.dim() != 1:
        fail("dloss", "a tensor of shape (N,) is expected")
    tensor("dloss", dloss[:, None], (N, 1), (torch.float32,), W.device)
    dh = torch.empty(N, D, dtype=W.dtype, device=W.device)
    dW = torch.empty(V, D, dtype=W.dtype, device=W.device)
    db = None if bias is None else torch.empty(V, dtype=torch.float32, device=W.device)
    with launch(W) as st:
        if N == 0:
            dW.zero_()
            if db is not None:
                db.zero_()
        else:
            work = torch.empty(call("rg_linear_ce_work_floats", N, V, D, 2), dtype=torch.float32, device=W.device)
            call("rg_linear_ce_bwd", ptr(W), stride(W, 0) or D, ptr(bias), ptr(dloss), stride(dloss, 0), TYPES[W.dtype],
                 N, V, D, ptr(saved.buffer), ptr(work), ptr(dh), ptr(dW), ptr(db), st)
    return dh, dW, db
