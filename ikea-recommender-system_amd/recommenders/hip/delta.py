"""Gated delta rule over sessions (csrc/delta.hip): a linear-attention encoder
beside the GRU, chunked for training and prefill, one token at a time for
serving.  Per value head, with a Dk x Dv state:

    S_t = exp(g_t)·S_{t-1} + beta_t·k_t (v_t − exp(g_t)·S_{t-1}ᵀ k_t)ᵀ,   o_t = scale·S_tᵀ q_t

q, k (B, T, Hk, Dk); v (B, T, Hv, Dv), Hv a multiple of Hk (value heads h of
key head h // (Hv / Hk)); g, beta (B, T, Hv) fp32, g <= 0 the log of the
decay (−inf resets).  q, k, v are fp32 or bf16; states and every sum are fp32.
Dk and Dv are multiples of 8 up to 128.  Strides are free as long as heads'
rows are contiguous and start at multiples of 16 bytes.

`lens` (B) int64 on the device: positions at or behind a row's length are not
read, leave the state as it is and get zeros (also as gradients); a length of
0 returns the initial state.  Nothing synchronises with the host; every call
can be captured in a graph.

    o, state, saved = delta_rule(q, k, v, g, beta, lens=lens, save=True)
    dq, dk, dv, dg, dbeta, _ = delta_rule_backward(saved, do)
    o = delta_rule_step(q1, k1, v1, g1, beta1, state)        # next click, state in place
"""
from __future__ import annotations

import ctypes as C

import torch

from . import call, ptr
from .operands import TYPES, fail, launch, stride, tensor, whole

_IO = (torch.float32, torch.bfloat16)


class Saved:
    """What the backward pass needs of a forward call: its operands (not copied: they have to keep their values) and the
    updates and chunk states it left."""

    def __init__(self, q, k, v, g, beta, scale, lens, state, U, S0):
        self.operands = (q, k, v, g, beta, lens, state)
        self.versions = [None if t is None else t._version for t in self.operands]
        self.scale, self.U, self.S0 = scale, U, S0


def _strides(*rows):
    flat = [s for r in rows for s in r]
    return (C.c_int64 * 18)(*flat, *([0] * (18 - len(flat))))


def _heads(q, k, v, lead):
    tensor("q", q, (*lead, None, None), _IO, align=16)
    Hk, Dk = q.shape[-2:]
    tensor("k", k, (*q.shape,), (q.dtype,), q.device, align=16)
    tensor("v", v, (*q.shape[:-2], None, None), (q.dtype,), q.device, align=16)
    Hv, Dv = v.shape[-2:]
    if Hk == 0 or Hv == 0 or Hv % Hk:
        fail("v", f"{Hv} value heads are no multiple of {Hk} key heads")
    for name, d in (("q", Dk), ("v", Dv)):
        if d == 0 or d % 8 or d > 128:
            fail(name, f"a head width that is a multiple of 8 up to 128 is expected, got {d}")
    return Hk, Hv, Dk, Dv


def _scalars(g, beta, shape, device):
    for name, t in (("g", g), ("beta", beta)):
        if not isinstance(t, torch.Tensor) or t.dim() != len(shape):
            fail(name, f"a tensor of shape {tuple(shape)} is expected")
        tensor(name, t[..., None], (*shape, 1), (torch.float32,), device)   # any strides


def delta_rule(q, k, v, g, beta, scale=None, lens=None, state=None, save=False):
    """-> o (B, T, Hv, Dv) of q's type, final state (B, Hv, Dk, Dv) fp32, and with save=True what
    delta_rule_backward() takes.  state: initial state (not written), zeros if None; scale: Dk ** -0.5 if None."""
    Hk, Hv, Dk, Dv = _heads(q, k, v, (None, None))
    B, T = q.shape[:2]
    _scalars(g, beta, (B, T, Hv), q.device)
    if lens is not None:
        whole("lens", lens, (B,), (torch.int64,), q.device)
    if state is not None:
        whole("state", state, (B, Hv, Dk, Dv), (torch.float32,), q.device)
        if state.data_ptr() % 16:
            fail("state", "has to start at a multiple of 16 bytes")
    scale = Dk ** -0.5 if scale is None else float(scale)
    o = torch.empty(B, T, Hv, Dv, dtype=q.dtype, device=q.device)
    final = torch.empty(B, Hv, Dk, Dv, dtype=torch.float32, device=q.device)
    U = S0 = None
    with launch(q) as st:
        if B == 0 or T == 0:
            final.copy_(state) if state is not None else final.zero_()
        else:
            if save:
                U = torch.empty(B, Hv, T, Dv, dtype=torch.float32, device=q.device)
                S0 = torch.empty(call("rg_delta_chunk_floats", B, T, Hv, Dk, Dv), dtype=torch.float32, device=q.device)
            call("rg_delta_fwd", ptr(q), ptr(k), ptr(v), ptr(g), ptr(beta),
                 _strides(*([stride(t, 0), stride(t, 1), stride(t, 2)] for t in (q, k, v, g, beta))), ptr(lens),
                 ptr(state), TYPES[q.dtype], B, T, Hk, Hv, Dk, Dv, scale, ptr(o), ptr(final), ptr(U),
                 None if S0 is None or not S0.numel() else ptr(S0), st)
    return (o, final, Saved(q, k, v, g, beta, scale, lens, state, U, S0)) if save else (o, final)


def delta_rule_backward(saved, do, dstate=None):
    """Gradients of sum(o·do) + sum(final·dstate): dq, dk, dv of their inputs' type, dg, dbeta fp32 (B, T, Hv), and
    dstate0 fp32 (None where the forward had no initial state).  Gradients of key heads are summed over their value
    heads in a fixed order.  Can be called again with other gradients."""
    if not isinstance(saved, Saved):
        fail("saved", "what delta_rule(..., save=True) returned is expected")
    q, k, v, g, beta, lens, state = saved.operands
    for t, at in zip(saved.operands, saved.versions):
        if t is not None and t._version != at:
            raise RuntimeError("delta_rule_backward: an operand of the forward call was changed in place since")
    B, T, Hk, Dk = q.shape
    Hv, Dv = v.shape[2:]
    tensor("do", do, (B, T, Hv, Dv), (q.dtype,), q.device, align=16)
    if dstate is not None:
        whole("dstate", dstate, (B, Hv, Dk, Dv), (torch.float32,), q.device)
        if dstate.data_ptr() % 16:
            fail("dstate", "has to start at a multiple of 16 bytes")
    new = lambda t: torch.empty(t.shape, dtype=t.dtype, device=t.device)  # noqa: E731
    dq, dk, dv = new(q), new(k), new(v)
    dg, dbeta = (torch.empty(B, T, Hv, dtype=torch.float32, device=q.device) for _ in range(2))
    dstate0 = None if state is None else new(state)
    with launch(q) as st:
        if B == 0 or T == 0:
            if dstate0 is not None:
                dstate0.copy_(dstate) if dstate is not None else dstate0.zero_()
        else:
            dX, dS = torch.empty_like(saved.U), torch.empty_like(saved.S0)
            there = dS.numel() > 0
            call("rg_delta_bwd", ptr(q), ptr(k), ptr(v), ptr(g), ptr(beta), ptr(do),
                 _strides(*([stride(t, 0), stride(t, 1), stride(t, 2)] for t in (q, k, v, g, beta, do))), ptr(lens),
                 ptr(state), ptr(dstate), ptr(saved.U), ptr(saved.S0) if there else None, TYPES[q.dtype], B, T, Hk, Hv,
                 Dk, Dv, saved.scale, ptr(dX), ptr(dS) if there else None, ptr(dq), ptr(dk), ptr(dv), ptr(dg),
                 ptr(dbeta), ptr(dstate0), st)
    return dq, dk, dv, dg, dbeta, dstate0


def delta_rule_step(q, k, v, g, beta, state, scale=None):
    """One token of every row: q, k (B, Hk, Dk), v (B, Hv, Dv), g, beta (B, Hv); state (B, Hv, Dk, Dv) fp32 is updated
    in place (its rows may lie apart, as in a larger pool, but not overlap).  -> o (B, Hv, Dv) of q's type."""
    Hk, Hv, Dk, Dv = _heads(q, k, v, (None,))
    B = q.shape[0]
    _scalars(g, beta, (B, Hv), q.device)
    tensor("state", state, (B, Hv, Dk, Dv), (torch.float32,), q.device, align=16)
    if B and not state[0].is_contiguous():
        fail("state", f"each row's (Hv, Dk, Dv) has to be contiguous, strides are {state.stride()}")
    if B > 1 and state.stride(0) < Hv * Dk * Dv:
        fail("state", f"rows overlap: stride {state.stride(0)}")
    scale = Dk ** -0.5 if scale is None else float(scale)
    o = torch.empty(B, Hv, Dv, dtype=q.dtype, device=q.device)
    if B:
        with launch(q) as st:
            call("rg_delta_step", ptr(q), ptr(k), ptr(v), ptr(g), ptr(beta),
                 _strides(*([stride(t, 0), 0, stride(t, 1)] for t in (q, k, v, g, beta))), TYPES[q.dtype], B, Hk, Hv, Dk,
                 Dv, scale, ptr(state), stride(state, 0), ptr(o), st)
    return o
