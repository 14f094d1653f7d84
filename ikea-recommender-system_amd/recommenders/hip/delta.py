"""Gated delta rule over sessions (csrc/delta.hip): a linear-attention encoder
beside the GRU, chunked for training and prefill, one token at a time for
serving.  Per value head, with a Dk x Dv state:

    S_t = exp(g_t)·S_{t-1} + beta_t·k_t (v_t − exp(g_t)·S_{t-1}ᵀ k_t)ᵀ,   o_t = scale·S_tᵀ q_t

q, k (B, T, Hk, Dk); v (B, T, Hv, Dv), Hv a multiple of Hk (value heads h of
key head h // (Hv / Hk)); g, beta (B, T, Hv) fp32, g <= 0 the log of the
decay (−inf resets a finite state, in delta_rule_step any).  q, k, v are fp32
or bf16; states and every sum are fp32.  Dk and Dv are multiples of 8 up to
128.  Strides are free as long as heads' rows are contiguous, start at
multiples of 16 bytes (delta_rule_step: anywhere) and do not overlap along T.

`lens` (B) int64 on the device: positions at or behind a row's length are not
read, leave the state as it is and get zeros (also as gradients); a length of
0 returns the initial state.  Nothing synchronises with the host; every call
can be captured in a graph.  Plain tensors in and out: no autograd graph is
built, whatever requires a gradient.

    o, state, saved = delta_rule(q, k, v, g, beta, lens=lens, save=True)
    dq, dk, dv, dg, dbeta, _ = delta_rule_backward(saved, do)
    o = delta_rule_step(q1, k1, v1, g1, beta1, state)        # next click, state in place
"""
from __future__ import annotations

import ctypes as C

import torch

from . import call, ptr
from .operands import TYPES, Plans, entry, fail, held, keep, layout, run, stream, stride, tensor, whole, wrote

_IO = (torch.float32, torch.bfloat16)


class Saved:
    """What the backward pass needs of a forward call: its operands (not copied: they have to keep their values), the
    updates and chunk states it left, and its segments' transitions."""

    def __init__(self, plan, operands, scale, U, S0, trans):
        self.plan, self.operands, self.scale, self.U, self.S0, self.trans = plan, operands, scale, U, S0, trans
        self.held, self.stream = [held(t) for t in operands], stream(plan.device)


_plans, _plans_back, _plans_step = Plans(), Plans(), Plans()


def _strides(*rows):
    flat = [s for r in rows for s in r]
    return (C.c_int64 * 18)(*flat, *([0] * (18 - len(flat))))


def _apart(name, t, width):
    if not width <= t.stride(1) < 1 << 23:
        fail(name, f"positions overlap or lie too far apart: stride {t.stride(1)}")


def _sizes(B, T, Hk, Hv, Dk, Dv, lead):
    """lead: 2 for (B, T), 1 for (B,), whose kernel takes any number of heads."""
    if B * Hv >= 1 << 24 or T > 65535 * 32:
        fail("q", f"less than 2^24 rows times value heads and at most 2^21 − 32 positions are expected, got {B}·{Hv} and {T}")
    if lead == 2 and max(Hk * Dk, Hv * Dv) >= 1 << 23:
        fail("q" if Hk * Dk >= Hv * Dv else "v", f"all heads of a position have to be less than 2^23 values, got {max(Hk * Dk, Hv * Dv)}")


class _Plan:
    """Checks of the operands that forward, backward and step share.  lead: 2 for (B, T), 1 for (B,)."""

    def __init__(self, q, k, v, g, beta, lead):
        align = 16 if lead == 2 else 1   # (one token is read value by value)
        tensor("q", q, (*[None] * lead, None, None), _IO, align=align)
        self.Hk, self.Dk = Hk, Dk = q.shape[-2:]
        tensor("k", k, (*q.shape,), (q.dtype,), q.device, align=align)
        tensor("v", v, (*q.shape[:-2], None, None), (q.dtype,), q.device, align=align)
        self.Hv, self.Dv = Hv, Dv = v.shape[-2:]
        if Hk == 0 or Hv == 0 or Hv % Hk:
            fail("v", f"{Hv} value heads are no multiple of {Hk} key heads")
        for name, d in (("q", Dk), ("v", Dv)):
            if d == 0 or d % 8 or d > 128:
                fail(name, f"a head width that is a multiple of 8 up to 128 is expected, got {d}")
        for name, t in (("g", g), ("beta", beta)):
            if not isinstance(t, torch.Tensor) or t.dim() != lead + 1:
                fail(name, f"a tensor of shape {(*q.shape[:-2], Hv)} is expected")
            tensor(name, t[..., None], (*q.shape[:-2], Hv, 1), (torch.float32,), q.device)   # any strides
        self.B, self.T = q.shape[0], q.shape[1] if lead == 2 else 1
        _sizes(self.B, self.T, Hk, Hv, Dk, Dv, lead)
        if self.T > 1:
            for name, t, d in (("q", q, Dk), ("k", k, Dk), ("v", v, Dv), ("g", g, 1), ("beta", beta, 1)):
                _apart(name, t, d)
        self.device, self.dtype, self.type, self.scale = q.device, q.dtype, TYPES[q.dtype], Dk ** -0.5
        self.state = (self.B, Hv, Dk, Dv)
        self.sizes = (self.B, self.T, Hk, Hv, Dk, Dv)
        self.empty = self.B == 0 or self.T == 0
        self.rows = [[stride(t, d) for d in range(lead)] for t in (q, k, v, g, beta)]
        self.rows = [(r if lead == 2 else [r[0], 0]) + [stride(t, lead)] for r, t in zip(self.rows, (q, k, v, g, beta))]
        self.strides = _strides(*self.rows)


def _aligned(**tensors):
    for name, t in tensors.items():
        if t is not None and t.data_ptr() & 15:
            fail(name, "has to start at a multiple of 16 bytes")


def _plan(q, k, v, g, beta, lens, state):
    p = _Plan(q, k, v, g, beta, 2)
    if lens is not None:
        whole("lens", lens, (p.B,), (torch.int64,), p.device)
    if state is not None:
        whole("state", state, p.state, (torch.float32,), p.device)
    p.forward, p.backward = entry("rg_delta_fwd"), entry("rg_delta_bwd")
    p.chunks = call("rg_delta_chunk_floats", p.B, p.T, p.Hv, p.Dk, p.Dv)
    n = call("rg_delta_segments", p.B, p.T, p.Hv, p.Dk, p.Dv)
    trans = call("rg_delta_trans_floats", p.B, p.T, p.Hv, p.Dk, p.Dv)
    p.trans, p.local = (trans, (p.B, p.Hv, n, p.Dk, p.Dv)) if n > 1 else (None, None)
    return p


def delta_rule(q, k, v, g, beta, scale=None, lens=None, state=None, save=False):
    """-> o (B, T, Hv, Dv) of q's type, final state (B, Hv, Dk, Dv) fp32, and with save=True what
    delta_rule_backward() takes.  state: initial state (not written), zeros if None; scale: Dk ** -0.5 if None."""
    operands = (q, k, v, g, beta, lens, state)
    key = tuple(map(layout, operands)) if isinstance(q, torch.Tensor) else None
    p = _plans.get(key) or _plans.put(key, _plan(*operands))
    at = q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(), ptr(lens), ptr(state)
    if (at[0] | at[1] | at[2] | (at[6] or 0)) & 15 and not p.empty:
        _aligned(q=q, k=k, v=v, state=state)
    scale = p.scale if scale is None else float(scale)
    o = torch.empty(p.B, p.T, p.Hv, p.Dv, dtype=p.dtype, device=p.device)
    final = torch.empty(p.state, dtype=torch.float32, device=p.device)
    U = S0 = trans = local = None
    if p.empty:
        final.copy_(state) if state is not None else final.zero_()
    else:
        if save:
            U = torch.empty(p.B, p.Hv, p.T, p.Dv, dtype=torch.float32, device=p.device)
            S0 = torch.empty(p.chunks, dtype=torch.float32, device=p.device) if p.chunks else None
        if p.trans:
            trans, local = (torch.empty(n, dtype=torch.float32, device=p.device) for n in (p.trans, p.local))
        run(p.forward, p.device, *at[:5], p.strides, *at[5:], p.type, *p.sizes, scale, o.data_ptr(), final.data_ptr(),
            ptr(U), ptr(S0), ptr(trans), ptr(local))
    return (o, final, Saved(p, operands, scale, U, S0, trans)) if save else (o, final)


def _back_plan(p, do, dstate):
    tensor("do", do, (p.B, p.T, p.Hv, p.Dv), (p.dtype,), p.device, align=16)
    if p.T > 1:
        _apart("do", do, p.Dv)
    if dstate is not None:
        whole("dstate", dstate, p.state, (torch.float32,), p.device)
    return _strides(*p.rows, [stride(do, d) for d in range(3)])


def delta_rule_backward(saved, do, dstate=None):
    """Gradients of sum(o·do) + sum(final·dstate): dq, dk, dv of their inputs' type, dg, dbeta fp32 (B, T, Hv), and
    dstate0 fp32 (None where the forward had no initial state).  Gradients of key heads are summed over their value
    heads in a fixed order.  Can be called again with other gradients."""
    if not isinstance(saved, Saved):
        fail("saved", "what delta_rule(..., save=True) returned is expected")
    p, (q, k, v, g, beta, lens, state) = saved.plan, saved.operands
    if [held(t) for t in saved.operands] != saved.held:
        raise RuntimeError("delta_rule_backward: an operand of the forward call was changed in place or given other memory since")
    key = (p, layout(do), layout(dstate)) if isinstance(do, torch.Tensor) else None
    strides = _plans_back.get(key) or _plans_back.put(key, _back_plan(p, do, dstate))
    if (do.data_ptr() | (ptr(dstate) or 0)) & 15 and not p.empty:
        _aligned(do=do, dstate=dstate)
    half = {"dtype": p.dtype, "device": p.device}
    full = {"dtype": torch.float32, "device": p.device}
    dq, dk = (torch.empty(p.B, p.T, p.Hk, p.Dk, **half) for _ in range(2))
    dv = torch.empty(p.B, p.T, p.Hv, p.Dv, **half)
    dg, dbeta = (torch.empty(p.B, p.T, p.Hv, **full) for _ in range(2))
    dstate0 = None if state is None else torch.empty(p.state, **full)
    if p.empty:
        if dstate0 is not None:
            dstate0.copy_(dstate) if dstate is not None else dstate0.zero_()
    else:
        keep(p.device, saved.stream, saved.U, saved.S0, saved.trans)
        dX = torch.empty(p.B, p.Hv, p.T, p.Dv, **full)
        dS = torch.empty(p.chunks, **full) if p.chunks else None
        local = torch.empty(p.local, **full) if p.local else None
        run(p.backward, p.device, q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(), do.data_ptr(),
            strides, ptr(lens), ptr(state), ptr(dstate), saved.U.data_ptr(), ptr(saved.S0), ptr(saved.trans), p.type, *p.sizes,
            saved.scale, dX.data_ptr(), ptr(dS), ptr(local), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dg.data_ptr(),
            dbeta.data_ptr(), ptr(dstate0))
    return dq, dk, dv, dg, dbeta, dstate0


def _step_plan(q, k, v, g, beta, state):
    p = _Plan(q, k, v, g, beta, 1)
    tensor("state", state, p.state, (torch.float32,), p.device, align=16)
    if p.B and not state[0].is_contiguous():
        fail("state", f"each row's (Hv, Dk, Dv) has to be contiguous, strides are {state.stride()}")
    if p.B > 1 and state.stride(0) < p.Hv * p.Dk * p.Dv:
        fail("state", f"rows overlap: stride {state.stride(0)}")
    p.step, p.apart, p.sizes = entry("rg_delta_step"), stride(state, 0), (p.B, p.Hk, p.Hv, p.Dk, p.Dv)
    return p


def delta_rule_step(q, k, v, g, beta, state, scale=None):
    """One token of every row: q, k (B, Hk, Dk), v (B, Hv, Dv), g, beta (B, Hv); state (B, Hv, Dk, Dv) fp32 is updated
    in place (its rows may lie apart, as in a larger pool, but not overlap).  -> o (B, Hv, Dv) of q's type."""
    key = tuple(map(layout, (q, k, v, g, beta, state))) if isinstance(q, torch.Tensor) else None
    p = _plans_step.get(key) or _plans_step.put(key, _step_plan(q, k, v, g, beta, state))
    o = torch.empty(p.B, p.Hv, p.Dv, dtype=p.dtype, device=p.device)
    if p.B:
        at = state.data_ptr()
        if at & 15:
            _aligned(state=state)
        run(p.step, p.device, q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(), p.strides, p.type,
            *p.sizes, p.scale if scale is None else float(scale), at, p.apart, o.data_ptr())
        wrote(state)
    return o
