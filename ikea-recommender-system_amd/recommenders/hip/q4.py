"""Item scores from a 4-bit item table (csrc/q4.hip): the output layer of a
served model at a quarter of its bf16 bytes.

    codes, scales = q4_pack(model_W, group=32)          # once
    scores = q4_scores(h, codes, scales, bias)          # (M, N) fp32, per request
    top = scores.topk(20)

codes  (N, K / 2) uint8, two codes a byte, the even column in the low half;
scales (N, K / group) bfloat16; a weight is scales[n, k // group]·(code − 8).
K is a multiple of `group` (32, 64 or 128) and at most 1024; any number of
items N, up to 1M rows M.  Sums are kept in fp32; x may be fp32 or bf16 and
enters exactly, infinities and NaN as a sum of x·w takes them (rows with values
from 2^96 on are slower: the table is read twice for them).  Capturable; no
workspace, no host synchronisation.  Weights have to be finite.
"""
from __future__ import annotations

import torch

from . import ptr
from .operands import TYPES, Plans, entry, fail, layout, run, shares_memory, stride, tensor, whole, wrote

GROUPS = (32, 64, 128)
K_MAX, M_MAX = 1024, 65535 * 16


def _table(K, group):
    if group not in GROUPS:
        fail("group", f"{' / '.join(map(str, GROUPS))} is expected, got {group}")
    if K == 0 or K % group or K > K_MAX:
        fail("columns", f"a multiple of the group size {group} up to {K_MAX} is expected, got {K}")


def _rows(name, t):
    if t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        fail(name, f"rows overlap: stride {t.stride(0)}, {t.shape[1]} columns")


def q4_pack(W, group=32):
    """Quantise a (N, K) fp32 or bf16 table: (codes, scales).  Per group the scale is max |w| / 7 rounded to bf16 and a
    code is round(w / scale) + 8, ties to even, clamped to 0 .. 15."""
    tensor("W", W, (None, None), (torch.float32, torch.bfloat16))
    N, K = W.shape
    _table(K, group)
    _rows("W", W)
    codes = torch.empty(N, K // 2, dtype=torch.uint8, device=W.device)
    scales = torch.empty(N, K // group, dtype=torch.bfloat16, device=W.device)
    if N:
        run(entry("rg_q4_pack"), W.device, ptr(W), TYPES[W.dtype], stride(W, 0) or K, N, K, group, ptr(codes), ptr(scales))
    return codes, scales


_plans = Plans()


def _plan(x, codes, scales, bias):
    tensor("x", x, (None, None), (torch.float32, torch.bfloat16))
    M, K = x.shape
    if M > M_MAX:
        fail("x", f"at most {M_MAX} rows are expected, got {M}")
    _rows("x", x)
    whole("codes", codes, (None, K // 2), (torch.uint8,), x.device)
    N = codes.shape[0]
    whole("scales", scales, (N, None), (torch.bfloat16,), x.device)
    groups = scales.shape[1]
    if groups == 0 or K % groups:
        fail("scales", f"{groups} groups do not divide {K} columns")
    _table(K, K // groups)
    if bias is not None:
        whole("bias", bias, (N,), (torch.float32,), x.device)
    return entry("rg_q4_scores"), x.device, M, N, K, K // groups, TYPES[x.dtype], stride(x, 0) or K


def q4_scores(x, codes, scales, bias=None, out=None):
    """x (M, K) · table (N, K)ᵀ + bias -> (M, N) fp32.  out: written instead of a new tensor; its rows may be strided, and
    it must not share memory with the operands."""
    key = (layout(x), layout(codes), layout(scales), layout(bias)) if isinstance(x, torch.Tensor) else None
    fn, device, M, N, K, group, kind, ldx = _plans.get(key) or _plans.put(key, _plan(x, codes, scales, bias))
    at = codes.data_ptr(), scales.data_ptr()
    if (at[0] | at[1]) & 15 and N:
        fail("codes" if at[0] & 15 else "scales", "has to start at a multiple of 16 bytes")
    if out is None:
        out = torch.empty(M, N, dtype=torch.float32, device=device)
        ldy = N
    else:
        tensor("out", out, (M, N), (torch.float32,), device)
        if M > 1 and out.stride(0) < N:
            fail("out", f"rows overlap: stride {out.stride(0)}, {N} items")
        for name, t in (("x", x), ("codes", codes), ("scales", scales), ("bias", bias)):
            if shares_memory(t, out):
                fail("out", f"shares memory with {name}, which is read while it is written")
        ldy = stride(out, 0) or N
    if M and N:
        run(fn, device, x.data_ptr(), kind, ldx, *at, ptr(bias), M, N, K, group, out.data_ptr(), ldy)
        wrote(out)
    return out
