"""Attention of rows with any mask in 64 bits, and how far a kernel that works
as the row kernels do may be from it."""
from __future__ import annotations

import math

import torch

U32 = 2.0 ** -24  # half a step of f32


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def attend(q, k, v, allow, scale=None, *, p_half=None, p_floor=0.0, out_dtype=torch.float32):
    """q [R, H, D], k and v [S, Hk, D], allow bool [R, S]: (out, tolerance), f64.

    The tolerance counts, per output element with A = sum p |v|:
      * half a step of the output's type at its value,
      * the rounding of every probability: p_half relative, p_floor absolute
        (relative to the largest probability of the row, whose sum is >= 1),
      * the score's error as a relative error of every p, twice (numerator and
        denominator): D + 8 roundings of f32 on sum |q k| * scale (the products'
        sum, the scaling and the split of f32 operands), and one step of the
        scaled score's exponent each for exp2 and its argument,
      * S + 8 roundings of f32 in the two sums over the keys.
    """
    rows, heads, d = q.shape
    group = heads // k.shape[1]
    scale = scale or 1.0 / math.sqrt(d)
    q64, k64, v64 = q.double(), k.double().repeat_interleave(group, 1), v.double().repeat_interleave(group, 1)
    s = torch.einsum("rhd,shd->hrs", q64, k64) * scale
    sabs = (torch.einsum("rhd,shd->hrs", q64.abs(), k64.abs()) * scale).masked_fill(~allow[None], 0.0)
    s = s.masked_fill(~allow[None], -math.inf)
    empty = ~allow.any(-1)
    top = s.amax(-1, keepdim=True).masked_fill(empty[None, :, None], 0.0)
    e = torch.exp(s - top)
    total = e.sum(-1, keepdim=True).masked_fill(empty[None, :, None], 1.0)
    p = e / total
    out = torch.einsum("hrs,shd->rhd", p, v64)
    a = torch.einsum("hrs,shd->rhd", p, v64.abs())
    keys = k.shape[0]
    delta = ((d + 8) * U32 * sabs.amax(-1) + 4 * U32 * (s - top).masked_fill(~allow[None], 0).abs().amax(-1) + 4 * U32)
    floor = p_floor * torch.einsum("rs,shd->rhd", allow.double(), v64.abs())
    p_half = half_step(q.dtype) if p_half is None else p_half
    tol = (half_step(out_dtype) * out.abs() + (p_half + (keys + 8) * U32) * a + 2 * delta.t()[..., None] * a + floor
           + torch.finfo(out_dtype).smallest_normal * torch.finfo(out_dtype).eps)
    return out, tol


def check(got, want, tol, what=""):
    err = (got.double().cpu() - want.cpu()).abs()
    bad = ~(err <= tol.cpu())
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / tol.cpu()).max()):.3g} "
                           f"tolerances, first at {bad.nonzero()[0].tolist()}")


def causal_mask(rows, before, window=0):
    keys = before + rows
    me, at = before + torch.arange(rows)[:, None], torch.arange(keys)[None, :]
    ok = at <= me
    return ok & (at > me - window) if window else ok
