"""The serving operators' definitions in 64 bits, for the tests (torch on any device; no kernel of this
repository).  Each attention returns its value and, for every output element, the bounds that the
tests' tolerances are made of (:class:`Attended`)."""

from __future__ import annotations

import dataclasses
import math

import torch

F64 = torch.float64


def qk_norm_rope(x, w, positions, base, eps, rotary):
    """[T, H, D] -> (value, |a| + |b| of each element's rotated pair) in 64 bits."""
    x = x.to(F64)
    y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.to(F64)
    r = rotary // 2
    angle = positions.to(F64)[:, None, None] * float(base) ** (-torch.arange(r, dtype=F64, device=x.device) / max(r, 1))
    a, b = y[..., :r], y[..., r : 2 * r]
    out = torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos(), y[..., 2 * r :]], -1)
    size = a.abs() + b.abs()
    return out, torch.cat([size, size, y[..., 2 * r :].abs()], -1)


# ---- the 4-bit cache ------------------------------------------------------------------------------


def kv4_quantise(x):
    """[T, H, D] 16-bit -> codes [T, H, G, 64] int64, scale, minimum [T, H, G] (bf16 values, 64 bits).

    The difference and the quotient are IEEE fp32 operations, as the format defines them."""
    g = x.float().unflatten(-1, (-1, 64))
    low, high = g.amin(-1), g.amax(-1)
    span = high - low
    # A quotient of tensors: torch multiplies by 1 / 15 where the divisor is a number.
    scale = (span / torch.full_like(span, 15)).bfloat16().float()
    minimum = low.bfloat16().float()
    codes = torch.round((g - minimum[..., None]) / scale[..., None]).clamp(0, 15)
    codes = torch.where(scale[..., None] > 0, codes, torch.zeros_like(codes))
    bad = ~torch.isfinite(span)
    scale = torch.where(bad, torch.zeros_like(scale), scale)
    minimum = torch.where(bad, torch.full_like(minimum, math.nan), minimum)
    codes = torch.where(bad[..., None], torch.zeros_like(codes), codes)
    return codes.long(), scale.to(F64), minimum.to(F64)


def kv4_values(codes, scale, minimum):
    return (minimum[..., None] + scale[..., None] * codes.to(F64)).flatten(-2)


def kv4_positions(dim, which, row):
    """(byte, shift) of each element of a row of codes: the layout's definition, element by element."""
    n_groups = dim // 64
    at = []
    for d in range(dim):
        g, e = divmod(d, 64)
        n = e % 8
        if which == 0:
            t, h = e // 16, (e % 16) // 8
            byte = t * 8 * n_groups + g * 8 + h * 4 + n // 2
        else:
            byte = ((e // 8) ^ (4 * ((row >> 1) & 1))) * 4 * n_groups + g * 4 + n // 2
        at.append((byte, 4 * (n % 2)))
    return at


def kv4_unpack(record, dim):
    """One record (uint8 [18 * dim], CPU) -> (codes [2, 16, dim], scale, minimum [2, 16, G])."""
    raw = record.tolist()
    groups = dim // 64
    codes = torch.zeros(2, 16, dim, dtype=torch.long)
    for which in (0, 1):
        for row in range(16):
            base = (which * 16 + row) * (dim // 2)
            for d, (byte, shift) in enumerate(kv4_positions(dim, which, row)):
                codes[which, row, d] = (raw[base + byte] >> shift) & 15
    params = record[16 * dim :].clone().view(torch.bfloat16).view(2, 16, groups, 2).to(F64)
    return codes, params[..., 0], params[..., 1]


# ---- attention ------------------------------------------------------------------------------------


@dataclasses.dataclass
class Attended:
    value: torch.Tensor   # sum_j p_j v_j
    mass: torch.Tensor    # sum_j p_j |v_j - centre_j|: what a relative error of the weights p can move
    size: torch.Tensor    # sum_j p_j |v_j|
    peak: torch.Tensor    # max_j |v_j - centre_j| over seen keys
    heaviest: torch.Tensor  # max_j p_j span_j, per row [.., 1]
    score: torch.Tensor   # max_j scale sum_d |q_d k_jd|, per row [.., 1]: what rounding in a score is relative to


def attend(q, k, v, scale, seen, centre=None, span=None):
    """q [R, D], k, v [S, D], seen [R, S] -> :class:`Attended` with [R, D] entries; rows that see
    nothing are zeros.  Unseen keys and values take no part, whatever they hold."""
    q, k, v = q.to(F64), k.to(F64), v.to(F64)
    dev = q.device
    centre = torch.zeros_like(v) if centre is None else centre.to(F64)
    span = torch.zeros(v.shape[0], dtype=F64, device=dev) if span is None else span
    used = seen.any(0)
    k, v, centre, span, seen = k[used], v[used], centre[used], span[used], seen[:, used]
    out = [torch.zeros(q.shape[0], v.shape[1], dtype=F64, device=dev) for _ in range(4)]
    score, heaviest = (torch.zeros(q.shape[0], 1, dtype=F64, device=dev) for _ in range(2))
    some = seen.any(1)
    if used.any() and some.any():
        w = torch.where(seen[some], q[some] @ k.T * scale, torch.full((), -math.inf, dtype=F64, device=dev))
        p = torch.softmax(w, -1)
        # A value that one row sees and another does not may be infinite or NaN.
        finite = torch.isfinite(v)
        vz = torch.where(finite, v, torch.zeros_like(v))
        out[0][some] = p @ vz
        if not finite.all():
            rows = out[0][some]
            for j in torch.nonzero(~finite.all(1)).flatten().tolist():
                hit = seen[some][:, j]
                rows[hit] = rows[hit] + torch.where(finite[j], torch.zeros_like(v[j]), p[hit][:, j : j + 1] * v[j])
            out[0][some] = rows
        off = torch.where(finite, v - centre, torch.zeros_like(v)).abs()
        out[1][some] = p @ off
        out[2][some] = p @ vz.abs()
        out[3][some] = off.amax(0, keepdim=True).expand(int(some.sum()), -1)
        bound = torch.where(seen[some], torch.nan_to_num(q[some].abs() @ k.abs().T * scale, nan=0.0, posinf=0.0), torch.zeros_like(w))
        heaviest[some] = (p * span).amax(-1, keepdim=True)
        score[some] = bound.amax(-1, keepdim=True)
    return Attended(*out, heaviest, score)


def window_mask(nq, nk, window, sinks, device="cpu"):
    p = (torch.arange(nq, device=device) + nk - nq)[:, None]
    j = torch.arange(nk, device=device)[None]
    seen = j <= p
    if window:
        seen = seen & ((j > p - window) | (j < sinks))
    return seen


def window_attention(q, k, v, cu_q, cu_k, scale, window, sinks):
    """Packed prompts: (row mask of all sequences' queries [Tq], :class:`Attended` with [Tq, Hq, D] entries)."""
    tq, hq, d = q.shape
    g = hq // k.shape[1]
    parts = [torch.zeros(tq, hq, d, dtype=F64, device=q.device) for _ in range(4)]
    score = torch.zeros(tq, hq, 1, dtype=F64, device=q.device)
    inside = torch.zeros(tq, dtype=torch.bool, device=q.device)
    for a, b, e, f in zip(cu_q, cu_q[1:], cu_k, cu_k[1:]):
        inside[a:b] = True
        seen = window_mask(b - a, f - e, window, sinks, q.device)
        for h in range(hq):
            r = attend(q[a:b, h], k[e:f, h // g], v[e:f, h // g], scale, seen)
            for part, x in zip(parts, (r.value, r.mass, r.size, r.peak)):
                part[a:b, h] = x
            score[a:b, h] = r.score
    return inside, Attended(*parts, torch.zeros_like(score), score)
