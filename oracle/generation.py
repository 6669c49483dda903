"""64-bit CPU definitions of the generation-side operators (test infrastructure).

The reference has no counterpart of these; each is the operator's formula in
fp64, one row or pair at a time where that is the plainer way.

How each function is pinned (tests/test_oracle_generation.py):
  rope_axes_ref       equal positions on every axis -> rope_ref; a pair's axis by hand on tiny sections
  norm_quant_ref      e4m3 values against torch's float8_e4m3fn cast; zeros -> q 0, scale 2^-100
  sample_ref          hand-worked distributions; draws over a grid of u give the kept probabilities
"""
from __future__ import annotations

import math

import numpy as np
import torch

__all__ = ["axis_of_pair", "rope_axes_ref", "norm_quant_ref", "e4m3_step", "sample_ref"]


def axis_of_pair(sections, interleaved):
    """The axis of each of the D/2 pairs."""
    half, axes = sum(sections), len(sections)
    out = []
    for i in range(half):
        if interleaved:
            a = i % axes
            out.append(a if a and i < axes * sections[a] else 0)
        else:
            end = 0
            for a, n in enumerate(sections):
                end += n
                if i < end:
                    out.append(a)
                    break
    return out


def rope_axes_ref(x, cos, sin, positions, sections, interleaved=False, inverse=False):
    """(y, room): the rotation in fp64 and |x1 c| + |x2 s| (the scale of its rounding errors).

    x (B, H, T, D); cos, sin (rows, D/2); positions (A, B or 1, T). Positions outside the table give NaN.
    """
    x, cos, sin = x.detach().cpu().double(), cos.cpu().double(), sin.cpu().double()
    B, H, T, D = x.shape
    half = D // 2
    pos = positions.cpu().long().expand(len(sections), B, T)
    c, s = torch.empty(B, T, half, dtype=torch.float64), torch.empty(B, T, half, dtype=torch.float64)
    for i, a in enumerate(axis_of_pair(sections, interleaved)):
        p = pos[a]
        bad = (p < 0) | (p >= cos.shape[0])
        at = p.clamp(0, max(0, cos.shape[0] - 1))
        for out, table in ((c, cos), (s, sin)):
            out[..., i] = torch.where(bad, math.nan, table[at, i])
    c, s = c[:, None], (-s if inverse else s)[:, None]
    x1, x2 = x[..., :half], x[..., half:]
    y = torch.cat((x1 * c - x2 * s, x2 * c + x1 * s), -1)
    room = torch.cat(((x1 * c).abs() + (x2 * s).abs(), (x2 * c).abs() + (x1 * s).abs()), -1)
    return y, room


def e4m3_step(v):
    """Distance of e4m3 values around v."""
    return torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)


def norm_quant_ref(x, w, r=None, eps=1e-6, group=None):
    """(y / scale before rounding, scale, s) in fp64; s is x + r rounded to x's type."""
    x = x.detach().cpu()
    s = x if r is None else (x.double() + r.detach().cpu().to(x.dtype).double()).to(x.dtype)
    f = s.double()
    y = f / torch.sqrt((f * f).mean(-1, keepdim=True) + eps) * w.detach().cpu().double()
    y = y.unflatten(-1, (-1, group or y.shape[-1]))
    scale = (y.abs().amax(-1) / 448).clamp_min(2.0 ** -100)
    return (y / scale[..., None]).flatten(-2), scale, s


def sample_ref(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(ids, logp, kept): one row of logits at a time, in numpy fp64. kept: a list of index arrays (None: no
    distribution)."""
    x = logits.detach().cpu().double().numpy()
    x = x.reshape(-1, x.shape[-1])
    rows, V = x.shape

    def each(v, kind=np.float64):
        v = v.detach().cpu().numpy().astype(kind).reshape(-1) if isinstance(v, torch.Tensor) else kind(v)
        return np.broadcast_to(v, (rows,))

    temp, top_p, min_p, u = (each(v) for v in (temperature, top_p, min_p, u))
    top_k = each(top_k, np.int64)
    ids, logp, sets = np.full(rows, -1, np.int64), np.full(rows, np.nan), []
    for i in range(rows):
        ok = np.isfinite(temp[i]) and 2.0 ** -64 <= temp[i] <= 2.0 ** 64 and 0 <= u[i] <= 1
        ok = ok and not np.isnan(top_p[i]) and not np.isnan(min_p[i])
        if not ok or np.isnan(x[i]).any() or x[i].max() == np.inf or x[i].max() == -np.inf:
            sets.append(None)
            continue
        z = (x[i] - x[i].max()) / temp[i]
        p = np.exp(z)
        order = np.lexsort((np.arange(V), -x[i]))
        if 0 < top_k[i] < V:
            order = order[:top_k[i]]
        if top_p[i] < 1:
            run = np.cumsum(p[order])
            before = np.concatenate(([0.0], run[:-1]))
            n = max(1, int((before < max(top_p[i], 0.0) * run[-1]).sum()))
            order = order[:n]
        kept = np.sort(order[p[order] >= min(max(min_p[i], 0.0), 1.0)])
        run = np.cumsum(p[kept])
        hit = np.nonzero(run > u[i] * run[-1])[0]
        ids[i] = kept[hit[0]] if len(hit) else kept[np.nonzero(p[kept])[0][-1]]
        logp[i] = z[ids[i]] - math.log(p.sum())
        sets.append(kept)
    shape = logits.shape[:-1]
    return torch.from_numpy(ids).view(shape), torch.from_numpy(logp).view(shape), sets
