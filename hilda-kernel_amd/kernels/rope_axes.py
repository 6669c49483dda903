"""RoPE with several position axes on MI355X, forward and backward.

Beside ``kernels/rope.py`` for prompts that hold images and video: every pair
of a head turns by the position of one axis (time, height, width), which the
tokens bring with them. The reference's RoPE (rope.py:90-228) has one axis and
the positions 0..T-1; the rotation and the cos/sin tables are the same.

q and k are (bsz, n_heads, seq_len, head_dim) with any strides in the first
three dims, as for ``hilda_rope``; outputs keep a dense input's layout.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .rope import RotaryEmbedding

_POS_CODE = {torch.int32: _lib.I32, torch.int64: _lib.I64}
_sections_cache: dict[tuple, ctypes.Array] = {}


def _sections_arg(sections):
    """The sections as a C array (made once for each tuple of counts)."""
    key = tuple(sections)
    arr = _sections_cache.get(key)
    if arr is None:
        if not 1 <= len(key) <= 4:
            raise ValueError(f"sections names 1 to 4 axes, got {len(key)}")
        arr = (ctypes.c_int64 * len(key))(*(int(c) for c in key))
        if len(_sections_cache) < 64:
            _sections_cache[key] = arr
    return arr


def _table(t):
    """(rows, D/2) of a cos or sin table given as that or as (1, rows, D/2)."""
    if t.dim() == 3:
        assert t.shape[0] == 1, f"cos/sin must be (1, positions, head_dim/2); got {tuple(t.shape)}"
        t = t[0]
    assert t.dim() == 2, f"cos/sin must be (1, positions, head_dim/2); got {tuple(t.shape)}"
    return t if t.stride(1) == 1 else t.contiguous()


def _rows(x):
    """x with unit stride in the head dim."""
    return x if x.stride(-1) == 1 else x.contiguous()


def _launch(q, k, cos, sin, positions, sections, interleaved, inverse):
    """(q_out, k_out): one launch over both."""
    dev = _lib.require_device(q, k, cos, sin, positions)
    assert q.dim() == 4 and k.dim() == 4, "q and k must be (bsz, n_heads, seq_len, head_dim)"
    bsz, hq, seq_len, hd = q.shape
    kb, hk, kt, kd = k.shape
    assert (kb, kt, kd) == (bsz, seq_len, hd), f"q and k differ: {tuple(q.shape)} and {tuple(k.shape)}"
    assert q.dtype == k.dtype, f"q and k have different dtypes: {q.dtype} and {k.dtype}"
    cos, sin = _table(cos), _table(sin)
    assert cos.shape == sin.shape and cos.dtype == sin.dtype, "cos and sin must be alike"
    assert cos.shape[1] * 2 == hd, f"cos/sin must be (1, positions, head_dim/2); got {tuple(cos.shape)}"
    if cos.stride() != sin.stride():
        cos, sin = cos.contiguous(), sin.contiguous()
    sec = _sections_arg(sections)
    axes = len(sec)
    if positions.dtype not in _POS_CODE:
        raise TypeError(f"positions must be int32 or int64, got {positions.dtype}")
    assert positions.dim() == 3 and positions.shape[0] == axes and positions.shape[2] == seq_len and \
        positions.shape[1] in (1, bsz), \
        f"positions must be ({axes}, {bsz} or 1, {seq_len}); got {tuple(positions.shape)}"
    pa, pb, pt = positions.stride()
    if positions.shape[1] == 1:
        pb = 0
    q, k = _rows(q), _rows(k)
    # empty_like keeps a dense input's layout and is contiguous for broadcast (zero-stride) ones
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    qi, ki, qo, ko = q.stride(), k.stride(), q_out.stride(), k_out.stride()
    assert qo[3] == 1 and ko[3] == 1
    _lib.call_on(dev, "hk_rope_axes", q_out.data_ptr(), q.data_ptr(), hq, qi[0], qi[1], qi[2], qo[0], qo[1], qo[2],
                 k_out.data_ptr(), k.data_ptr(), hk, ki[0], ki[1], ki[2], ko[0], ko[1], ko[2],
                 cos.data_ptr(), sin.data_ptr(), cos.shape[0], cos.stride(0), positions.data_ptr(),
                 _POS_CODE[positions.dtype], pa, pb, pt, sec, axes, int(interleaved), bsz, seq_len, hd,
                 _lib.dtype_code(q), _lib.dtype_code(cos), int(inverse))
    return q_out, k_out


def rope_axes_forward(q, k, cos, sin, positions, sections, interleaved=False):
    """Forward: returns q_out, k_out (new tensors)."""
    return _launch(q, k, cos, sin, positions, sections, interleaved, False)


def rope_axes_backward(dq, dk, cos, sin, positions, sections, interleaved=False):
    """Backward: the transpose rotation, i.e. the forward with -sin."""
    return _launch(dq, dk, cos, sin, positions, sections, interleaved, True)


class HildaRopeAxesFunction(torch.autograd.Function):
    """Autograd wrapper: q, k = HildaRopeAxesFunction.apply(q, k, cos, sin, positions, sections, interleaved)."""

    @staticmethod
    def forward(ctx, q, k, cos, sin, positions, sections, interleaved):
        ctx.save_for_backward(cos, sin, positions)
        ctx.sections, ctx.interleaved = sections, interleaved
        return rope_axes_forward(q, k, cos, sin, positions, sections, interleaved)

    @staticmethod
    def backward(ctx, dq, dk):
        cos, sin, positions = ctx.saved_tensors
        dq, dk = rope_axes_backward(dq, dk, cos, sin, positions, ctx.sections, ctx.interleaved)
        return dq, dk, None, None, None, None, None


def hilda_rope_axes(q, k, cos, sin, positions, sections, interleaved=False):
    """RoPE with several position axes: returns q_out, k_out.

    q (B, Hq, T, D), k (B, Hk, T, D); cos, sin (1, P, D/2) as of ``RotaryEmbedding``; positions (A, B or 1, T) int32
    or int64; sections A counts of pairs with sum D/2. Pair i turns by row positions[a(i), b, t] of the tables, where
    a(i) is the section it falls in, or with ``interleaved`` i mod A while i < A * sections[i mod A], else axis 0.
    A position outside [0, P) gives NaN in the pairs of its axis. Gradients go to q and k.
    """
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad):
        return HildaRopeAxesFunction.apply(q, k, cos, sin, positions, sections, interleaved)
    return rope_axes_forward(q, k, cos, sin, positions, sections, interleaved)


class MultiAxisRotaryEmbedding(RotaryEmbedding):
    """``RotaryEmbedding`` (same buffers) whose tokens bring a position for each axis.

    sections: pairs of each axis, sum dim // 2; positions: (axes, batch or 1, seq_len).
    """

    def __init__(self, dim, sections, max_position_embeddings=2048, base=10000, interleaved=False, device=None):
        super().__init__(dim, max_position_embeddings, base, device)
        if sum(sections) != dim // 2:
            raise ValueError(f"sections {tuple(sections)} must sum to dim // 2 = {dim // 2}")
        self.sections = tuple(int(c) for c in sections)
        self.interleaved = bool(interleaved)

    def forward(self, q, k, positions):
        return hilda_rope_axes(q, k, self.cos_cached, self.sin_cached, positions, self.sections, self.interleaved)
