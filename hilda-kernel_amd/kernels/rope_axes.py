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


def _launch(q, k, cos, sin, positions, sections, interleaved, inverse):
    """(q_out, k_out): one launch over both."""
    # shapes and strides are read once each (host time: a decode step's call is bound by it)
    dev = _lib.require_device(q, k, cos, sin, positions)
    qs, ks, cs, ps = q.shape, k.shape, cos.shape, positions.shape
    assert len(qs) == 4 and len(ks) == 4, "q and k must be (bsz, n_heads, seq_len, head_dim)"
    bsz, hq, seq_len, hd = qs
    kb, hk, kt, kd = ks
    assert kb == bsz and kt == seq_len and kd == hd, f"q and k differ: {tuple(qs)} and {tuple(ks)}"
    dtype, table_dtype = q.dtype, cos.dtype
    assert k.dtype == dtype, f"q and k have different dtypes: {dtype} and {k.dtype}"
    assert sin.shape == cs and sin.dtype == table_dtype, "cos and sin must be alike"
    assert (len(cs) == 2 or len(cs) == 3 and cs[0] == 1) and cs[-1] * 2 == hd, \
        f"cos/sin must be (1, positions, head_dim/2); got {tuple(cs)}"
    sec = _sections_arg(sections)
    axes = len(sec)
    pos_code = _POS_CODE.get(positions.dtype)
    if pos_code is None:
        raise TypeError(f"positions must be int32 or int64, got {positions.dtype}")
    assert len(ps) == 3 and ps[0] == axes and ps[2] == seq_len and (ps[1] == bsz or ps[1] == 1), \
        f"positions must be ({axes}, {bsz} or 1, {seq_len}); got {tuple(ps)}"
    pa, pb, pt = positions.stride()
    if ps[1] == 1:
        pb = 0
    cst = cos.stride()
    if cst[-1] != 1 or sin.stride() != cst:
        cos, sin = cos.contiguous(), sin.contiguous()
        cst = cos.stride()
    qi, ki = q.stride(), k.stride()
    if qi[3] != 1:
        q = q.contiguous()
        qi = q.stride()
    if ki[3] != 1:
        k = k.contiguous()
        ki = k.stride()
    # empty_like keeps a dense input's layout and is contiguous for broadcast (zero-stride) ones
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    qo, ko = q_out.stride(), k_out.stride()
    assert qo[3] == 1 and ko[3] == 1
    _lib.call_on(dev, "hk_rope_axes", q_out.data_ptr(), q.data_ptr(), hq, qi[0], qi[1], qi[2], qo[0], qo[1], qo[2],
                 k_out.data_ptr(), k.data_ptr(), hk, ki[0], ki[1], ki[2], ko[0], ko[1], ko[2],
                 cos.data_ptr(), sin.data_ptr(), cs[-2], cst[-2], positions.data_ptr(), pos_code, pa, pb, pt, sec, axes,
                 interleaved, bsz, seq_len, hd, _lib.dtype_code(q), _lib.dtype_code(cos), inverse)
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
