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
# (device, hk_rope_axes_shape) of the layouts that have been checked, by everything the checks look at
_shapes: dict[tuple, tuple] = {}


def _row_stride(table):
    """Elements from one row of a cos or sin table to the next (its width where there is no next)."""
    return table.stride(-2) if table.shape[-2] > 1 else table.shape[-1]


def _checked(q, k, cos, sin, positions, sections, interleaved, inverse):
    """(device, shape) of a call whose head dims and table rows are contiguous; raises if it is not one."""
    dev = _lib.require_device(q, k, cos, sin, positions)
    assert q.dim() == 4 and k.dim() == 4, "q and k must be (bsz, n_heads, seq_len, head_dim)"
    bsz, hq, seq_len, hd = q.shape
    kb, hk, kt, kd = k.shape
    assert (kb, kt, kd) == (bsz, seq_len, hd), f"q and k differ: {tuple(q.shape)} and {tuple(k.shape)}"
    assert q.dtype == k.dtype, f"q and k have different dtypes: {q.dtype} and {k.dtype}"
    assert cos.shape == sin.shape and cos.dtype == sin.dtype, "cos and sin must be alike"
    assert (cos.dim() == 2 or cos.dim() == 3 and cos.shape[0] == 1) and cos.shape[-1] * 2 == hd, \
        f"cos/sin must be (1, positions, head_dim/2); got {tuple(cos.shape)}"
    axes = len(sections)
    if not 1 <= axes <= 4:
        raise ValueError(f"sections names 1 to 4 axes, got {axes}")
    if positions.dtype not in _POS_CODE:
        raise TypeError(f"positions must be int32 or int64, got {positions.dtype}")
    assert positions.dim() == 3 and positions.shape[0] == axes and positions.shape[2] == seq_len and \
        positions.shape[1] in (1, bsz), \
        f"positions must be ({axes}, {bsz} or 1, {seq_len}); got {tuple(positions.shape)}"
    s = _lib.RopeAxesShape(B=bsz, T=seq_len, D=hd, Hq=hq, Hk=hk, table_rows=cos.shape[-2], table_ld=_row_stride(cos),
                           axes=axes, interleaved=bool(interleaved), pos_type=_POS_CODE[positions.dtype],
                           dtype_x=_lib.dtype_code(q), dtype_cs=_lib.dtype_code(cos), inverse=inverse)
    s.sections[:axes] = [int(c) for c in sections]
    s.pos[:] = positions.stride()
    if positions.shape[1] == 1:
        s.pos[1] = 0
    for x, rows_in, rows_out in ((q, s.q_in, s.q_out), (k, s.k_in, s.k_out)):
        out = torch.empty_like(x)
        assert x.stride(3) == 1 and out.stride(3) == 1
        rows_in[:], rows_out[:] = x.stride()[:3], out.stride()[:3]
    return dev, s


def _launch(q, k, cos, sin, positions, sections, interleaved, inverse):
    """(q_out, k_out): one launch over both. A layout is checked once (host time: a decode step's call is bound by it)."""
    sections = tuple(sections)
    key = (q.shape, q.stride(), k.shape, k.stride(), cos.shape, cos.stride(), sin.shape, sin.stride(), positions.shape,
           positions.stride(), q.dtype, k.dtype, cos.dtype, sin.dtype, positions.dtype, q.device, k.device, cos.device,
           sin.device, positions.device, sections, interleaved, inverse)
    known = _shapes.get(key)
    if known is None:
        again = [x if x.dim() == 0 or x.stride(-1) == 1 else x.contiguous() for x in (q, k, cos, sin)]
        if cos.dim() >= 2 and cos.shape == sin.shape and not \
                cos.shape[-1] <= _row_stride(again[2]) == _row_stride(again[3]):
            again[2:] = again[2].contiguous(), again[3].contiguous()
        if any(a is not b for a, b in zip(again, (q, k, cos, sin))):
            return _launch(*again, positions, sections, interleaved, inverse)
        known = _checked(q, k, cos, sin, positions, sections, interleaved, inverse)
        if len(_shapes) >= 1024:
            _shapes.clear()
        _shapes[key] = known
    dev, shape = known
    # empty_like keeps a dense input's layout and is contiguous for broadcast (zero-stride) ones
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    _lib.call_on(dev, "hk_rope_axes", q_out.data_ptr(), q.data_ptr(), k_out.data_ptr(), k.data_ptr(), cos.data_ptr(),
                 sin.data_ptr(), positions.data_ptr(), ctypes.addressof(shape))
    return q_out, k_out


def rope_axes_forward(q, k, cos, sin, positions, sections, interleaved=False):
    """Forward: returns q_out, k_out (new tensors)."""
    return _launch(q, k, cos, sin, positions, sections, interleaved, False)


def rope_axes_backward(dq, dk, cos, sin, positions, sections, interleaved=False):
    """Backward: the transpose rotation, i.e. the forward with -sin."""
    return _launch(dq, dk, cos, sin, positions, sections, interleaved, True)


class HildaRopeAxesFunction(torch.autograd.Function):
    """Autograd wrapper: q, k = HildaRopeAxesFunction.apply(q, k, cos, sin, positions, sections, interleaved). The
    rotation is linear, so its backward is one of the other sense, and can be differentiated again."""

    @staticmethod
    def forward(ctx, q, k, cos, sin, positions, sections, interleaved=False, inverse=False):
        ctx.save_for_backward(cos, sin, positions)
        ctx.args = sections, interleaved, not inverse
        return _launch(q, k, cos, sin, positions, sections, interleaved, inverse)

    @staticmethod
    def backward(ctx, dq, dk):
        call = HildaRopeAxesFunction.apply if torch.is_grad_enabled() else _launch
        dq, dk = call(dq, dk, *ctx.saved_tensors, *ctx.args)
        return dq, dk, None, None, None, None, None, None


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
