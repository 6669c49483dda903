"""RMSNorm and FusedAddRMSNorm with an 8-bit output on MI355X.

Beside ``kernels/rms_norm.py`` and ``kernels/fused_add_rms_norm.py`` for 8-bit
projections: one HBM pass reads X (and R), writes S = X + R, and writes the
normalised row as OCP e4m3 values with fp32 scales, one a row or one for each
group of columns. The reference has the unquantised norms only
(rms_norm.py:279-304, fused_add_rms_norm.py:172-188).

A rounding to 8 bits has no gradient, so these operators refuse inputs that
want one. A training step that feeds an 8-bit product and takes the gradient
of the unrounded norm calls ``rms_norm_quant_forward``, which returns RSTD,
and then ``rms_norm_backward`` / ``fused_add_rms_norm_backward``.
"""
from __future__ import annotations

import torch

from . import _lib


def _forward(X, W, eps, group_size, R, want_rstd):
    # (host time: a decode step's call is bound by it, so only what is asked for is allocated)
    dev = _lib.require_device(X, R, W)
    shape = X.shape
    hidden = shape[-1]
    assert W.dim() == 1 and W.shape[0] == hidden, f"Hidden dim mismatch: {hidden} vs {tuple(W.shape)}"
    if R is not None:
        assert R.shape == shape, f"X and R shapes differ: {tuple(shape)} vs {tuple(R.shape)}"
    group = 0
    if group_size is not None:
        group = int(group_size)
        if group not in (32, 64, 128, 256):
            raise ValueError(f"group_size must be None (the row), 32, 64, 128 or 256, got {group_size}")
        if hidden % group:
            raise ValueError(f"the hidden size {hidden} is not a multiple of group_size {group}")
    X = X.contiguous()
    W = W.contiguous()
    n_rows = X.numel() // hidden if hidden else 0
    S = X
    if R is not None:
        R = R.contiguous()
        if R.dtype != X.dtype:
            R = R.to(X.dtype)
        S = torch.empty_like(X)
    Q = torch.empty_like(X, dtype=torch.float8_e4m3fn)
    scale = torch.empty((*shape[:-1], hidden // group if group else 1), dtype=torch.float32, device=dev)
    RSTD = torch.empty(n_rows, dtype=torch.float32, device=dev) if want_rstd else None
    _lib.call_on(dev, "hk_rms_norm_quant_fwd", Q.data_ptr(), scale.data_ptr(), None if R is None else S.data_ptr(),
                 _lib.ptr(RSTD), X.data_ptr(), _lib.ptr(R), W.data_ptr(), n_rows, hidden, hidden, group,
                 _lib.dtype_code(X), _lib.dtype_code(W), eps)
    return Q, scale, S, RSTD


def rms_norm_quant_forward(X, W, eps=1e-6, group_size=None, R=None):
    """Forward. Returns (Q, scale, S, RSTD): Q float8_e4m3fn of X's shape, scale fp32 X.shape[:-1] + (groups,), S = X + R
    (X itself without R), RSTD fp32 of the rows."""
    with torch.no_grad():
        return _forward(X, W, eps, group_size, R, True)


def _no_gradient(*tensors):
    if any(t.requires_grad for t in tensors):
        raise RuntimeError("the 8-bit norms have no gradient: call them under torch.no_grad(), or use "
                           "rms_norm_quant_forward with the unquantised norms' backward")


def hilda_rms_norm_quant(X, W, eps=1e-6, group_size=None):
    """Y = RMSNorm(X) * W in 8 bits: returns (Q, scale) with Y ~ Q * scale.

    Q float8_e4m3fn; scale fp32 X.shape[:-1] + (1,), or + (H / group_size,) with group_size 32, 64, 128 or 256:
    max(max|Y| / 448, 2^-100) over the row or group.
    """
    if torch.is_grad_enabled():
        _no_gradient(X, W)
    Q, scale, _, _ = _forward(X, W, eps, group_size, None, False)
    return Q, scale


def hilda_fused_add_rms_norm_quant(X, R, W, eps=1e-6, group_size=None):
    """S = X + R, Y = RMSNorm(S) * W in 8 bits: returns (Q, scale, S) with Y ~ Q * scale (see hilda_rms_norm_quant)."""
    if torch.is_grad_enabled():
        _no_gradient(X, R, W)
    Q, scale, S, _ = _forward(X, W, eps, group_size, R, False)
    return Q, scale, S


class RMSNormQuant(torch.nn.Module):
    """``RMSNorm`` (same parameter) with the output in 8 bits; forward(x) returns (Q, scale)."""

    def __init__(self, hidden_dim, eps=1e-6, group_size=None):
        super().__init__()
        self.eps, self.group_size = eps, group_size
        self.weight = torch.nn.Parameter(torch.ones(hidden_dim))

    def forward(self, X):
        return hilda_rms_norm_quant(X, self.weight, self.eps, self.group_size)


class FusedAddRMSNormQuant(torch.nn.Module):
    """``FusedAddRMSNorm`` (same parameter) with Y in 8 bits; forward(X, R) returns (Q, scale, S)."""

    def __init__(self, hidden_dim, eps=1e-6, group_size=None):
        super().__init__()
        self.eps, self.group_size = eps, group_size
        self.weight = torch.nn.Parameter(torch.ones(hidden_dim))

    def forward(self, X, R):
        return hilda_fused_add_rms_norm_quant(X, R, self.weight, self.eps, self.group_size)
