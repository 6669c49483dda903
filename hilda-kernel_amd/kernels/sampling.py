"""Token sampling on MI355X: temperature, top-k, top-p and min-p from given uniform numbers.

The drawing side of GRPO: the ids are ``completion_ids`` and the
log-probabilities ``old_logp`` of ``hilda_grpo_loss`` (the reference scores
completions, grpo_loss.py:65-80, and draws none). The random numbers are an
input, so a draw can be repeated, and nothing is synchronised.
"""
from __future__ import annotations

import torch

from . import _lib

_workspace_bytes: dict[tuple, int] = {}  # of a shape
_TOP_K_CODE = {torch.int32: _lib.I32, torch.int64: _lib.I64}


def _rows_of(t, shape, name, device=None):
    """A per-row setting as a contiguous tensor of the rows."""
    assert t.shape == shape, f"{name} must have one value for each row {tuple(shape)}, got {tuple(t.shape)}"
    if device is not None and t.device != device:
        raise RuntimeError(f"{name} is on {t.device}, the logits on {device}")
    return t.contiguous()


def _setting(value, shape, name, device):
    """(tensor or None, number) of a float setting."""
    if not isinstance(value, torch.Tensor):
        return None, float(value)
    if value.dtype != torch.float32:
        raise TypeError(f"{name} must be float32, got {value.dtype}")
    return _rows_of(value, shape, name, device), 0.0


def hilda_sample(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Draw a token for each row of logits (..., V): returns (ids, logp) of shape (...), int64 and fp32.

    uniform: fp32 numbers in [0, 1), one a row. Filters in this order, each a number or a tensor of one value a row
    (top_k int32 or int64, the others fp32): the ``top_k`` largest logits (<= 0 or >= V: all; the lower index first
    among equal ones), of these the shortest prefix in descending order whose probability reaches ``top_p`` of theirs
    (>= 1: all), of these the tokens with at least ``min_p`` times the largest probability. The id is the first kept
    token, by index, whose cumulative probability exceeds ``uniform``. logp is its log_softmax(logits / temperature)
    over all tokens, as ``fused_selective_log_softmax`` gives it. Neither carries a gradient.

    A row that holds a NaN or +inf or nothing above -inf, or whose own temperature, uniform number or setting is NaN
    or out of range, gives id -1 and logp NaN.
    """
    dev = _lib.require_device(logits, uniform)
    shape = logits.shape[:-1]
    vocab = logits.shape[-1]
    if vocab == 0:
        raise ValueError("logits of no tokens")
    if uniform.dtype != torch.float32:
        raise TypeError(f"uniform must be float32, got {uniform.dtype}")
    uniform = _rows_of(uniform, shape, "uniform")
    t_rows, t = _setting(temperature, shape, "temperature", dev)
    p_rows, p = _setting(top_p, shape, "top_p", dev)
    m_rows, m = _setting(min_p, shape, "min_p", dev)
    k_rows, k, k_code = None, 0, 0
    if isinstance(top_k, torch.Tensor):
        if top_k.dtype not in _TOP_K_CODE:
            raise TypeError(f"top_k must be int32 or int64, got {top_k.dtype}")
        k_rows, k_code = _rows_of(top_k, shape, "top_k", dev), _TOP_K_CODE[top_k.dtype]
    else:
        k = min(max(int(top_k), 0), vocab)
    strides = logits.stride()
    if len(strides) != 2 or strides[1] != 1 or strides[0] < vocab:
        logits = logits.detach().reshape(-1, vocab).contiguous()
    rows, code = logits.shape[0], _lib.dtype_code(logits)
    ids = torch.empty(shape, dtype=torch.int64, device=dev)
    logp = torch.empty(shape, dtype=torch.float32, device=dev)
    cuts = k_rows is not None or p_rows is not None or 0 < k < vocab or p < 1
    key = (rows, vocab, cuts, code, dev.index)
    nbytes = _workspace_bytes.get(key)
    if nbytes is None:
        nbytes = _lib.load().hk_sample_workspace_size(*key)
        if len(_workspace_bytes) < 1024:
            _workspace_bytes[key] = nbytes
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _lib.call_on(dev, "hk_sample", ids.data_ptr(), logp.data_ptr(), logits.data_ptr(), uniform.data_ptr(), rows, vocab,
                 logits.stride(0) if rows > 1 else vocab, _lib.ptr(t_rows), t, _lib.ptr(k_rows), k_code, k,
                 _lib.ptr(p_rows), p, _lib.ptr(m_rows), m, code, ws.data_ptr(), nbytes)
    return ids, logp
