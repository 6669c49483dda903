"""GPU parity: the norms with an e4m3 output against their definition in 64 bits.

Tolerances. s: the bits of x + r in the type. scale: the sum of squares adds at
most 16 terms a lane and 16 + 6 partial sums (cols / 1024 a lane in the long
form), each sum within 2^-24, halved by the root; the root, the products and
the division add a handful of 2^-24 and two 2^-23: (cols / 1024 + 64) * 2^-24
covers them. q: half an e4m3 step at the exact y / scale, whose own relative
error is within twice that.
"""
import pytest
import torch

import oracle
from _util import gpu

from kernels import (FusedAddRMSNorm, FusedAddRMSNormQuant, RMSNorm, RMSNormQuant, hilda_fused_add_rms_norm_quant,
                     hilda_rms_norm_quant)
from kernels.fused_add_rms_norm import fused_add_rms_norm_backward
from kernels.rms_norm import rms_norm_backward
from kernels.rms_norm_quant import rms_norm_quant_forward

pytestmark = pytest.mark.gpu


def _inputs(rows, cols, dtype, add, seed=0, w_dtype=None):
    g = torch.Generator().manual_seed(seed)
    x = (3 * torch.randn(rows, cols, generator=g)).to(dtype)
    w = (1 + 0.2 * torch.randn(cols, generator=g)).to(w_dtype or dtype)
    r = torch.randn(rows, cols, generator=g).to(dtype) if add else None
    return x, w, r


def _check(got, x, w, r, eps=1e-6, group=None):
    q, scale = got[0].cpu().double(), got[1].cpu().double()
    v, want, s = oracle.norm_quant_ref(x, w, r, eps, group)
    cols = x.shape[-1]
    rel = (cols / 1024 + 64) * 2.0 ** -24
    assert got[0].dtype == torch.float8_e4m3fn and got[1].dtype == torch.float32
    assert scale.shape == want.shape and q.shape == x.shape
    assert ((scale - want).abs() <= rel * want).all(), f"scale off by {((scale - want).abs() / want).max():.3e}"
    allowed = oracle.e4m3_step(torch.maximum(v.abs(), q.abs())) / 2 + 2 * rel * v.abs()
    off = (q - v).abs() - allowed
    assert off.max() <= 0, f"q over the bound by {off.max().item():.3e}"
    if r is not None:
        assert torch.equal(got[2].cpu(), s)


def _run(x, w, r, eps=1e-6, group=None):
    dev = gpu()
    if r is None:
        return hilda_rms_norm_quant(x.to(dev), w.to(dev), eps, group)
    return hilda_fused_add_rms_norm_quant(x.to(dev), r.to(dev), w.to(dev), eps, group)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("group", [None, 32, 64, 128, 256])
def test_types_and_groups(dtype, add, group):
    x, w, r = _inputs(37, 1280, dtype, add)
    _check(_run(x, w, r, group=group), x, w, r, group=group)


@pytest.mark.parametrize("cols", [1, 2, 7, 8, 9, 255, 511, 1023, 2049, 4096, 4099, 8192, 16384, 20000, 32767, 65537])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_row_lengths(cols, dtype):
    """Odd lengths (rows at element alignment), and rows past what registers hold."""
    x, w, r = _inputs(5, cols, dtype, True, seed=cols)
    _check(_run(x, w, r), x, w, r)


@pytest.mark.parametrize("cols,group", [(32, 32), (256, 256), (16640, 256), (65792, 256), (33280, 64), (66048, 32)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_groups_of_short_and_long_rows(cols, group, dtype):
    x, w, r = _inputs(3, cols, dtype, True, seed=1)
    _check(_run(x, w, r, group=group), x, w, r, group=group)
    _check(_run(x, w, None, group=group), x, w, None, group=group)


@pytest.mark.parametrize("rows", [0, 1, 2, 3, 1025])
def test_row_counts(rows):
    x, w, r = _inputs(rows, 512, torch.bfloat16, True)
    got = _run(x, w, r)
    assert got[0].shape == (rows, 512) and got[1].shape == (rows, 1)
    if rows:
        _check(got, x, w, r)


def test_fp32_weight_and_leading_shape():
    x, w, r = _inputs(12, 384, torch.bfloat16, True, w_dtype=torch.float32)
    q, scale, s = _run(x.view(3, 4, 384), w, r.view(3, 4, 384), group=128)
    assert q.shape == (3, 4, 384) and scale.shape == (3, 4, 3) and s.shape == (3, 4, 384)
    _check((q.view(12, 384), scale.view(12, 3), s.view(12, 384)), x, w, r, group=128)


def test_misaligned_and_strided_inputs():
    dev = gpu()
    g = torch.Generator().manual_seed(3)
    flat = torch.randn(1 + 6 * 256, generator=g).to(torch.bfloat16)
    x = flat[1:].view(6, 256)
    wide = torch.randn(6, 300, generator=g).to(torch.bfloat16)
    w = torch.ones(256, dtype=torch.bfloat16)
    got = hilda_fused_add_rms_norm_quant(flat.to(dev)[1:].view(6, 256), wide.to(dev)[:, 7:263], w.to(dev), 1e-6, 64)
    _check(got, x, w, wide[:, 7:263], group=64)


def test_zero_rows_and_groups():
    x, w, _ = _inputs(4, 512, torch.bfloat16, False)
    x[1] = 0
    x[2, 128:256] = 0
    q, scale = _run(x, w, None, group=128)
    _check((q, scale), x, w, None, group=128)
    assert (scale[1] == 2.0 ** -100).all() and scale[2, 1] == 2.0 ** -100
    assert (q[1].float() == 0).all() and (q[2, 128:256].float() == 0).all()


def test_largest_value_maps_to_448():
    x, w, r = _inputs(64, 1024, torch.bfloat16, True)
    q, _, _ = _run(x, w, r, group=64)
    assert (q.float().view(64, 16, 64).abs().amax(-1) == 448).all()


def test_nan_and_infinity_stay_in_their_rows():
    x, w, _ = _inputs(5, 512, torch.float16, False)
    x[1, 7], x[3, 200] = float("nan"), float("inf")
    good = [0, 2, 4]
    for group in (None, 128):
        q, scale = _run(x, w, None, group=group)
        _check((q[good], scale[good]), x[good], w, None, group=group)
        assert torch.isnan(scale[1]).all() and torch.isnan(q[1].float()).all()
        # an infinite mean square: 1 / rms = 0, so the row is 0 * finite, and NaN at the infinity
        assert torch.isnan(q[3, 200].float())
    w2 = w.clone()
    w2[130] = float("nan")
    q, scale = _run(x[good], w2, None, group=128)
    assert torch.isnan(scale[:, 1]).all() and not torch.isnan(scale[:, [0, 2, 3]]).any()


def test_repeats_are_equal():
    x, w, r = _inputs(300, 4096, torch.bfloat16, True)
    a, b = _run(x, w, r, group=128), _run(x, w, r, group=128)
    assert all(torch.equal(s.view(torch.uint8) if s.dtype == torch.float8_e4m3fn else s,
                           t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t) for s, t in zip(a, b))


def test_modules_take_the_unquantised_state():
    dev = gpu()
    x, w, r = _inputs(6, 256, torch.float32, True)
    plain, quant = FusedAddRMSNorm(256), FusedAddRMSNormQuant(256, group_size=64)
    plain.weight.data.copy_(w)
    quant.load_state_dict(plain.state_dict())
    with torch.no_grad():
        _check(quant.to(dev)(x.to(dev), r.to(dev)), x, w, r, group=64)
        single = RMSNormQuant(256)
        single.load_state_dict({**RMSNorm(256).state_dict(), "weight": w})
        _check(single.to(dev)(x.to(dev)), x, w, None)
    with pytest.raises(RuntimeError, match="no gradient"):
        quant(x.to(dev), r.to(dev))


def test_backward_of_the_unrounded_norm():
    """What the forward hands on (S, RSTD) is what the unquantised norms' backward takes."""
    dev = gpu()
    x, w, r = _inputs(40, 512, torch.float32, True)
    g = torch.Generator().manual_seed(4)
    dy = torch.randn(40, 512, generator=g)
    _, _, S, rstd = rms_norm_quant_forward(x.to(dev), w.to(dev), 1e-6, 128, r.to(dev))
    dx, dr, dw = fused_add_rms_norm_backward(dy.to(dev), None, S, w.to(dev), rstd)
    want_dx, want_dw = oracle.rms_norm_bwd_closed_form(dy, (x + r).double(), w.double())
    assert torch.allclose(dx.cpu().double(), want_dx, rtol=1e-5, atol=1e-5) and torch.equal(dx, dr)
    assert torch.allclose(dw.cpu().double(), want_dw, rtol=1e-5, atol=1e-5)
    _, _, S, rstd = rms_norm_quant_forward(x.to(dev), w.to(dev))
    got = rms_norm_backward(dy.to(dev), S, w.to(dev), rstd)
    assert torch.allclose(got[0].cpu().double(), oracle.rms_norm_bwd_closed_form(dy, x.double(), w.double())[0],
                          rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("bad", ["group", "divides", "weight", "residual", "dtype", "device"])
def test_refusals(bad):
    dev = gpu()
    x, w, group, r = torch.zeros(2, 96, device=dev), torch.ones(96, device=dev), None, torch.zeros(2, 96, device=dev)
    if bad == "group":
        group = 48
    elif bad == "divides":
        group = 64
    elif bad == "weight":
        w = torch.ones(95, device=dev)
    elif bad == "residual":
        r = r[:1]
    elif bad == "dtype":
        x = x.double()
    else:
        w = w.cpu()
    with pytest.raises((AssertionError, TypeError, ValueError, RuntimeError)):
        hilda_fused_add_rms_norm_quant(x, r, w, 1e-6, group)
