"""CPU: the 64-bit definitions of the generation-side operators against something other than their own formulas, and
the operators' refusals, none of which reaches a device."""
import ctypes
import os

import numpy as np
import pytest
import torch

import oracle
from kernels import _lib, hilda_fused_add_rms_norm_quant, hilda_rms_norm_quant, hilda_rope_axes, hilda_sample
from kernels import MultiAxisRotaryEmbedding

needs_lib = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built")


def test_axis_of_pair_by_hand():
    assert oracle.axis_of_pair((2, 1, 1), False) == [0, 0, 1, 2]
    assert oracle.axis_of_pair((4, 2, 2), True) == [0, 1, 2, 0, 1, 2, 0, 0]
    assert oracle.axis_of_pair((3, 0), True) == [0, 0, 0]
    assert oracle.axis_of_pair((0, 3), False) == [1, 1, 1]


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_axes_with_equal_positions_is_rope(interleaved):
    g = torch.Generator().manual_seed(1)
    q = torch.randn(2, 3, 9, 16, generator=g, dtype=torch.float64)
    cos, sin = oracle.rope_tables(16, 9, 10000.0)
    want = oracle.rope_ref(q, q, cos.double(), sin.double())[0]
    pos = torch.arange(9).expand(3, 1, 9)
    got, room = oracle.rope_axes_ref(q, cos[0], sin[0], pos, (4, 2, 2), interleaved)
    assert torch.allclose(got, want, rtol=0, atol=1e-12)
    assert (room >= got.abs() - 1e-12).all()
    back, _ = oracle.rope_axes_ref(got, cos[0], sin[0], pos, (4, 2, 2), interleaved, inverse=True)
    assert torch.allclose(back, q, atol=1e-6)  # cos^2 + sin^2 of fp32 tables


def test_rope_axes_each_pair_follows_its_axis():
    cos, sin = oracle.rope_tables(8, 50, 100.0)
    x = torch.ones(1, 1, 1, 8, dtype=torch.float64)
    base, _ = oracle.rope_axes_ref(x, cos[0], sin[0], torch.tensor([[[5]], [[5]], [[5]]]), (2, 1, 1))
    for axis, pairs in ((0, (0, 1)), (1, (2,)), (2, (3,))):
        pos = torch.full((3, 1, 1), 5)
        pos[axis] = 17
        y, _ = oracle.rope_axes_ref(x, cos[0], sin[0], pos, (2, 1, 1))
        moved = {i % 4 for i in torch.nonzero((y - base).flatten().abs() > 1e-9).flatten().tolist()}
        assert moved == set(pairs)


def test_norm_quant_against_the_float8_cast():
    g = torch.Generator().manual_seed(2)
    x, w = torch.randn(5, 64, generator=g), torch.randn(64, generator=g)
    v, scale, _ = oracle.norm_quant_ref(x, w)
    q = v.float().to(torch.float8_e4m3fn).double()
    assert ((q - v).abs() <= oracle.e4m3_step(torch.maximum(v.abs(), q.abs())) / 2 + 1e-6).all()
    assert torch.allclose(v.abs().amax(-1), torch.full((5,), 448.0, dtype=torch.float64))
    y = oracle.rms_norm_ref(x.double(), w.double())
    assert torch.allclose(v * scale, y)
    v, scale, _ = oracle.norm_quant_ref(torch.zeros(2, 64), w, group=32)
    assert (v == 0).all() and (scale == 2.0 ** -100).all() and scale.shape == (2, 2)


def test_sample_by_hand():
    x = torch.log(torch.tensor([[0.1, 0.4, 0.2, 0.3]], dtype=torch.float64))
    draw = lambda u, **kw: int(oracle.sample_ref(x, torch.tensor([u]), **kw)[0])  # noqa: E731
    assert [draw(u) for u in (0.0, 0.05, 0.11, 0.49, 0.51, 0.69, 0.71, 1.0)] == [0, 0, 1, 1, 2, 2, 3, 3]
    assert [draw(u, top_k=2) for u in (0.0, 0.56, 0.58, 1.0)] == [1, 1, 3, 3]
    assert [draw(u, top_p=0.75) for u in (0.0, 0.43, 0.45, 0.66, 0.68)] == [1, 1, 2, 2, 3]
    assert oracle.sample_ref(x, torch.tensor([0.5]), top_p=0.65)[2][0].tolist() == [1, 3]
    assert oracle.sample_ref(x, torch.tensor([0.5]), min_p=0.6)[2][0].tolist() == [1, 3]
    assert oracle.sample_ref(x, torch.tensor([0.5]), top_k=3, top_p=0.7, min_p=0.9)[2][0].tolist() == [1]
    # ties: the lower index first
    assert oracle.sample_ref(torch.zeros(1, 5), torch.tensor([0.5]), top_k=3)[2][0].tolist() == [0, 1, 2]
    assert oracle.sample_ref(torch.zeros(1, 5), torch.tensor([0.5]), top_p=0.5)[2][0].tolist() == [0, 1, 2]
    logp = oracle.sample_ref(x, torch.tensor([0.2]), temperature=0.5)[1]
    p = torch.tensor([0.01, 0.16, 0.04, 0.09], dtype=torch.float64)
    assert torch.allclose(logp, torch.log(p[1] / p.sum()))


def test_sample_frequencies_over_a_grid():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(1, 12, generator=g, dtype=torch.float64)
    u = (torch.arange(4000) + 0.5) / 4000
    ids = oracle.sample_ref(x.expand(4000, 12), u)[0]
    share = np.bincount(ids.numpy(), minlength=12) / 4000
    # a grid of 4000 points meets each interval to within one point
    assert np.abs(share - torch.softmax(x, -1)[0].numpy()).max() <= 1 / 4000 + 1e-9


# ---- refusals ---------------------------------------------------------------

def test_no_cpu_path():
    x = torch.zeros(2, 64)
    w = torch.ones(64)
    with torch.no_grad():
        for call in (lambda: hilda_rms_norm_quant(x, w), lambda: hilda_fused_add_rms_norm_quant(x, x, w),
                     lambda: hilda_sample(x, torch.zeros(2)),
                     lambda: hilda_rope_axes(torch.zeros(1, 1, 2, 8), torch.zeros(1, 1, 2, 8), torch.zeros(1, 4, 4),
                                             torch.zeros(1, 4, 4), torch.zeros(1, 1, 2, dtype=torch.long), (4,))):
            with pytest.raises(RuntimeError, match="ROCm"):
                call()


def test_no_gradient_through_eight_bits():
    x, w = torch.zeros(2, 64, requires_grad=True), torch.ones(64)
    with pytest.raises(RuntimeError, match="no gradient"):
        hilda_rms_norm_quant(x, w)
    with pytest.raises(RuntimeError, match="no gradient"):
        hilda_fused_add_rms_norm_quant(x.detach(), x, w)


def test_module_refuses_sections():
    with pytest.raises(ValueError, match="sum to"):
        MultiAxisRotaryEmbedding(16, (4, 2))
    m = MultiAxisRotaryEmbedding(16, (4, 2, 2), 32)
    assert set(m.state_dict()) == {"inv_freq", "cos_cached", "sin_cached"}


def _einval(status, fragment):
    assert status == -1
    assert fragment in _lib.last_error(), _lib.last_error()


@needs_lib
def test_rope_axes_refusals():
    lib = _lib.load()
    p = ctypes.c_void_p(256)  # never dereferenced: the checks come first

    def call(sections=(16, 24, 24), axes=None, interleaved=0, B=2, T=4, D=128, dtype=2, cs=0, pos=_lib.I64, stride=128,
             rows=100, ld=64, ptr=p):
        s = _lib.RopeAxesShape(B=B, T=T, D=D, Hq=2, Hk=1, table_rows=rows, table_ld=ld, interleaved=interleaved,
                               pos_type=pos, dtype_x=dtype, dtype_cs=cs, axes=len(sections) if axes is None else axes)
        s.sections[:] = (tuple(sections) + (0, 0, 0, 0))[:4]
        s.q_in[:] = (stride,) * 3
        return lib.hk_rope_axes(ptr, p, p, p, p, p, p, ctypes.addressof(s), None)

    _einval(call(D=127), "even")
    _einval(call(sections=(16, 24, 23)), "sum to")
    _einval(call(sections=(70, -3, -3)), "negative")
    _einval(call(axes=5), "axes")
    _einval(call(axes=0), "axes")
    # (their sum passes 64 bits and comes to 64)
    _einval(call(sections=(1 << 62, 1 << 62, 1 << 62, (1 << 62) + 64)), "pairs of")
    # axis 1 of 2 over 64 pairs owns at most 32
    _einval(call(sections=(30, 34), interleaved=1), "interleaved section")
    _einval(call(sections=(0, 32, 32), interleaved=1), "interleaved section")
    _einval(call(dtype=7), "dtype")
    _einval(call(cs=7), "cos/sin dtype")
    _einval(call(pos=_lib.F32), "positions")
    _einval(call(stride=-1), "negative strides")
    _einval(call(ld=63), "row stride")
    _einval(call(B=1 << 20, T=1 << 20), "too large")
    _einval(call(B=-1), "invalid shape")
    _einval(call(ptr=None), "null")
    assert call(B=0, ptr=None) == 0
    _einval(lib.hk_rope_axes(p, p, p, p, p, p, p, None, None), "null")


@needs_lib
def test_norm_quant_refusals():
    lib = _lib.load()
    p = ctypes.c_void_p(256)

    def call(q=p, s=p, r=p, rows=4, cols=256, ld=256, group=0, dx=2, dw=2):
        return lib.hk_rms_norm_quant_fwd(q, p, s, None, p, r, p, rows, cols, ld, group, dx, dw, 1e-6, None)

    _einval(call(dx=7), "dtype")
    _einval(call(dx=1, dw=2), "dtype pair")
    _einval(call(rows=-1), "shape")
    _einval(call(cols=0), "shape")
    _einval(call(ld=255), "stride")
    _einval(call(group=48), "group")
    _einval(call(cols=288, ld=288, group=64), "multiple")
    _einval(call(s=None), "together")
    _einval(call(q=None), "null")
    _einval(call(rows=1 << 31), "too large")
    assert call(rows=0) == 0


@needs_lib
def test_sample_refusals():
    lib = _lib.load()
    p = ctypes.c_void_p(256)

    def call(ids=p, rows=4, cols=100, ld=100, t=1.0, k_rows=None, k_type=0, top_p=1.0, min_p=0.0, dtype=2, ws=p):
        return lib.hk_sample(ids, p, p, p, rows, cols, ld, None, t, k_rows, k_type, 0, None, top_p, None, min_p, dtype,
                             ws, 1 << 20, None)

    _einval(call(dtype=5), "dtype")
    _einval(call(rows=-1), "shape")
    _einval(call(cols=0), "shape")
    _einval(call(cols=(1 << 30) + 1, ld=1 << 31), "too large")
    _einval(call(ld=99), "stride")
    for t in (0.0, -1.0, float("nan"), float("inf")):
        _einval(call(t=t), "temperature")
    for v in (-0.1, 1.1, float("nan")):
        _einval(call(top_p=v), "top_p")
        _einval(call(min_p=v), "min_p")
    _einval(call(k_rows=p, k_type=_lib.F32), "top_k")
    _einval(call(ids=None), "null")
    _einval(call(ws=None), "workspace")
    _einval(call(ws=ctypes.c_void_p(264)), "aligned")
    assert call(rows=0) == 0
    # more for the cuts' bins, nothing that grows with rows * cols but the runs' records
    small, large = (lib.hk_sample_workspace_size(256, 151936, cuts, 2, 0) for cuts in (0, 1))
    assert 0 < small < large < 64 * 2 ** 20
    assert lib.hk_sample_workspace_size(1 << 20, 300, 1, 2, 0) < 64 * 2 ** 20
    assert lib.hk_sample_workspace_size(-1, 300, 1, 2, 0) == lib.hk_sample_workspace_size(4, 0, 1, 2, 0) == 0
