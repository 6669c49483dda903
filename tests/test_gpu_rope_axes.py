"""GPU parity: multi-axis RoPE against its definition in 64 bits.

Tolerance, element by element: the kernel forms x1 c - x2 s in fp32 (two
products and a sum, each within 2^-24 of its terms, so 3 * 2^-24 of
|x1 c| + |x2 s| at most) and rounds once to the type (half a step).
"""
import pytest
import torch

import oracle
from _util import gpu

from kernels import MultiAxisRotaryEmbedding, RotaryEmbedding, hilda_rope, hilda_rope_axes

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}  # half of fp16's smallest step


def _check(got, want, room, dtype, what):
    got = got.detach().cpu().double()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), f"{what}: NaNs differ"
    allowed = 3 * 2.0 ** -24 * room + HALF_STEP[dtype] * want.abs() * (1 + 1e-6) + TINY[dtype]
    off = ((got - want).abs() - allowed)[~nan]
    assert off.numel() == 0 or off.max() <= 0, f"{what}: {off.max().item():.3e} over the bound"


def _heads(g, B, H, T, D, dtype, layout):
    if layout == "bhtd":
        return torch.randn(B, H, T, D, generator=g).to(dtype)
    if layout == "bthd":
        return torch.randn(B, T, H, D, generator=g).to(dtype).transpose(1, 2)
    assert layout == "slice"  # heads of a wider projection: rows not dense
    return torch.randn(B, T, H + 3, D, generator=g).to(dtype)[:, :, 1:H + 1].transpose(1, 2)


def _positions(g, A, B, T, rows, dtype=torch.int64):
    return torch.randint(0, rows, (A, B, T), generator=g).to(dtype)


def _case(B, T, Hq, Hk, D, sections, interleaved, dtype, layout, table=torch.float32, pos=torch.int64, rows=97, seed=0):
    g = torch.Generator().manual_seed(seed)
    q, k = _heads(g, B, Hq, T, D, dtype, layout), _heads(g, B, Hk, T, D, dtype, layout)
    dq, dk = _heads(g, B, Hq, T, D, dtype, layout), _heads(g, B, Hk, T, D, dtype, layout)
    cos, sin = oracle.rope_tables(D, rows, 10000.0)
    cos, sin = cos.to(table), sin.to(table)
    positions = _positions(g, len(sections), B, T, rows, pos)
    dev = gpu()
    # (.to keeps dense layouts; the sliced one is rebuilt as a slice on the device)
    move = (lambda t: t.to(dev)) if layout != "slice" else \
        (lambda t: torch.cat((t.transpose(1, 2)[:, :, :1], t.transpose(1, 2)), 2).to(dev)[:, :, 1:].transpose(1, 2))
    qd, kd = move(q).requires_grad_(), move(k).requires_grad_()
    qo, ko = hilda_rope_axes(qd, kd, cos.to(dev), sin.to(dev), positions.to(dev), sections, interleaved)
    assert qo.dtype == dtype and qo.shape == q.shape
    gq, gk = torch.autograd.grad((qo, ko), (qd, kd), (move(dq), move(dk)))
    for got, x, inverse, what in ((qo, q, False, "q"), (ko, k, False, "k"), (gq, dq, True, "dq"), (gk, dk, True, "dk")):
        _check(got, *oracle.rope_axes_ref(x, cos[0], sin[0], positions, sections, interleaved, inverse), dtype, what)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout", ["bthd", "bhtd", "slice"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_layouts_and_types(dtype, layout, interleaved):
    _case(2, 37, 5, 2, 64, (12, 10, 10), interleaved, dtype, layout)


@pytest.mark.parametrize("T", [1, 2, 63, 257])
@pytest.mark.parametrize("layout", ["bthd", "bhtd"])
def test_lengths(T, layout):
    _case(3, T, 8, 1, 128, (16, 24, 24), False, torch.bfloat16, layout, seed=T)


@pytest.mark.parametrize("D,sections", [(2, (1,)), (2, (0, 1)), (6, (1, 1, 1)), (80, (20, 20)), (72, (12, 12, 12)),
                                        (100, (20, 15, 10, 5)), (256, (64, 0, 64)), (520, (100, 80, 80))])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_head_dims_and_sections(D, sections, dtype):
    _case(2, 11, 3, 3, D, sections, False, dtype, "bthd")


@pytest.mark.parametrize("heads", [(1, 1), (7, 1), (32, 8), (40, 40), (3, 9)])
def test_head_counts(heads):
    _case(1, 19, *heads, 64, (16, 8, 8), True, torch.bfloat16, "bthd")


@pytest.mark.parametrize("table", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("pos", [torch.int32, torch.int64])
def test_table_and_position_types(table, pos):
    _case(2, 13, 4, 2, 64, (16, 16), False, torch.float16, "bthd", table, pos)


def test_equal_positions_give_rope():
    """Positions 0..T-1 on every axis: the single-axis operator's result, bit for bit."""
    dev = gpu()
    g = torch.Generator().manual_seed(5)
    q = torch.randn(2, 33, 4, 64, generator=g).to(dev, torch.bfloat16).transpose(1, 2)
    k = torch.randn(2, 33, 2, 64, generator=g).to(dev, torch.bfloat16).transpose(1, 2)
    rot = RotaryEmbedding(64, 50).to(dev)
    want = hilda_rope(q, k, *rot(q, 33))
    multi = MultiAxisRotaryEmbedding(64, (12, 10, 10), 50).to(dev)
    multi.load_state_dict(rot.state_dict())
    got = multi(q, k, torch.arange(33, device=dev).expand(3, 1, 33))
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_positions_broadcast_over_the_batch_and_strided():
    dev = gpu()
    g = torch.Generator().manual_seed(6)
    q = torch.randn(3, 2, 10, 32, generator=g).to(dev)
    cos, sin = oracle.rope_tables(32, 40, 10000.0)
    pos = torch.randint(0, 40, (10, 2), generator=g)  # (tokens, axes) storage
    args = (q, q, cos.to(dev), sin.to(dev))
    got = hilda_rope_axes(*args, pos.to(dev).t()[:, None], (8, 8))[0]
    want = hilda_rope_axes(*args, pos.t()[:, None].expand(2, 3, 10).contiguous().to(dev), (8, 8))[0]
    assert torch.equal(got, want)
    _check(got, *oracle.rope_axes_ref(q, cos[0], sin[0], pos.t()[:, None], (8, 8)), torch.float32, "q")


def test_positions_outside_the_table_are_nan():
    dev = gpu()
    cos, sin = oracle.rope_tables(16, 8, 10000.0)
    pos = torch.tensor([[[0, 8, 3, -1, 7]], [[7, 1, 2 ** 40, 2, 0]]])
    x = torch.ones(1, 2, 5, 16)
    got = hilda_rope_axes(x.to(dev), x.to(dev), cos.to(dev), sin.to(dev), pos.to(dev), (4, 4))
    for y in got:
        _check(y, *oracle.rope_axes_ref(x, cos[0], sin[0], pos, (4, 4)), torch.float32, "y")
    assert torch.isnan(got[0][0, 0, 1, :4]).all() and not torch.isnan(got[0][0, 0, 1, 4:8]).any()


def test_far_positions_read_their_own_rows():
    """A table of 2^20 positions: rows behind the 32-bit byte offset of the start of the table (2^20 * 1024 * 4 B)."""
    dev = gpu()
    rows, half = 1 << 20, 1024
    cos = torch.zeros(rows, half, device=dev)
    sin = torch.zeros(rows, half, device=dev)
    at = torch.tensor([rows - 1, rows - 7, 5])
    g = torch.Generator().manual_seed(7)
    angle = torch.randn(3, half, generator=g, dtype=torch.float64)
    cos[at.to(dev)], sin[at.to(dev)] = angle.cos().float().to(dev), angle.sin().float().to(dev)
    x = torch.randn(1, 2, 3, 2 * half, generator=g)
    got = hilda_rope_axes(x.to(dev), x.to(dev), cos, sin, at.view(1, 1, 3).to(dev), (half,))[0]
    _check(got, *oracle.rope_axes_ref(x, cos[at.to(dev)], sin[at.to(dev)], torch.arange(3).view(1, 1, 3), (half,)),
           torch.float32, "far")


def test_misaligned_and_broadcast_inputs():
    """A view that starts off a 16-byte border, gradients that are expanded scalars, and a transposed head dim."""
    dev = gpu()
    g = torch.Generator().manual_seed(8)
    flat = torch.randn(1 + 2 * 5 * 4 * 32, generator=g).to(dev, torch.bfloat16)
    q = flat[1:].view(2, 4, 5, 32).requires_grad_()
    k = torch.randn(2, 32, 5, 4, generator=g).to(dev, torch.bfloat16).permute(0, 3, 2, 1).requires_grad_()
    cos, sin = oracle.rope_tables(32, 20, 10000.0)
    pos = _positions(g, 2, 2, 5, 20)
    qo, ko = hilda_rope_axes(q, k, cos.to(dev), sin.to(dev), pos.to(dev), (8, 8))
    (qo.sum() + 2 * ko.sum()).backward()
    for got, x, inv, what in ((qo, q, False, "q"), (ko, k, False, "k"), (q.grad, torch.ones(2, 4, 5, 32), True, "dq"),
                              (k.grad, torch.full((2, 4, 5, 32), 2.0), True, "dk")):
        _check(got, *oracle.rope_axes_ref(x, cos[0], sin[0], pos, (8, 8), inverse=inv), torch.bfloat16, what)


def test_one_gradient_only_and_differences():
    """Only q wants a gradient; it matches differences of the operator itself (linear, so exact up to rounding)."""
    dev = gpu()
    g = torch.Generator().manual_seed(9)
    q = torch.randn(1, 2, 3, 16, generator=g).to(dev).requires_grad_()
    k = torch.randn(1, 1, 3, 16, generator=g).to(dev)
    cos, sin = (t.to(dev) for t in oracle.rope_tables(16, 20, 10000.0))
    pos = _positions(g, 3, 1, 3, 20).to(dev)
    call = lambda t: hilda_rope_axes(t, k, cos, sin, pos, (4, 2, 2), True)  # noqa: E731
    weight = torch.randn(1, 2, 3, 16, generator=g).to(dev)
    qo, ko = call(q)
    (qo * weight).sum().backward()
    step = torch.randn(1, 2, 3, 16, generator=g).to(dev)
    with torch.no_grad():
        change = ((call(q + step)[0].double() - call(q - step)[0].double()) * weight.double()).sum() / 2
    # 96 products of numbers of size ~1, each output within 2^-22 of them
    assert abs(change - (q.grad.double() * step.double()).sum()) <= 96 * 4 * 2.0 ** -22 * 9


def test_gradient_of_the_gradient():
    """Linear: the second derivative along v of <w, y(q)^2> / 2 is the rotation of v back and forth, v itself."""
    dev = gpu()
    g = torch.Generator().manual_seed(11)
    q = torch.randn(1, 2, 3, 16, generator=g).to(dev).requires_grad_()
    k = torch.randn(1, 1, 3, 16, generator=g).to(dev)
    cos, sin = (t.to(dev) for t in oracle.rope_tables(16, 20, 10000.0))
    pos = _positions(g, 2, 1, 3, 20).to(dev)
    y = hilda_rope_axes(q, k, cos, sin, pos, (4, 4))[0]
    first = torch.autograd.grad((y * y).sum() / 2, q, create_graph=True)[0]
    v = torch.randn(1, 2, 3, 16, generator=g).to(dev)
    second = torch.autograd.grad(first, q, v)[0]
    # two rotations, each within 3 * 2^-24 of terms of size |v|, and cos^2 + sin^2 of fp32 tables
    assert (second - v).abs().max() <= 8 * 2.0 ** -23 * v.abs().max() * 2


def test_table_layouts():
    """Tables as rows only, cut from wider ones, laid out unlike each other, of one position, and one row for all."""
    dev = gpu()
    g = torch.Generator().manual_seed(10)
    x = torch.randn(1, 2, 6, 16, generator=g)
    cos, sin = oracle.rope_tables(16, 20, 10000.0)
    pos = _positions(g, 2, 1, 6, 20)
    wide = torch.cat((cos, sin), -1).to(dev)
    flipped = sin.to(dev).transpose(1, 2).contiguous().transpose(1, 2)
    for c, s in ((cos[0].to(dev), sin[0].to(dev)), (wide[..., :8], wide[..., 8:]), (cos.to(dev), wide[..., 8:]),
                 (cos.to(dev), flipped), (cos[:, None].to(dev)[:, 0], sin.to(dev))):
        for _ in range(2):
            got = hilda_rope_axes(x.to(dev), x.to(dev), c, s, pos.to(dev), [4, 4])[0]
            _check(got, *oracle.rope_axes_ref(x, cos[0], sin[0], pos, (4, 4)), torch.float32, "y")
    one = torch.zeros(2, 1, 6, dtype=torch.int32)
    for c, s in ((cos[:, :1], sin[:, :1]), (cos[:, :1].expand(1, 20, 8), sin[:, :1].expand(1, 20, 8))):
        got = hilda_rope_axes(x.to(dev), x.to(dev), c.to(dev), s.to(dev), one.to(dev), (4, 4))[0]
        _check(got, *oracle.rope_axes_ref(x, cos[0], sin[0], one, (4, 4)), torch.float32, "y")


def test_empty_calls():
    dev = gpu()
    cos, sin = (t.to(dev) for t in oracle.rope_tables(16, 20, 10000.0))
    for B, Hq, T in ((0, 2, 3), (2, 2, 0), (1, 0, 3)):
        q, k = torch.zeros(B, Hq, T, 16, device=dev), torch.ones(B, 1, T, 16, device=dev)
        pos = torch.zeros(2, B, T, dtype=torch.int64, device=dev)
        qo, ko = hilda_rope_axes(q, k, cos, sin, pos, (4, 4))
        assert qo.shape == q.shape and torch.equal(ko, k)  # position 0: the identity


@pytest.mark.parametrize("bad", ["pos_shape", "pos_type", "sections", "many_axes", "tables", "dtypes", "device"])
def test_refusals(bad):
    dev = gpu()
    q = torch.zeros(2, 2, 3, 16, device=dev)
    k = q
    cos = sin = torch.zeros(1, 20, 8, device=dev)
    pos = torch.zeros(2, 2, 3, dtype=torch.int64, device=dev)
    sections = (4, 4)
    if bad == "pos_shape":
        pos = pos[:, :, :2]
    elif bad == "pos_type":
        pos = pos.float()
    elif bad == "sections":
        sections = (4, 5)
    elif bad == "many_axes":
        sections = (1,) * 8
    elif bad == "tables":
        cos = cos[..., :4]
    elif bad == "dtypes":
        k = k.half()
    else:
        pos = pos.cpu()
    with pytest.raises((AssertionError, TypeError, ValueError, RuntimeError)):
        hilda_rope_axes(q, k, cos, sin, pos, sections)
