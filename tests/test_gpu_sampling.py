"""GPU parity: token sampling against its definition in 64 bits, row by row.

The ids have to be equal. Both sides compare cumulative masses held to better
than 1e-11 of the total with u * total; a token of a row of V has some 1 / V of
it, so a draw lands in between with a probability of about V * 1e-11 (1e-6 at
V = 1e5, for any of the rows below less than 1e-3 in all).

logp: the sum of V fp32 exponentials adds ceil(V / 1024) terms a lane and 16 + 6
partial sums, each within 2^-24; an exponential's argument, of size |z - max|
log2(e), is off by 2^-23 of itself, weighted by its share of the sum, whose mean
|z - max| is under 32 here; the instructions for 2^x and log2 add a few 2^-23.
"""
import math

import pytest
import torch

import oracle
from _util import gpu

from kernels import _lib, fused_selective_log_softmax, hilda_grpo_loss, hilda_sample

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _check(x, u, got=None, **kw):
    dev = gpu()
    if got is None:
        on = {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
        got = hilda_sample(x.to(dev), u.to(dev), **on)
    ids, logp = got[0].cpu(), got[1].cpu().double()
    assert ids.dtype == torch.int64 and got[1].dtype == torch.float32
    want, want_logp, _ = oracle.sample_ref(x, u, **kw)
    assert torch.equal(ids, want), f"ids differ at {torch.nonzero(ids != want).flatten().tolist()[:8]}: " \
        f"{ids[ids != want].tolist()[:8]} against {want[ids != want].tolist()[:8]}"
    assert torch.equal(torch.isnan(logp), torch.isnan(want_logp))
    fine = ~torch.isnan(want_logp)
    allowed = (x.shape[-1] / 1024 + 64) * 2.0 ** -24 + 40 * 2.0 ** -23 + 2.0 ** -22 * want_logp[fine].abs()
    assert ((logp[fine] - want_logp[fine]).abs() <= allowed).all(), (logp[fine] - want_logp[fine]).abs().max()
    return ids


def _rows(rows, V, dtype, seed=0, lo=1.0, hi=6.0):
    g = torch.Generator().manual_seed(seed)
    sharp = lo + (hi - lo) * torch.rand(rows, 1, generator=g)
    return (torch.randn(rows, V, generator=g) * sharp).to(dtype), torch.rand(rows, generator=g), g


FILTERS = {"none": {}, "t": dict(temperature=0.7), "k": dict(top_k=20), "k1": dict(top_k=1), "p": dict(top_p=0.9),
           "m": dict(min_p=0.05), "kp": dict(top_k=100, top_p=0.8),
           "kpm": dict(temperature=1.3, top_k=300, top_p=0.95, min_p=0.02), "pm": dict(top_p=0.5, min_p=0.3),
           "p0": dict(top_p=0.0), "m1": dict(min_p=1.0), "ktail": dict(top_k=900), "p9999": dict(top_p=0.9999)}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", list(FILTERS))
def test_filters(dtype, name):
    x, u, _ = _rows(24, 1003, dtype, seed=len(name))
    _check(x, u, **FILTERS[name])


@pytest.mark.parametrize("V", [1, 2, 3, 7, 8, 9, 63, 64, 65, 511, 513, 1024, 8191, 8193, 16385, 50257, 151936])
@pytest.mark.parametrize("name", ["none", "kpm", "p"])
def test_vocabularies(V, name):
    x, u, _ = _rows(4, V, torch.bfloat16, seed=V)
    _check(x, u, **FILTERS[name])


@pytest.mark.parametrize("dtype", TYPES)
def test_large_vocabulary_each_type(dtype):
    x, u, _ = _rows(3, 128256, dtype, seed=3)
    _check(x, u, top_p=0.99)
    _check(x, u, top_k=5000, top_p=0.97)


@pytest.mark.parametrize("dtype", TYPES)
def test_settings_of_each_row(dtype):
    x, u, g = _rows(40, 5003, dtype, seed=4)
    temperature = 0.3 + 2 * torch.rand(40, generator=g)
    top_k = torch.randint(-2, 6000, (40,), generator=g)
    top_k[::3] = torch.randint(1, 30, (14,), generator=g)
    top_p = 0.3 + 0.8 * torch.rand(40, generator=g)  # some above 1: off
    min_p = (0.4 * torch.rand(40, generator=g) - 0.2).clamp_min(0)
    _check(x, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    _check(x, u, temperature=temperature, top_k=top_k.int(), top_p=0.9, min_p=min_p)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kw", [{}, dict(top_k=5), dict(top_k=100), dict(top_p=0.3), dict(top_p=0.37),
                                dict(top_k=333, top_p=0.6), dict(min_p=0.5)])
def test_ties(dtype, kw):
    """Few distinct values: the cut falls inside a run of equal logits and the lowest indices stay."""
    g = torch.Generator().manual_seed(5)
    x = torch.randint(-2, 3, (16, 2053), generator=g).to(dtype)
    x[3] = 0
    x[4] = -7.5
    x[5, ::2], x[5, 1::2] = 0.0, -0.0  # equal, though their bits differ
    _check(x, torch.rand(16, generator=g), **kw)


@pytest.mark.parametrize("kw", [{}, dict(top_k=3), dict(top_p=0.9), dict(min_p=0.1), dict(top_k=40, top_p=0.5)])
def test_masked_tokens(kw):
    g = torch.Generator().manual_seed(6)
    x = (3 * torch.randn(12, 3001, generator=g)).to(torch.bfloat16)
    x[0, :2990] = -math.inf
    x[1] = -math.inf
    x[1, 1234] = -5.0  # the only one left
    x[2, 1:] = -math.inf
    x[3, :-1] = -math.inf
    x[4] = torch.finfo(torch.bfloat16).min  # a mask of the type's lowest value everywhere: uniform
    x[5, 5:] = torch.finfo(torch.bfloat16).min
    ids = _check(x, torch.rand(12, generator=g), **kw)
    assert ids[1] == 1234 and ids[2] == 0 and ids[3] == 3000


def test_rows_without_a_distribution():
    g = torch.Generator().manual_seed(7)
    x = torch.randn(8, 777, generator=g)
    x[1, 3], x[2, 776], x[3], x[4, 0] = math.nan, math.inf, -math.inf, math.nan
    x[4, 1:] = -math.inf
    x[5] = math.nan
    for kw in ({}, dict(top_k=4), dict(top_p=0.5), dict(min_p=0.2)):
        ids = _check(x, torch.rand(8, generator=g), **kw)
        assert (ids[1:6] == -1).all() and (ids[[0, 6, 7]] >= 0).all()


def test_settings_out_of_range():
    g = torch.Generator().manual_seed(8)
    x = torch.randn(9, 100, generator=g)
    u = torch.tensor([0.5, -0.1, 1.5, math.nan, 0.5, 0.5, 0.5, 0.5, 0.5])
    t = torch.tensor([1.0, 1, 1, 1, 0.0, -1.0, math.nan, math.inf, 1])
    p = torch.tensor([1.0, 1, 1, 1, 1, 1, 1, 1, math.nan])
    ids = _check(x, u, temperature=t, top_p=p)
    assert ids[0] >= 0 and (ids[1:] == -1).all()
    # out of range but with an order: as the nearest bound
    _check(x, torch.rand(9, generator=g), top_p=torch.full((9,), -1.0), min_p=torch.full((9,), -1.0))
    _check(x, torch.rand(9, generator=g), min_p=torch.full((9,), 3.0))


@pytest.mark.parametrize("dtype", TYPES)
def test_ends_of_the_unit_interval(dtype):
    x, _, _ = _rows(6, 4001, dtype, seed=9)
    x[0, 0] = x[1, -1] = -math.inf
    for u in (0.0, 1.0, 1 - 2.0 ** -24, 2.0 ** -30):
        for name in ("none", "k", "p", "m"):
            _check(x, torch.full((6,), u), **FILTERS[name])


def test_extreme_logits_and_temperatures():
    g = torch.Generator().manual_seed(10)
    base = torch.randn(6, 900, generator=g)
    u = torch.rand(6, generator=g)
    for scale in (1e-38, 1e-20, 1e6, 3e37):
        for kw in ({}, dict(top_k=7), dict(top_p=0.6)):
            _check(base * scale, u, **kw)
    for t in (2.0 ** -64, 1e-3, 1e4, 2.0 ** 64):
        for kw in ({}, dict(top_k=7), dict(top_p=0.6), dict(min_p=0.3)):
            _check(base, u, temperature=t, **kw)
    wide = base.clone()
    wide[:, ::2] = -3e38
    wide[:, 1] = 3e38
    _check(wide, u, top_k=5, top_p=0.5)


def test_peaked_and_flat_rows():
    g = torch.Generator().manual_seed(11)
    x = 0.01 * torch.randn(8, 20011, generator=g)
    x[:4, 777] = torch.tensor([5.0, 20.0, 50.0, 300.0])
    for kw in ({}, dict(top_k=50), dict(top_p=0.95), dict(top_p=0.999999), dict(min_p=1e-6), dict(top_k=2, top_p=0.9999)):
        _check(x, torch.rand(8, generator=g), **kw)


def test_shapes_strides_and_alignment():
    dev = gpu()
    x, u, _ = _rows(12, 999, torch.bfloat16, seed=12)
    want = _check(x, u, top_k=50)
    wide = torch.zeros(12, 1200, dtype=torch.bfloat16, device=dev)
    wide[:, 3:1002] = x.to(dev)
    assert torch.equal(hilda_sample(wide[:, 3:1002], u.to(dev), top_k=50)[0].cpu(), want)
    ids, logp = hilda_sample(x.to(dev).view(3, 4, 999), u.to(dev).view(3, 4), top_k=50)
    assert ids.shape == logp.shape == (3, 4) and torch.equal(ids.cpu().view(-1), want)
    turned = x.to(dev).t().contiguous().t()  # columns contiguous
    assert torch.equal(hilda_sample(turned, u.to(dev), top_k=50)[0].cpu(), want)
    same = x[:1].to(dev).expand(12, 999)  # one row for all draws
    assert torch.equal(hilda_sample(same, u.to(dev), top_k=50)[0].cpu(), oracle.sample_ref(x[:1].expand(12, 999), u, top_k=50)[0])
    ids, logp = hilda_sample(x[0].to(dev), u[0].to(dev), top_k=50)
    assert ids.shape == logp.shape == () and ids.item() == want[0]
    ids, logp = hilda_sample(x[:0].to(dev), u[:0].to(dev))
    assert ids.shape == (0,)


def test_draws_follow_the_probabilities():
    """A grid of u over one row: each token is drawn as often as its share, to within one point of the grid."""
    dev = gpu()
    g = torch.Generator().manual_seed(13)
    x = torch.randn(1, 300, generator=g)
    n = 20000
    u = ((torch.arange(n, dtype=torch.float64) + 0.5) / n).float()
    ids, _ = hilda_sample(x.to(dev).expand(n, 300), u.to(dev), top_p=0.9)
    kept = oracle.sample_ref(x, u[:1], top_p=0.9)[2][0]
    p = torch.zeros(300, dtype=torch.float64)
    p[kept] = torch.softmax(x.double(), -1)[0][kept]
    share = torch.bincount(ids.cpu(), minlength=300) / n
    # (u in fp32 moves a point by 2^-25 at most)
    assert (share - p / p.sum()).abs().max() <= 1.01 / n


def test_repeats_are_equal():
    dev = gpu()
    x, u, _ = _rows(64, 32000, torch.bfloat16, seed=14)
    x, u = x.to(dev), u.to(dev)
    a, b = hilda_sample(x, u, 0.9, 80, 0.9, 0.01), hilda_sample(x, u, 0.9, 80, 0.9, 0.01)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_many_rows():
    x, u, _ = _rows(1500, 130, torch.float16, seed=15)
    _check(x, u, top_k=40, top_p=0.9)


def test_rollout_feeds_grpo():
    """Draw completions, take their log-probabilities as old_logp: the policy's ratio is 1, nothing is clipped, and the
    loss is the mean of -advantage."""
    dev = gpu()
    B, L, V = 3, 6, 1031
    g = torch.Generator(device=dev).manual_seed(16)
    logits = (2 * torch.randn(B, L + 1, V, generator=g, device=dev)).requires_grad_()
    u = torch.rand(B, L, generator=g, device=dev)
    ids, logp = hilda_sample(logits[:, :-1], u, temperature=0.9, top_k=50, top_p=0.95)
    again = fused_selective_log_softmax(logits.detach(), ids, temperature=0.9)
    assert torch.allclose(logp, again, rtol=0, atol=2e-5)
    adv = torch.randn(B, generator=g, device=dev)
    loss, _, clip = hilda_grpo_loss(logits, ids, adv, old_logp=logp, temperature=0.9)
    loss.backward()
    # ratio = exp(difference of two fp32 log-probabilities, each within 2e-5)
    assert abs(loss.item() + adv.mean().item()) <= 4e-5 * adv.abs().max().item() + 1e-6
    assert clip.item() == 0 and torch.isfinite(logits.grad).all()


@pytest.mark.parametrize("bad", ["uniform_type", "uniform_shape", "temperature", "setting_type", "setting_shape", "top_k",
                                 "dtype", "vocab", "device"])
def test_refusals(bad):
    dev = gpu()
    x, u, kw = torch.zeros(4, 10, device=dev), torch.zeros(4, device=dev), {}
    if bad == "uniform_type":
        u = u.double()
    elif bad == "uniform_shape":
        u = u[:3]
    elif bad == "temperature":
        kw = dict(temperature=0.0)
    elif bad == "setting_type":
        kw = dict(top_p=u.double())
    elif bad == "setting_shape":
        kw = dict(min_p=u[:1])
    elif bad == "top_k":
        kw = dict(top_k=u)
    elif bad == "dtype":
        x = x.double()
    elif bad == "vocab":
        x = x[:, :0]
    else:
        u = u.cpu()
    with pytest.raises((AssertionError, TypeError, ValueError, RuntimeError)):
        hilda_sample(x, u, **kw)


def test_workspace_is_checked():
    dev = gpu()
    x, u = torch.zeros(4, 5000, device=dev), torch.zeros(4, device=dev)
    ids, logp = torch.empty(4, dtype=torch.int64, device=dev), torch.empty(4, device=dev)
    need = _lib.load().hk_sample_workspace_size(4, 5000, 1, _lib.F32, dev.index)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    for nbytes, ok in ((need, True), (need - 256, False)):
        status = _lib.load().hk_sample(ids.data_ptr(), logp.data_ptr(), x.data_ptr(), u.data_ptr(), 4, 5000, 5000, None, 1.0,
                                       None, 0, 7, None, 1.0, None, 0.0, _lib.F32, ws.data_ptr(), nbytes,
                                       _lib.stream_of(dev))
        assert (status == 0) == ok
    assert "workspace too small" in _lib.last_error()
    assert ids.tolist() == [0] * 4


@pytest.mark.parametrize("rows", [1, 5, 600, 1100])
@pytest.mark.parametrize("dtype", TYPES)
def test_ways_a_call_is_cut_up(rows, dtype):
    """Few rows are split over many blocks, many rows take one block each, with runs of 512 to 2048 columns."""
    V = 40011 if rows <= 5 else 2500
    x, u, g = _rows(rows, V, dtype, seed=rows)
    _check(x, u, temperature=0.8)
    _check(x, u, temperature=0.8, top_k=60, top_p=0.9)
    _check(x, u, temperature=0.4, top_p=0.97, min_p=0.001)


def test_bf16_values_outside_the_bins_of_one_value():
    """bf16 logits of 2^8 and more, below 2^-16, and rows whose maximum is one of those."""
    g = torch.Generator().manual_seed(17)
    x = torch.randn(10, 6007, generator=g)
    x[0] *= 300
    x[1] *= 2.0 ** -18
    x[2] = x[2].clamp(max=0)  # (the maximum is 0)
    x[3] = -x[3].abs() - 2.0 ** -17
    x[4] = 0
    x[4, 100:200] = 2.0 ** -20 * torch.randn(100, generator=g)
    x[5, ::3] *= 2.0 ** -17
    x[6] -= 400
    x[7, 11] = 256.0
    x[8] = torch.where(x[8] > 0, 255.0, -257.0)
    x[9, :5000] = -math.inf
    x = x.to(torch.bfloat16)
    u = torch.rand(10, generator=g)
    for kw in ({}, dict(temperature=0.01), dict(temperature=30.0), dict(top_k=7), dict(top_k=3000), dict(top_p=0.4),
               dict(top_p=0.999), dict(temperature=0.03, top_p=0.9), dict(top_k=2000, top_p=0.6, min_p=1e-3),
               dict(temperature=200.0, top_p=0.7)):
        _check(x, u, **kw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 24, 300])
def test_few_kept_of_many(dtype, rows):
    """top-k small enough for a list of candidates, up to where it is not, for one k and a k each."""
    V = 20011
    x, u, g = _rows(rows, V, dtype, seed=rows)
    for k in (1, 2, 50, 160, 161, 207, 208, 209, 257):
        _check(x, u, top_k=k)
    _check(x, u, top_k=50, top_p=0.9, min_p=0.01)
    _check(x, u, top_k=208, top_p=0.7, temperature=2.5)
    k = torch.randint(1, 230, (rows,), generator=g)
    _check(x, u, top_k=k, top_p=0.95)
    _check(x, u, top_k=k * (torch.arange(rows) % 3 > 0), min_p=torch.rand(rows, generator=g) * 0.1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [40009, 151936])
def test_more_candidates_than_a_list_holds(dtype, V):
    """Ties at the k-th logit: more than a list holds, in one part of a row and over all of them, and just as many."""
    g = torch.Generator().manual_seed(V)
    x = (0.5 * torch.randn(10, V, generator=g)).clamp(-4, 2.5).to(dtype)
    x[0] = 1.0
    x[1, :5000] = 3.0
    x[2, torch.randperm(V, generator=g)[:900]] = 3.0
    x[3, torch.randperm(V, generator=g)[:768]] = 3.0
    x[4, torch.randperm(V, generator=g)[:769]] = 3.0
    x[5, -513:] = 3.0
    x[6, :512] = 3.0
    x[7] = torch.finfo(dtype).min
    x[8, 3::7] = -math.inf
    x[8, 5::7] = math.nan
    x[9, 40:] = -math.inf
    u = torch.rand(10, generator=g)
    for kw in (dict(top_k=60), dict(top_k=60, top_p=0.6), dict(top_k=1), dict(top_k=200, min_p=0.2),
               dict(top_k=torch.full((10,), 77), top_p=0.9)):
        _check(x, u, **kw)
    many = torch.arange(300) % 10
    _check(x[many, :40009], u[many], top_k=60, top_p=0.8)
    _check(x[many, :40009], u[many], top_k=torch.full((300,), 33))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 24, 300])
def test_one_filter_over_many_kept(dtype, rows):
    """One filter whose cut lies among many different logits, next to min-p and ties at the cut."""
    V = 30011
    x, u, g = _rows(rows, V, dtype, seed=rows + 1, lo=0.3, hi=4.0)
    some = torch.rand(rows, V, generator=g) < 0.02
    x = torch.where(some, x[:, :1].expand(rows, V), x)  # 600 equal logits somewhere in the row
    for kw in (dict(top_p=0.95), dict(top_p=0.5), dict(top_k=3000), dict(top_k=301), dict(top_k=3000, min_p=0.001),
               dict(top_p=0.9, min_p=0.05), dict(top_p=0.7, temperature=3.0), dict(top_k=25000),
               dict(top_p=torch.rand(rows, generator=g)), dict(top_k=torch.randint(1, V, (rows,), generator=g))):
        _check(x, u, **kw)


@pytest.mark.parametrize("dtype", TYPES)
def test_cuts_among_masked_tokens(dtype):
    """A top-k larger than what is left, masks of the lowest value, ties of all a mask leaves."""
    V = 9001
    x, u, g = _rows(8, V, dtype, seed=9)
    x[0, 300:] = -math.inf
    x[1, 300:] = torch.finfo(dtype).min
    x[2, :8700] = -math.inf
    x[3, 400:] = -60.0
    x[4, 1:] = -math.inf
    x[5] = -math.inf
    x[5, ::30] = 2.0
    x[6] = x[6].abs() * 200
    for kw in (dict(top_k=400), dict(top_k=8999), dict(top_p=0.999), dict(top_k=500, top_p=0.99), dict(top_k=1000, min_p=0.5)):
        _check(x, u, **kw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [40009, 151936])
def test_parts_of_a_row(dtype, V):
    """Rows that several blocks share: draws at both ends of each share, shares without mass, ties over all of them."""
    rows = 30
    x, u, g = _rows(rows, V, dtype, seed=V + 1, lo=0.5, hi=5.0)
    x[0] = 0.0
    x[1, : V // 3] = -math.inf
    x[2, V // 5:] = -math.inf
    x[3, V // 5: -V // 5] = torch.finfo(dtype).min
    x[4] = torch.where(torch.rand(V, generator=g) < 0.5, 1.5, -20.0).to(dtype)
    x[5] = (x[5].float() * 1e-6).to(dtype)
    x[6] = (x[6].float() * 200).clamp(-6e4, 6e4).to(dtype)
    x[7] = -x[7].abs() - 3
    x[8, ::2] = 0.0
    x[9] = -math.inf
    x[9, -1] = 3.0
    x[10, V // 2] = math.nan
    u[11], u[12], u[13], u[14] = 0.0, 1.0, 1 - 2.0 ** -24, 0.5
    u[1], u[2], u[9] = 0.0, 1.0, 1.0
    for kw in (dict(top_p=0.95), dict(top_p=0.6, min_p=0.01), dict(top_k=1000), dict(top_k=V // 2, temperature=0.7),
               dict(top_k=5000, top_p=0.9), dict(top_p=0.5, temperature=0.05)):
        _check(x, u, **kw)
        _check(x, u.flip(0), **kw)
    _check(x, u, top_k=torch.randint(-5, 3000, (rows,), generator=g), top_p=0.5 + torch.rand(rows, generator=g),
           min_p=0.01 * torch.rand(rows, generator=g), temperature=0.5 + torch.rand(rows, generator=g))
    # one row over many blocks, from end to end
    for v in torch.linspace(0, 1, 41).tolist():
        _check(x[14:15], torch.tensor([v]), top_p=0.9)
        _check(x[4:5], torch.tensor([v]), top_k=V // 3)


# every chain of launches: no filter, min-p alone, lists, bins (one filter, two, parts that are chosen), a value each
CHAINS = [(1, 9001, dict()), (3, 9001, dict(min_p=0.1)), (1, 30011, dict(top_k=40)), (300, 9001, dict(top_k=40, top_p=0.9)),
          (2, 30011, dict(top_p=0.9)), (300, 9001, dict(top_p=0.9)), (2, 30011, dict(top_k=900, top_p=0.9)),
          (100, 140011, dict(top_p=0.95, min_p=1e-4)), (40, 30011, "each"), (300, 9001, "each")]


def _chain(case, dtype, seed):
    rows, V, kw = case
    x, u, g = _rows(rows, V, dtype, seed=seed)
    if kw == "each":
        kw = dict(temperature=0.5 + torch.rand(rows, generator=g), top_k=torch.randint(-50, 400, (rows,), generator=g),
                  top_p=0.6 + 0.5 * torch.rand(rows, generator=g), min_p=0.01 * torch.rand(rows, generator=g))
    dev = gpu()
    return [x.to(dev), u.to(dev)], {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in kw.items()}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", CHAINS, ids=lambda c: f"{c[0]}x{c[1]}-{c[2] if c[2] == 'each' else '-'.join(c[2])}")
def test_repeats_graphs_and_used_workspaces(dtype, case):
    """The same numbers on every call, in a captured graph with new logits, and whatever the workspace held before."""
    (x, u), kw = _chain(case, dtype, 40)
    (x2, u2), kw2 = _chain(case, dtype, 41)
    first, other = hilda_sample(x, u, **kw), hilda_sample(x2, u2, **kw2)
    for fill in (0, 255, 127):
        junk = torch.full((64 << 20,), fill, dtype=torch.uint8, device=gpu())
        del junk  # the next workspace is cut from it
        again = hilda_sample(x, u, **kw)
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        hilda_sample(x, u, **kw)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = hilda_sample(x, u, **kw)
    held = [t.clone() for t in (x, u)], {k: v.clone() for k, v in kw.items() if isinstance(v, torch.Tensor)}
    for n in range(4):
        src, want = ((x2, u2), kw2), other
        if n % 2:
            src, want = held, first
        x.copy_(src[0][0])
        u.copy_(src[0][1])
        for k, v in kw.items():
            if isinstance(v, torch.Tensor):
                v.copy_(src[1][k])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]), f"replay {n}"


@pytest.mark.parametrize("kw", [dict(top_p=0.95), dict(top_k=2000, min_p=1e-3), "each"], ids=["p", "km", "each"])
def test_few_long_parts(kw):
    """As test_parts_of_a_row, with so many rows that two blocks share one: the token's part is told by the counts."""
    V, rows = 140011, 120
    x, _, g = _rows(24, V, torch.bfloat16, seed=50, lo=0.5, hi=5.0)
    x[0] = 0.0
    x[1, : V // 3] = -math.inf
    x[2, V // 5:] = -math.inf
    x[3, 100: V // 2] = torch.finfo(torch.bfloat16).min
    x[4] = torch.where(torch.rand(V, generator=g) < 0.5, 1.5, -20.0).to(torch.bfloat16)
    x[5] = (x[5].float() * 1e-6).to(torch.bfloat16)
    x[6] = (x[6].float() * 200).to(torch.bfloat16)
    x[7] = -x[7].abs() - 3
    x[8, ::2], x[8, 5::8] = 0.0, 2.0 ** -30
    x[9] = -math.inf
    x[9, -1] = 3.0
    x[10, V // 2] = math.nan
    x = x.repeat(rows // 24, 1)
    u = torch.rand(rows, generator=g)
    u[:24], u[24:48], u[48:72], u[72:96] = 0.0, 1.0, 1 - 2.0 ** -24, 0.5
    if kw == "each":
        kw = dict(top_k=torch.randint(-9000, 9000, (rows,), generator=g), top_p=0.5 + torch.rand(rows, generator=g),
                  min_p=0.01 * torch.rand(rows, generator=g), temperature=0.05 + torch.rand(rows, generator=g))
    _check(x, u, **kw)
