"""ops.group_norm_act's sums where they cancel or grow long: flat groups, groups far from zero, and channel sums of many terms of one sign,
against the formulas in float64."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _last(t):
    return t.contiguous(memory_format=torch.channels_last)


def _refs(x, g, w, b, dy, eps):
    """y and the gradients of (x, w, b) without an activation, two passes in float64"""
    n, c, h, wd = x.shape
    v, d = x.double().reshape(n, g, -1), dy.double()
    first = v[:, :, :1]
    mean = first + (v - first).mean(2, keepdim=True)  # (exactly the value of a flat group)
    cen = v - mean
    rstd = 1 / torch.sqrt((cen * cen).mean(2, keepdim=True) + eps)
    xhat = (cen * rstd).reshape(x.shape)
    gw = (d * w.double().view(1, c, 1, 1)).reshape(n, g, -1)
    xg = xhat.reshape(n, g, -1)
    dx = rstd * (gw - gw.mean(2, keepdim=True) - xg * (gw * xg).mean(2, keepdim=True))
    y = xhat * w.double().view(1, c, 1, 1) + b.double().view(1, c, 1, 1)
    return y, dx.reshape(x.shape), (d * xhat).sum((0, 2, 3)), d.sum((0, 2, 3)), rstd


# a sample in registers; in chunks, in vectors and in single elements; one group of many channels
SHAPES = [(3, 64, 15, 15, 8), (2, 24, 64, 63, 3), (2, 15, 40, 41, 5), (1, 300, 32, 33, 1), (1, 32, 128, 127, 2)]


def _case(shape, value, noise, seed):
    n, c, h, w, g = shape
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    x = _last(torch.full((n, c, h, w), value, device="cuda") + noise * rn(n, c, h, w))
    return x, (1 + 0.2 * rn(c)), 0.2 * rn(c), _last(rn(n, c, h, w))


def _check(shape, value, noise, eps=1e-5):
    from alphazero_amd import ops

    g = shape[4]
    x, w, b, dy = _case(shape, value, noise, 3)
    ts = [t.requires_grad_(True) for t in (x, w, b)]
    y = ops.group_norm_act(x, g, w, b, eps=eps, activation="none")
    dx, dw, db = torch.autograd.grad(y, ts, dy)
    ry, rdx, rdw, rdb, rstd = _refs(x.detach(), g, w.detach(), b.detach(), dy, eps)
    # fewer than 16 f32 operations, each off by 2^-24 of a term of at most 32 (forward), 64 rstd (dx; |dz w|, |m1| and |xhat m2| stay below 64)
    assert float((y.detach().double() - ry).abs().max()) <= 2.0 ** -15
    assert bool(((dx.double() - rdx).abs() <= 2.0 ** -14 * rstd.amax()).all()), (float((dx.double() - rdx).abs().max()), float(rstd.amax()))
    # the channel sums: 2^-16 of the sum of magnitudes (|xhat| <= 8)
    mag = dy.double().abs().sum((0, 2, 3))
    assert bool(((db.double() - rdb).abs() <= 2.0 ** -16 * mag).all()) and bool(((dw.double() - rdw).abs() <= 2.0 ** -13 * mag).all())


@pytest.mark.parametrize("value", [0.1, 1000.1, -77777.77, 333333.34, 3e30])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_a_flat_group_has_no_variance(shape, value):
    """every value alike: the variance is 0 and 1 / sqrt(eps) scales dx, whatever the value's square loses"""
    _check(shape, value, 0.0)


@pytest.mark.parametrize("ratio", [1e5, 1e6, 4e6])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_a_mean_of_many_deviations(shape, ratio):
    """values of `ratio` deviations beside zero, rounded to f32 as they come: the statistics are those of the rounded values"""
    _check(shape, ratio, 1.0)


def test_a_first_value_unlike_the_others():
    """a group's first value is far from all others, which are alike"""
    from alphazero_amd import ops

    for shape in SHAPES:
        n, c, h, w, g = shape
        x, wt, b, dy = _case(shape, 0.0, 1.0, 5)
        x[:, ::c // g, 0, 0] = 1e4
        x = _last(x)
        y = ops.group_norm_act(x, g, wt, b, activation="none")
        ry = _refs(x, g, wt, b, dy, 1e-5)[0]
        assert bool(((y.double() - ry).abs() <= 2.0 ** -20 * ry.abs() + 2.0 ** -15).all())


def test_channel_sums_of_many_terms_of_one_sign():
    """4,096 pixels of a sample one after the other (129 channels: each thread has one), every term of a channel's sums alike, so that
    roundings do not cancel.  The f32 runs hold 64 terms at most (64 * 2^-24 of their sum), everything after them is f64 but for three
    roundings to f32, and xhat carries four: 2^-18 + 7 * 2^-24 < 2^-17"""
    from alphazero_amd import ops

    n, c, h, w = 1024, 129, 64, 64
    off = torch.linspace(0.7, 1.3, c, device="cuda") * torch.where(torch.arange(c, device="cuda") % 2 == 0, 1.0, -1.0)
    x = off.expand(n, h, w, c).contiguous().permute(0, 3, 1, 2)
    dy = torch.full((n, h, w, c), 1 / 3, device="cuda").permute(0, 3, 1, 2)
    wt, b = torch.ones(c, device="cuda", requires_grad=True), torch.zeros(c, device="cuda", requires_grad=True)
    y = ops.group_norm_act(x, 1, wt, b, activation="none")
    dw, db = torch.autograd.grad(y, [wt, b], dy)
    each = float(dy[0, 0, 0, 0]) * n * h * w
    assert float((db.double() - each).abs().max()) <= 2.0 ** -17 * each, float((db.double() / each - 1).abs().max())
    v = off.double()
    want = each * (v - v.mean()) / torch.sqrt(((v - v.mean()) ** 2).mean() + 1e-5)
    assert bool(((dw.double() - want).abs() <= 2.0 ** -17 * want.abs()).all()), float((dw.double() / want - 1).abs().max())
