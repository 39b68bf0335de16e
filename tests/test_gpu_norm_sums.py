"""ops.group_norm_act's sums where they cancel: flat groups and groups far from zero, against the formulas in float64."""
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
