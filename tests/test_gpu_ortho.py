"""ops.orthogonalize against its definition in float64, and learner.Muon.

Tolerance: the same float64 iteration with its X, A and B disturbed at every step by random relative errors of the size that the kernel's
formats may make -- two f16 halves hold 22 bits (2^-22 of an entry), one f16 holds 2^-11, an f32 sum of K products loses about
2^-24 sqrt(K) of its terms' size -- says how far rounding can carry a result (early errors in directions of small singular values grow
3.4-fold a step).  Four times the larger of two such runs (Frobenius norm) is allowed, plus the result's own rounding; single entries may
be off by 16 times that norm's share of one entry."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

COEF = (3.4445, -4.7750, 2.0315)
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def plain(m, steps=5, coef=COEF, eps=1e-7, noise=0.0, gen=None):
    a, b, c = coef
    x = m.double()
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    x = x / (x.pow(2).sum().sqrt() + eps)
    jog = (lambda t: t * (1 + noise * torch.randn(t.shape, dtype=t.dtype, device=t.device, generator=gen))) if noise else (lambda t: t)
    x = jog(x)
    for _ in range(steps):
        s = jog(x @ x.t().contiguous())
        x = jog(a * x + jog(b * s + c * (s @ s)) @ x)
    return x.t().contiguous() if tall else x


def check(m, got, steps=5, coef=COEF, eps=1e-7):
    assert got.shape == m.shape and got.dtype == m.dtype and got.is_contiguous()
    ref = plain(m, steps, coef, eps)
    level = (2.0 ** -11 if m.dtype == torch.bfloat16 else 2.0 ** -22) + 2.0 ** -24 * math.sqrt(max(m.shape))
    gen = torch.Generator(device=m.device).manual_seed(1)
    drift = max(float((plain(m, steps, coef, eps, level, gen) - ref).norm()) for _ in range(2))
    err = (got.double() - ref)
    tol = 4 * drift + HALF[m.dtype] * float(ref.norm()) + 2.0 ** -24
    assert float(err.norm()) <= tol, (tuple(m.shape), m.dtype, float(err.norm()), tol, float(ref.norm()))
    one = 16 * tol / math.sqrt(m.numel()) + 2.0 ** -24
    assert bool((err.abs() <= HALF[m.dtype] * ref.abs() + one).all()), (tuple(m.shape), float(err.abs().max()), one)


def make(shape, dtype, seed, scale=1e-3, strong=4):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r, c = shape
    k = min(r, c, strong)
    return (scale * (torch.randn(r, c, device="cuda", generator=g) + torch.randn(r, k, device="cuda", generator=g) @ torch.randn(k, c, device="cuda", generator=g))).to(dtype)


SHAPES = [(1, 1), (1, 7), (7, 1), (2, 3000), (3000, 2), (63, 65), (65, 63), (64, 64), (64, 576), (576, 64), (64, 81), (128, 81), (64, 450), (225, 225),
          (128, 1152), (1152, 128), (64, 768), (768, 33), (64, 769), (32, 768), (33, 32), (20, 700), (31, 257), (300, 1000), (1000, 300), (129, 4097), (513, 511), (1025, 700)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_against_the_definition(shape, dtype):
    from alphazero_amd import ops

    m = make(shape, dtype, shape[0] * 31 + shape[1], 0.1)
    got = ops.orthogonalize(m)
    check(m, got)
    assert torch.equal(got, ops.orthogonalize(m))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_list_is_its_matrices(dtype):
    """a whole net's matrices (and more than one launch takes) give what each gives alone"""
    from alphazero_amd import ops

    ms = [make(s, dtype, i, 0.01) for i, s in enumerate(SHAPES[:14] * 5 + [(0, 5), (5, 0)] + [(64, 576)] * 10)]
    got = ops.orthogonalize(ms)
    assert isinstance(got, list) and len(got) == len(ms)
    small = [m for m in ms if min(m.shape) <= 64 and max(m.shape) <= 768]  # (alone, these take another kernel)
    for m, o in zip(ms, got):
        if min(m.shape) > 64 or max(m.shape) > 768:
            assert torch.equal(o, ops.orthogonalize(m))
    for m, o in zip(small, ops.orthogonalize(small)):
        if m.numel():
            assert torch.equal(o, ops.orthogonalize(m))
    for i in (0, 3, 5, 69):
        check(ms[i], got[i])
    check(ms[-1], got[-1])
    assert ops.orthogonalize([]) == []


def test_batches_views_and_shapes():
    from alphazero_amd import ops

    b = torch.stack([make((40, 90), torch.float32, i) for i in range(5)])
    got = ops.orthogonalize(b)
    assert got.shape == b.shape
    for i in range(5):
        assert torch.equal(got[i], ops.orthogonalize(b[i]))
    t = b[0].t()  # a transposed view
    assert torch.equal(ops.orthogonalize(t), ops.orthogonalize(t.contiguous()))
    assert torch.equal(ops.orthogonalize(b[1][::2, 3:50]), ops.orthogonalize(b[1][::2, 3:50].contiguous()))
    assert ops.orthogonalize(b[:0]).shape == (0, 40, 90) and ops.orthogonalize(b[0, :0]).shape == (0, 90)


def test_sizes_of_values():
    from alphazero_amd import ops

    for scale in (1e-30, 1e-6, 1.0, 1e30):
        m = make((64, 100), torch.float32, 3, scale)
        check(m, ops.orthogonalize(m, eps=0.0), eps=0.0)
        check(m, ops.orthogonalize(m))  # (eps counts beside a norm of 1e-28: X0 is small, and so is the result)
    z = torch.zeros(64, 100, device="cuda")
    assert float(ops.orthogonalize(z).abs().max()) == 0 and float(ops.orthogonalize(z, eps=0.0).abs().max()) == 0
    for bad in (float("nan"), float("inf")):
        m = make((64, 100), torch.float32, 4)
        m[3, 5] = bad
        n = make((64, 100), torch.float32, 5)
        got = ops.orthogonalize([m, n])
        assert bool(torch.isnan(got[0]).all()) and torch.equal(got[1], ops.orthogonalize(n))
    one = make((96, 200), torch.float32, 6, 1.0, 1) * 0 + torch.randn(96, 1, device="cuda") @ torch.randn(1, 200, device="cuda")  # rank one
    check(one, ops.orthogonalize(one))


def test_steps_and_coefficients():
    from alphazero_amd import ops

    m = make((80, 130), torch.float32, 8)
    for steps in (1, 2, 3, 8):
        check(m, ops.orthogonalize(m, steps=steps), steps)
    cubic = (1.5, -0.5, 0.0)  # converges to the nearest orthogonal matrix
    got = ops.orthogonalize(m, steps=30, coefficients=cubic)
    check(m, got, 30, cubic)
    eye = got.double() @ got.double().t().contiguous()
    assert float((eye - torch.eye(80, device="cuda")).abs().max()) < 1e-5
    u, s, v = torch.linalg.svd(m.double().cpu(), full_matrices=False)
    assert float((got.double().cpu() - u @ v).abs().max()) < 1e-4


def test_another_stream_and_a_graph():
    from alphazero_amd import ops

    ms = [make((64, 576), torch.float32, 1), make((225, 225), torch.float32, 2)]
    want = ops.orthogonalize(ms)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.orthogonalize(ms)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = ops.orthogonalize(ms)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    for seed in (11, 12, 13):
        for m in ms:
            m.copy_(make(tuple(m.shape), torch.float32, seed))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, ops.orthogonalize(ms)))


def test_muon_steps():
    """three steps against the update rules in float64.  Tolerance per parameter: lr times what the update itself may be off"""
    from alphazero_amd.learner import Muon

    g = torch.Generator(device="cuda").manual_seed(4)
    shapes = [(64, 9, 3, 3), (30, 50), (64,), (120, 7), ()]
    ps = [torch.nn.Parameter(torch.randn(s, device="cuda", generator=g)) for s in shapes]
    ps[0].data = ps[0].data.contiguous(memory_format=torch.channels_last)
    frozen = torch.nn.Parameter(torch.ones(3, 3, device="cuda"))  # no gradient: stays
    opt = Muon(ps + [frozen], lr=0.02, weight_decay=0.1, adam_lr=0.01)
    ref = [p.detach().double().clone() for p in ps]
    buf = [torch.zeros_like(r) for r in ref]
    avg, sq = [torch.zeros_like(r) for r in ref], [torch.zeros_like(r) for r in ref]
    for t in range(1, 4):
        for i, p in enumerate(ps):
            p.grad = torch.randn(p.shape, device="cuda", generator=g) * 0.1
            d = p.grad.double()
            if d.dim() >= 2:
                buf[i] = buf[i] * 0.95 + d * 0.05
                u = (d * 0.05 + buf[i] * 0.95).reshape(d.shape[0], -1)
                o = plain(u).reshape(d.shape) * max(1.0, u.shape[0] / u.shape[1]) ** 0.5
                ref[i] = ref[i] * (1 - 0.02 * 0.1) - 0.02 * o
            else:
                avg[i] = avg[i] * 0.9 + d * 0.1
                sq[i] = sq[i] * 0.999 + d * d * 0.001
                ref[i] = ref[i] * (1 - 0.01 * 0.1) - 0.01 * (avg[i] / (1 - 0.9 ** t)) / ((sq[i] / (1 - 0.999 ** t)).sqrt() + 1e-8)
        opt.step()
    for p, r in zip(ps, ref):  # three updates of 0.02 whose entries are off by 1e-4 at most, and f32 parameters of size 4
        assert float((p.detach().double() - r).abs().max()) < 3 * (0.02 * 1e-4 + 8 * 2.0 ** -24)
    assert bool((frozen == 1).all())
    state = opt.state_dict()
    opt2 = Muon(ps + [frozen], lr=0.5)
    opt2.load_state_dict(state)
    assert opt2.param_groups[0]["lr"] == 0.02 and torch.equal(opt2.state[ps[0]]["momentum"], opt.state[ps[0]]["momentum"])


def test_workspace_beyond_32_bit_offsets():
    """the second matrix's buffers start past 4 GiB of the workspace; a matrix's result is the same there, bit for bit"""
    from alphazero_amd import ops

    m = torch.randn(4096, 65536, device="cuda", generator=torch.Generator(device="cuda").manual_seed(71))
    one = ops.orthogonalize(m, steps=2)
    two = ops.orthogonalize([m, m], steps=2)
    assert torch.equal(two[0], one) and torch.equal(two[1], one)
    check(m, one, steps=2)


@pytest.mark.parametrize("shape,dtype", [((2900, 2950), torch.float32), ((2990, 2890), torch.float16), ((4090, 4150), torch.bfloat16), ((2000, 2500), torch.bfloat16)],
                         ids=lambda v: str(v))
def test_large_matrices_of_which_a_few_tiles_are_cut(shape, dtype):
    """23 x 23 tiles of 128 leave 20 after a whole turn of 256, 32 x 32 leave 16 after one of 512"""
    from alphazero_amd import ops

    m = make(shape, dtype, 81)
    one = ops.orthogonalize(m)
    check(m, one)
    other = make((300, 200), dtype, 82)
    two = ops.orthogonalize([other, m, m])
    assert torch.equal(two[1], one) and torch.equal(two[2], one)
    check(other, two[0])
