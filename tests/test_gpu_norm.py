"""ops.group_norm_act, forward and backward, against the formulas in float64 (plain torch on planes-first copies), and the gradient
against central differences.

Tolerances, for values of size about 1 (weights, standard deviations and gradients here are): an output is rounded once, by eps / 2 of
its value (bf16 2^-8 / f16 2^-11 / f32 2^-24 at most); the f32 arithmetic before it is fewer than 16 operations, each off by at most
2^-24 of a term no larger than |xhat w| + |b| + |r| <= 32 (forward) or rstd (|dz w| + |m1| + |xhat m2|) <= 128 (backward; dx is the sum of
three such terms): 16 * 32 * 2^-24 = 2^-15 and 16 * 128 * 2^-24 = 2^-13.  The channel sums are of at most 2^18 terms of size <= 32 in f32
partial sums of a workgroup's share (<= 2^13 terms, pairwise over at least 2 threads): relative to the sum of magnitudes 2^13 * 2^-24 =
2^-11 at the very most; 2^-16 of it is asked here (errors of both signs: square root of the count), plus the rounding to the type."""
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def plain(x, g, w, b, r, eps, act):
    n, c, h, wd = x.shape
    v = x.reshape(n, g, -1)
    mean = v.mean(2, keepdim=True)
    var = ((v - mean) ** 2).mean(2, keepdim=True)
    z = ((v - mean) / torch.sqrt(var + eps)).reshape(n, c, h, wd)
    if w is not None:
        z = z * w.view(1, c, 1, 1)
    if b is not None:
        z = z + b.view(1, c, 1, 1)
    if r is not None:
        z = z + r
    return z.clamp(min=0) if act == "relu" else z * torch.sigmoid(z) if act == "silu" else z


def make(n, c, h, w, dtype, pdtype, seed, affine=True, residual=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g)
    last = lambda t: t.to(dtype).contiguous(memory_format=torch.channels_last)
    x = last(rn(n, c, h, w) * (0.5 + torch.rand(c, 1, 1, device="cuda", generator=g)) + 0.5 * rn(c, 1, 1))
    wt = (1 + 0.2 * rn(c)).to(pdtype) if affine else None
    b = (0.2 * rn(c)).to(pdtype) if affine else None
    r = last(rn(n, c, h, w)) if residual else None
    return x, wt, b, r, last(rn(n, c, h, w))


def check(x, w, b, r, dy, g, act, eps=1e-5):
    from alphazero_amd import ops

    ts = [t for t in (x, w, b, r) if t is not None]
    for t in ts:
        t.requires_grad_(True)
    y = ops.group_norm_act(x, g, w, b, eps=eps, activation=act, residual=r)
    assert y.dtype == x.dtype and y.shape == x.shape and (y.numel() == 0 or y.is_contiguous(memory_format=torch.channels_last))
    with torch.no_grad():
        assert torch.equal(y, ops.group_norm_act(x, g, w, b, eps=eps, activation=act, residual=r))
    grads = torch.autograd.grad(y, ts, dy)
    ds = {id(t): t.detach().double().requires_grad_(True) for t in ts}
    at = lambda t: None if t is None else ds[id(t)]
    ref = plain(at(x), g, at(w), at(b), at(r), eps, act)
    rgrads = torch.autograd.grad(ref, [ds[id(t)] for t in ts], dy.double())
    half = HALF[x.dtype]
    assert bool(((y.double() - ref).abs() <= half * ref.abs() + 2.0 ** -15).all()), float((y.double() - ref).abs().max())
    for t, got, want in zip(ts, grads, rgrads):
        assert got.shape == t.shape and got.dtype == t.dtype
        if t is w or t is b:
            with torch.no_grad():  # the sum of magnitudes the channel sums are taken over
                mag = dy.double().abs() * (1.1 if act == "silu" else 1.0)
                if t is w:
                    one = torch.ones_like(w, dtype=torch.float64)
                    mag = mag * plain(x.double(), g, one, None, None, eps, "none").abs()
                mag = mag.sum((0, 2, 3))
            tol = 2.0 ** -16 * mag + HALF[t.dtype] * want.abs() + 2.0 ** -20
        else:
            tol = half * want.abs() + 2.0 ** -13
        assert got.numel() == 0 or bool(((got.double() - want).abs() <= tol).all()), (got.shape, float((got.double() - want).abs().max()))
    return y, grads


SHAPES = [(64, 64, 9, 9, 8), (5, 64, 15, 15, 8), (3, 128, 15, 15, 8), (2, 64, 3, 3, 16), (7, 64, 4, 4, 32), (1, 1, 9, 9, 1), (3, 2, 15, 15, 1),
          (2, 12, 7, 5, 4), (2, 15, 6, 6, 5), (2, 7, 5, 3, 7), (1, 320, 33, 31, 32), (2, 24, 64, 63, 3), (1, 1000, 9, 10, 8), (300, 8, 3, 4, 2),
          (1, 513, 11, 11, 27), (2, 2048, 5, 5, 16), (1, 64, 1, 40, 8), (1, 16, 128, 127, 1)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_against_the_formulas(shape, dtype):
    n, c, h, w, g = shape
    for i, (act, residual, affine) in enumerate([("relu", False, True), ("relu", True, True), ("silu", False, True), ("none", True, True), ("silu", True, False), ("none", False, False)]):
        x, wt, b, r, dy = make(n, c, h, w, dtype, dtype if i % 2 else torch.float32, 10 * n + c + i, affine, residual)
        check(x, wt, b, r, dy, g, act)


@pytest.mark.parametrize("shape", [(1100, 128, 15, 15, 8), (4000, 64, 15, 15, 8), (2, 512, 128, 127, 32), (70000, 4, 2, 2, 2)], ids=lambda s: "x".join(map(str, s)))
def test_large(shape):
    n, c, h, w, g = shape
    for dtype, act, residual in ((torch.float32, "relu", True), (torch.bfloat16, "silu", False)):
        x, wt, b, r, dy = make(n, c, h, w, dtype, torch.float32, 3, True, residual)
        check(x, wt, b, r, dy, g, act)


def test_weight_or_bias_alone_and_gradients_not_asked_for():
    from alphazero_amd import ops

    x, w, b, r, dy = make(3, 32, 5, 5, torch.bfloat16, torch.bfloat16, 1, True, True)
    for ww, bb in ((w, None), (None, b)):
        check(x.detach(), ww.detach() if ww is not None else None, bb.detach() if bb is not None else None, None, dy, 4, "relu")
    ref = {}
    full = [t.detach().requires_grad_(True) for t in (x, w, b, r)]
    y = ops.group_norm_act(full[0], 4, full[1], full[2], residual=full[3])
    for t, gr in zip("xwbr", torch.autograd.grad(y, full, dy)):
        ref[t] = gr
    for only in "xwbr":
        ts = {k: t.detach() for k, t in zip("xwbr", (x, w, b, r))}
        ts[only] = ts[only].requires_grad_(True)
        y = ops.group_norm_act(ts["x"], 4, ts["w"], ts["b"], residual=ts["r"])
        assert torch.equal(torch.autograd.grad(y, ts[only], dy)[0], ref[only])


def test_gradient_against_differences():
    """(f(t + h e) - f(t - h e)) / 2h of a weighted sum of the outputs; h = 2^-6: the silu's third derivative leaves h^2, and f's f32
    rounding 2^-22 * sqrt(1500) / h = 6e-4"""
    from alphazero_amd import ops

    x, w, b, r, dy = make(2, 8, 9, 9, torch.float32, torch.float32, 5, True, True)
    ts = [t.clone().requires_grad_(True) for t in (x, w, b, r)]

    def f(ts):
        return (ops.group_norm_act(ts[0], 2, ts[1], ts[2], activation="silu", residual=ts[3]).double() * dy).sum()

    grads = torch.autograd.grad(f(ts), ts)
    g = torch.Generator(device="cuda").manual_seed(8)
    h = 2.0 ** -6
    for i, t in enumerate(ts):
        for _ in range(4):
            e = torch.randn(t.shape, device="cuda", generator=g).to(t.dtype)
            e = e / e.norm()
            with torch.no_grad():
                up, down = list(ts), list(ts)
                up[i], down[i] = t + h * e, t - h * e
                diff = float((f(up) - f(down)) / (2 * h))
            want = float((grads[i].double() * e).sum())
            assert abs(diff - want) <= 5e-3 * max(1.0, abs(want)), (i, diff, want)


def test_relu_next_to_zero_takes_the_sign_of_the_exact_value():
    """residual = -(the normalised value), rounded to f32: z is a rounding error, and its sign decides the gradient"""
    from alphazero_amd import ops

    x, w, b, _, dy = make(2, 64, 15, 15, torch.float32, torch.float32, 6)
    exact = plain(x.double(), 8, w.double(), b.double(), None, 1e-5, "none")
    r = (-exact).float().contiguous(memory_format=torch.channels_last).requires_grad_(True)
    y = ops.group_norm_act(x, 8, w, b, residual=r)
    dr, = torch.autograd.grad(y, r, dy)
    z = exact + r.detach().double()
    sure = z.abs() > 1e-13  # (the f64 evaluations agree to this)
    assert bool((torch.where(z > 0, dy, torch.zeros_like(dy)) == dr)[sure].all()) and float(sure.float().mean()) > 0.99


def test_offset_far_from_zero():
    """mean 1000, deviation 1: f32 inputs hold 2^-14 of it; the statistics must not lose more"""
    from alphazero_amd import ops

    x, w, b, r, dy = make(2, 32, 15, 15, torch.float32, torch.float32, 7)
    x = (x + 1000.0).contiguous(memory_format=torch.channels_last)
    check(x, w, b, r, dy, 4, "silu")
    flat = torch.full((1, 8, 4, 4), 3.25, device="cuda").contiguous(memory_format=torch.channels_last)  # no variance at all
    assert float(ops.group_norm_act(flat, 2, activation="none").abs().max()) == 0.0


def test_infinities_and_nan_stay_in_their_group():
    from alphazero_amd import ops

    for bad in (float("inf"), float("-inf"), float("nan")):
        x, w, b, _, _ = make(2, 16, 5, 5, torch.float32, torch.float32, 9)
        clean = ops.group_norm_act(x, 4, w, b, activation="none")
        x[1, 5, 2, 2] = bad
        y = ops.group_norm_act(x, 4, w, b, activation="none")
        assert bool(torch.isnan(y[1, 4:8]).all())
        keep = torch.ones_like(y, dtype=torch.bool)
        keep[1, 4:8] = False
        assert torch.equal(y[keep], clean[keep])
        assert bool(torch.isnan(ops.group_norm_act(x, 4, w, b)[1, 4:8]).all())  # relu passes NaN on


def test_layouts():
    """planes-first, sliced, expanded and odd-offset inputs give what their dense copy gives"""
    from alphazero_amd import ops

    x, w, b, r, dy = make(4, 64, 9, 9, torch.bfloat16, torch.float32, 11, True, True)
    want = ops.group_norm_act(x, 8, w, b, residual=r)
    assert torch.equal(ops.group_norm_act(x.contiguous(), 8, w, b, residual=r.contiguous()), want)
    wide = torch.cat([x, x], 1).contiguous(memory_format=torch.channels_last)
    assert torch.equal(ops.group_norm_act(wide[:, 64:], 8, w, b, residual=r), want)
    flat = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")
    odd = flat[1:].view(4, 9, 9, 64).permute(0, 3, 1, 2)  # dense, at an odd address
    odd.copy_(x)
    assert torch.equal(ops.group_norm_act(odd, 8, w, b, residual=r), want)
    one = r[:1].expand(4, 64, 9, 9).detach().requires_grad_(True)
    y = ops.group_norm_act(x, 8, w, b, residual=one)
    assert torch.equal(y, ops.group_norm_act(x, 8, w, b, residual=one.detach().contiguous()))
    leaf = r[:1].detach().clone().requires_grad_(True)  # a broadcast input's gradient is summed
    y = ops.group_norm_act(x, 8, w, b, residual=leaf.expand(4, 64, 9, 9))
    part, = torch.autograd.grad(y, leaf, dy)
    assert part.shape == leaf.shape
    wn = torch.stack([w, w], 1)[:, 0]  # strided parameters
    assert torch.equal(ops.group_norm_act(x, 8, wn, b, residual=r), want)
    ya = ops.group_norm_act(x.detach().requires_grad_(True), 8, w, b, residual=r)
    yb = ops.group_norm_act(x, 8, w.requires_grad_(True), b, residual=r)
    ga, = torch.autograd.grad(yb, w, dy.contiguous())  # a gradient that arrives planes first, or expanded
    assert torch.equal(ga, torch.autograd.grad(ops.group_norm_act(x, 8, w, b, residual=r), w, dy)[0])
    ya.sum().backward()


def test_nothing_to_do():
    from alphazero_amd import ops

    for shape in ((0, 8, 3, 3), (2, 8, 0, 3)):
        x = torch.empty(shape, device="cuda", requires_grad=True)
        w = torch.ones(8, device="cuda", requires_grad=True)
        b = torch.ones(8, device="cuda", requires_grad=True)
        y = ops.group_norm_act(x, 2, w, b)
        assert y.shape == x.shape
        gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.empty(shape, device="cuda"))
        assert gx.shape == x.shape and float(gw.abs().sum()) == 0 and float(gb.abs().sum()) == 0


def test_another_stream_and_a_graph():
    from alphazero_amd import ops

    x, w, b, r, dy = make(6, 64, 15, 15, torch.float32, torch.float32, 13, True, True)
    ts = [t.requires_grad_(True) for t in (x, w, b, r)]

    def step():
        y = ops.group_norm_act(ts[0], 8, ts[1], ts[2], residual=ts[3])
        return [y.detach(), *torch.autograd.grad(y, ts, dy)]

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = step()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    for seed in (1, 2, 3):
        new = make(6, 64, 15, 15, torch.float32, torch.float32, seed, True, True)
        with torch.no_grad():
            for t, v in zip((*ts, dy), new):
                t.copy_(v)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, step()))


def test_in_a_training_step():
    """the group-norm net through the learner's step: its gradients against the same net from plain operations in f64.
    Tolerance: MIOpen's f32 convolutions, six layers deep; 2^-10 of a gradient's largest entry"""
    from alphazero_amd.learner import calculate_loss
    from alphazero_amd.nets import GomokuNet

    torch.manual_seed(0)
    net = GomokuNet(9, 16, 2, norm="group", groups=4).cuda()
    for p in net.parameters():
        if p.dim() == 1:
            p.data.add_(0.1 * torch.randn_like(p))
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randint(-1, 2, (8, 9, 9, 9), device="cuda", generator=g).float()
    pi = torch.softmax(torch.randn(8, 81, device="cuda", generator=g), 1)
    z = torch.randn(8, 1, device="cuda", generator=g).sign()
    loss, _, _ = calculate_loss(net, x, pi, z)
    loss.backward()
    ref = _PlainNet(net)
    rloss, _, _ = calculate_loss(ref, x.double().cpu(), pi.double().cpu(), z.double().cpu())
    rloss.backward()
    assert abs(float(loss.detach()) - float(rloss.detach())) < 1e-4
    for name, p in net.named_parameters():
        want = ref.p[name].grad
        assert float((p.grad.cpu().double() - want).abs().max()) <= 2.0 ** -10 * float(want.abs().max()) + 1e-7, name


class _PlainNet:
    def __init__(self, net):
        self.p = {k: v.detach().cpu().double().requires_grad_(True) for k, v in net.named_parameters()}
        self.net = net

    def __call__(self, x):
        p, F = self.p, torch.nn.functional

        def conv(name, t):
            w = p[name + ".weight"]
            return F.conv2d(t, w, padding=w.shape[2] // 2)

        def norm(name, t, g, r=None):
            return plain(t, g, p[name + ".weight"], p[name + ".bias"], r, 1e-5, "relu")

        h = norm("_shared_layers.1", conv("_shared_layers.0", x), 4)
        for k in (2, 3):
            s = f"_shared_layers.{k}."
            h = norm(s + "_gn2", conv(s + "_conv2", norm(s + "_gn1", conv(s + "_conv1", h), 4)), 4, h)
        lin = lambda n, t: F.linear(t, p[n + ".weight"], p[n + ".bias"])
        a = lin("_policy_head.3", norm("_policy_head.1", conv("_policy_head.0", h), 1).flatten(1))
        v = norm("_value_head.1", conv("_value_head.0", h), 1).flatten(1)
        return a, torch.tanh(lin("_value_head.5", torch.relu(lin("_value_head.3", v))))


def test_self_play_on_a_group_norm_net():
    """the net plays through SelfPlayRunner's own-forward path, and the fused towers refuse it"""
    from alphazero_amd import Engine, EngineError
    from alphazero_amd.arena import SelfPlayRunner
    from alphazero_amd.fused import evaluator_available
    from alphazero_amd.nets import GomokuNet

    torch.manual_seed(1)
    net = GomokuNet(9, 64, 2, norm="group").cuda().eval()
    eng = Engine(2, 6, 12, board_size=9, device="cuda:0")
    assert not evaluator_available(2, net, torch.float32)
    with pytest.raises(EngineError):
        SelfPlayRunner(eng, net, 12, fused=True)
    run = SelfPlayRunner(eng, net, 12, seed=3)
    acts, _ = run.move_round(torch.ones(6, device="cuda"))
    eng.check()
    assert bool((acts >= 0).all()) and bool((acts < 81).all())
    eng.close()


@pytest.mark.parametrize("shape", [(1900000, 128, 3, 3, 8), (9, 64, 2048, 2048, 8)], ids=lambda s: "x".join(map(str, s)))
def test_more_than_2_31_elements(shape):
    """the last samples, whose offsets pass 32 bits, forward and backward; the parameters' gradients in f64 sums over shares of the batch"""
    from alphazero_amd import ops

    n, c, h, w, g = shape
    base = torch.randn(4096 * 9 * 128 + 1, device="cuda", generator=torch.Generator(device="cuda").manual_seed(61)).bfloat16()
    total = n * c * h * w
    x, dy = (torch.empty(total, dtype=torch.bfloat16, device="cuda").view(n, h, w, c).permute(0, 3, 1, 2) for _ in range(2))
    for t, shift in ((x, 0), (dy, 1000)):  # (the numbers repeat, out of step with the samples)
        flat, m = t.permute(0, 2, 3, 1).reshape(-1), base.numel()
        reps = total // m
        flat[:reps * m].view(reps, m).copy_(base.roll(shift).expand(reps, m))
        flat[reps * m:] = base[:total - reps * m]
    wt, b = torch.linspace(0.5, 1.5, c, device="cuda").requires_grad_(True), torch.linspace(-0.3, 0.3, c, device="cuda").requires_grad_(True)
    x.requires_grad_(True)
    y = ops.group_norm_act(x, g, wt, b, activation="relu")
    dx, dw, db = torch.autograd.grad(y, [x, wt, b], dy)
    k = max(1, min(n, (1 << 28) // (c * h * w)))
    sw, sb, mw, mb = (torch.zeros(c, dtype=torch.float64, device="cuda") for _ in range(4))
    for lo in range(0, n, k):
        ts = [t.detach()[lo:lo + k].double() if t.dim() == 4 else t.detach().double() for t in (x, wt, b)]
        for t in ts:
            t.requires_grad_(True)
        d = dy[lo:lo + k].double()
        ref = plain(ts[0], g, ts[1], ts[2], None, 1e-5, "relu")
        rdx, rdw, rdb = torch.autograd.grad(ref, ts, d)
        sw += rdw
        sb += rdb
        with torch.no_grad():
            mw += (d.abs() * plain(ts[0], g, torch.ones_like(ts[1]), None, None, 1e-5, "none").abs()).sum((0, 2, 3))
            mb += d.abs().sum((0, 2, 3))
            assert bool(((y[lo:lo + k].double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -15).all())
            assert bool(((dx[lo:lo + k].double() - rdx).abs() <= 2.0 ** -8 * rdx.abs() + 2.0 ** -13).all())
        del ts, d, ref, rdx
    assert bool(((dw.double() - sw).abs() <= 2.0 ** -16 * mw).all()) and bool(((db.double() - sb).abs() <= 2.0 ** -16 * mb).all())
