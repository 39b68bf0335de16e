"""ops.sample_actions against a plain statement of its definition in float64 (numpy, sorted rows).

Indices have to be equal: the kernel's masses are integers in units of 2^-44 of the largest weight, so a border between two
neighbours moves by at most n 2^-45 of it, and a uniform number falls into that gap with a probability below 1e-6 per row of the
lengths used here.  Log-probabilities are compared to 2^-23 relative plus 2^-23: one rounding to f32 (2^-24 relative) and the gap
between the kernel's total and the sum here (1e-9 at most)."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def plain(scores, u, t, k, p, mp, legal=None):
    """scores float64 (n,), the other arguments numbers -> (index, log-probability)"""
    s = np.where(np.isnan(scores), -np.inf, scores)
    if legal is not None:
        s = np.where(legal, s, -np.inf)
    ids = np.flatnonzero(s > -np.inf)
    if ids.size == 0:
        return -1, -np.inf
    s = s[ids]
    if t <= 0:
        return int(ids[np.argmax(s)]), 0.0
    d = np.where(s == np.inf, 0.0, -np.inf) if s.max() == np.inf else (s - s.max()) / t
    w = np.exp(d)
    order = np.argsort(-s, kind="stable")
    if k > 0:
        order = order[:k]
    if p < 1:
        mass = np.cumsum(w[order])
        before = np.concatenate([[0.0], mass[:-1]])
        keep = before < p * mass[-1]
        keep[0] = True
        order = order[keep]
    if mp > 0:
        order = order[w[order] >= mp]
    kept = np.sort(order)
    mass = np.cumsum(w[kept])
    j = min(int(np.searchsorted(mass, u * mass[-1], side="right")), kept.size - 1)
    return int(ids[kept[j]]), float(d[kept[j]] - math.log(mass[-1]))


def check(scores, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, legal=None):
    from alphazero_amd import ops

    got, logp = ops.sample_actions(scores, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p, legal=legal, return_logprobs=True)
    again = ops.sample_actions(scores, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p, legal=legal)
    assert torch.equal(got, again)
    s, uh = scores.float().cpu().numpy().astype(np.float64), u.cpu().numpy().astype(np.float64)
    lg = legal.cpu().numpy() if legal is not None else None

    def row(v, r):
        return float(v[r]) if isinstance(v, torch.Tensor) else v

    got, logp = got.cpu().numpy(), logp.cpu().numpy().astype(np.float64)
    for r in range(s.shape[0]):
        a, lp = plain(s[r], uh[r], row(temperature, r), int(row(top_k, r)), row(top_p, r), row(min_p, r), None if lg is None else lg[r])
        assert got[r] == a, (r, got[r], a)
        assert lp == logp[r] if lp == -np.inf else abs(lp - logp[r]) <= 2.0 ** -23 * (1 + abs(lp)), (r, lp, logp[r])
    return got


def rand(rows, n, dtype, seed, spread=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(rows, n, device="cuda", generator=g) * spread).to(dtype), torch.rand(rows, device="cuda", generator=g)


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 5, 1.0, 0.0), (1.3, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.05), (0.5, 40, 0.8, 0.01), (0.0, 0, 0.5, 0.0),
            (1.0, 1, 1.0, 0.0), (1.0, 0, 0.0, 0.0), (1e-3, 0, 0.99, 0.0), (100.0, 7, 0.5, 1.0)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 2, 9, 63, 64, 65, 225, 255, 256, 257, 1000, 1024, 1025, 2049, 4097, 33000])
def test_against_the_definition(n, dtype):
    for i, (t, k, p, mp) in enumerate(SETTINGS):
        s, u = rand(7 if n < 5000 else 3, n, dtype, 100 * n + i)
        check(s, u, t, k, p, mp)


@pytest.mark.parametrize("n,rows", [(131072, 1), (131071, 2), (262144, 1), (524288, 1), (70001, 3)])
def test_long_rows(n, rows):
    for i, (t, k, p, mp) in enumerate([(0.8, 50, 0.95, 0.0), (1.0, 0, 0.9, 0.0), (1.0, 3000, 1.0, 0.0), (1.0, 0, 1.0, 0.0)]):
        for dtype in (torch.bfloat16, torch.float32):
            s, u = rand(rows, n, dtype, n + i, 3.0)
            check(s, u, t, k, p, mp)


@pytest.mark.parametrize("n", [10, 225, 700, 3000, 70000])
def test_equal_scores_are_ordered_by_index(n):
    for i, (t, k, p, mp) in enumerate([(1.0, 4, 1.0, 0.0), (1.0, 0, 0.5, 0.0), (1.0, n // 2, 0.3, 0.0), (0.0, 0, 1.0, 0.0), (1.0, n - 1, 1.0, 0.0), (1.0, 0, 0.75, 0.3)]):
        g = torch.Generator(device="cuda").manual_seed(n + i)
        u = torch.rand(6, device="cuda", generator=g)
        check(torch.zeros(6, n, device="cuda"), u, t, k, p, mp)  # one value
        check(torch.randint(0, 3, (6, n), device="cuda", generator=g).float(), u, t, k, p, mp)  # three values
        s = torch.randint(0, 2, (6, n), device="cuda", generator=g).float()
        check(torch.where(s > 0, 0.0, -0.0), u, t, k, p, mp)  # both zeros are one score


@pytest.mark.parametrize("n", [5, 225, 5000])
def test_rows_that_hold_nothing_infinities_and_nan(n):
    s, u = rand(16, n, torch.float32, 5)
    s[0] = -math.inf
    s[1] = math.nan
    s[2, 1:] = -math.inf  # one score left
    s[3, ::2] = math.nan
    s[4, 1] = math.inf
    s[5, 1] = s[5, n - 1] = math.inf  # two share the mass
    s[6] = torch.finfo(torch.float32).min
    s[7, :3] = torch.finfo(torch.float32).min
    s[8] = torch.finfo(torch.float32).max
    s[9, 0] = torch.finfo(torch.float32).max
    s[9, 1] = torch.finfo(torch.float32).min
    s[10] = math.inf
    s[11, 2:] = -1e30
    s[12] = 1e-45
    legal = torch.rand(16, n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) < 0.5
    legal[13] = False
    legal[14] = False
    legal[14, n - 1] = True
    legal[5] = True
    s[15] = torch.where(legal[15], s[15], math.nan)  # NaN under the mask
    for t, k, p, mp in SETTINGS:
        check(s, u, t, k, p, mp)
        got = check(s, u, t, k, p, mp, legal)
        assert got[13] == -1 and got[14] == n - 1
    assert check(s, u)[0] == -1 and check(s, u)[1] == -1


def test_uniform_numbers_at_their_ends():
    s, _ = rand(8, 300, torch.float32, 9)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 2.0 ** -149, 0.5, 1.0, 2.0, -1.0, math.nan], device="cuda")
    from alphazero_amd import ops

    got = ops.sample_actions(s, u, top_k=20)
    # outside [0, 1): below counts as 0, above as the last kept index
    want = torch.tensor([0.0, 1.0 - 2.0 ** -24, 2.0 ** -149, 0.5, 1.0 - 2.0 ** -24, 1.0 - 2.0 ** -24, 0.0, 0.0], device="cuda")
    assert torch.equal(got, ops.sample_actions(s, want, top_k=20))
    check(s, want, top_k=20)


@pytest.mark.parametrize("n", [225, 3001])
def test_settings_per_row(n):
    rows = 12
    s, u = rand(rows, n, torch.bfloat16, 21)
    t = torch.tensor([1.0, 0.5, 0.0, 2.0, -1.0, 0.1, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0], device="cuda")
    k = torch.tensor([0, 1, 5, 40, -3, n, n + 7, 2, 0, 0, 9, 0], dtype=torch.int32, device="cuda")
    p = torch.tensor([1.0, 0.9, 0.5, 0.3, 1.5, 0.8, 0.7, 0.0, 0.01, 0.999, 1.0, 0.6], device="cuda")
    mp = torch.tensor([0.0, 0.1, 0.2, 0.0, 0.3, 0.0, 1.0, 0.5, -1.0, 0.01, 0.02, 0.9], device="cuda")
    check(s, u, t, k, p, mp)
    check(s, u, t, 7, 0.9, 0.0)
    check(s, u, 1.0, k, 1.0, mp)


def test_strides_and_alignment():
    base, u = rand(9, 1000, torch.bfloat16, 31)
    legal = torch.rand(9, 1000, device="cuda") < 0.6
    for a, b in ((0, 1000), (1, 1000), (3, 500), (7, 8), (5, 300)):
        check(base[:, a:b], u, top_k=6, legal=legal[:, a:b])
        check(base[1::2, a:b], u[:4].contiguous(), top_p=0.9)
    one = base[:1].expand(9, 1000)  # one row for all draws
    check(one, u, 0.9, 0, 0.9, 0.0)
    check(base[:, 5:6], u)


def test_a_batch_is_its_rows():
    """every row of a big batch draws what it draws alone, whatever the launch"""
    from alphazero_amd import ops

    for n in (225, 5000):
        s, u = rand(700, n, torch.float32, 77)
        all_ = ops.sample_actions(s, u, top_k=30, top_p=0.9)
        for r in (0, 1, 350, 699):
            assert torch.equal(all_[r:r + 1], ops.sample_actions(s[r:r + 1], u[r:r + 1], top_k=30, top_p=0.9))
    assert ops.sample_actions(s[:0], u[:0]).shape == (0,)


def test_another_stream_and_a_graph():
    from alphazero_amd import ops

    s, u = rand(50, 225, torch.float32, 41)
    long_s, long_u = rand(4, 40000, torch.bfloat16, 42)
    want, want_l = ops.sample_actions(s, u, top_p=0.9), ops.sample_actions(long_s, long_u, top_k=50, top_p=0.9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.sample_actions(s, u, top_p=0.9)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out, out_l = ops.sample_actions(s, u, top_p=0.9), ops.sample_actions(long_s, long_u, top_k=50, top_p=0.9)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    for seed in (43, 44, 45):
        s2, u2 = rand(50, 225, torch.float32, seed)
        l2, lu2 = rand(4, 40000, torch.bfloat16, seed)
        s.copy_(s2), u.copy_(u2), long_s.copy_(l2), long_u.copy_(lu2)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.sample_actions(s2, u2, top_p=0.9))
        assert torch.equal(out_l, ops.sample_actions(l2, lu2, top_k=50, top_p=0.9))


def test_frequencies_follow_the_weights():
    """visits ** (1 / temperature), as play_moves samples: 200,000 draws, every cell within 5 standard deviations"""
    from alphazero_amd import ops

    visits = torch.tensor([0.0, 1.0, 7.0, 20.0, 2.0, 0.0, 10.0], device="cuda")
    rows = 200000
    u = torch.rand(rows, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    a = ops.sample_actions(visits.log().expand(rows, 7), u, temperature=2.0)
    p = (visits.double().cpu() ** 0.5)
    p = p / p.sum()
    n = torch.bincount(a.long().cpu(), minlength=7).double()
    assert n[0] == 0 and n[5] == 0
    assert bool(((n / rows - p).abs() <= 5 * (p * (1 - p) / rows).sqrt()).all())


@pytest.mark.parametrize("n", [225, 5000])
def test_temperatures_next_to_infinity(n):
    """the weights of scores however far apart become alike; masked scores still weigh nothing"""
    s, u = rand(8, n, torch.float32, 51)
    s[1] *= 1e38
    s[2, ::2] = 3e38
    s[2, 1::2] = -3e38
    s[3, ::3] = -math.inf
    s[4] *= 1e-30
    s[5, 0] = math.inf
    legal = torch.rand(8, n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(52)) < 0.5
    for t in (math.inf, 1e300, 1e39, 1e37, 1e30):
        check(s, u, t, 0, 0.5, 0.0, legal)
        check(s, u, t, 0, 0.75)
        check(s, u, t, 40, 0.5, 0.1, legal)


@pytest.mark.parametrize("n", [5, 1100])
def test_more_rows_than_one_launch_holds(n):
    from alphazero_amd import ops

    rows = (1 << 21) + 70
    s, _ = rand(1, n, torch.float32, 53)
    g = torch.Generator(device="cuda").manual_seed(54)
    u = torch.rand(rows, device="cuda", generator=g)
    k = torch.zeros(rows, dtype=torch.int32, device="cuda")
    k[-50:] = 1  # (the last launch reads its own rows' settings)
    got, logp = ops.sample_actions(s.expand(rows, n), u, top_k=k, temperature=torch.ones(rows, device="cuda"), return_logprobs=True)
    w = torch.exp((s[0].double() - s[0].max().double()))
    mass = torch.cumsum(w, 0)
    want = torch.searchsorted(mass, u.double() * mass[-1], right=True)
    want[-50:] = s[0].argmax()
    assert torch.equal(got.long(), want)
    lp = (w / mass[-1]).log()[want]
    lp[-50:] = 0.0
    assert bool(((logp.double() - lp).abs() <= 2.0 ** -23 * (1 + lp.abs())).all())


def test_rows_beyond_32_bit_offsets():
    """rows 2^30 scores apart: the last one starts at byte 2^33"""
    rows, far = 5, 1 << 30
    s = torch.empty(rows * far, dtype=torch.bfloat16, device="cuda").view(rows, far)
    on = torch.empty(rows * far, dtype=torch.bool, device="cuda").view(rows, far)
    for n in (300, 5000):
        v, u = rand(rows, n, torch.bfloat16, 55)
        s[:, :n], on[:, :n] = v, torch.rand(rows, n, device="cuda") < 0.5
        check(s[:, :n], u, 0.9, 0, 0.8, 0.0, on[:, :n])


@pytest.mark.parametrize("n", [8193, 65537, 131072])
def test_many_long_rows_draw_what_each_draws_alone(n):
    """512 rows and more take smaller workgroups: the same actions and log-probabilities, bit for bit"""
    from alphazero_amd import ops

    s, u = rand(520, n, torch.bfloat16, 78, 3.0)
    for kw in (dict(top_k=30, top_p=0.9), dict(top_p=0.8), dict(temperature=0.5, min_p=0.01), dict(top_k=2000)):
        a, lp = ops.sample_actions(s, u, return_logprobs=True, **kw)
        b, lq = ops.sample_actions(s[:500], u[:500], return_logprobs=True, **kw)
        assert torch.equal(a[:500], b) and torch.equal(lp[:500], lq)
    check(s[518:], u[518:].contiguous(), 1.0, 0, 0.8)
