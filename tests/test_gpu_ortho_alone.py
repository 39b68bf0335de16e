"""ops.orthogonalize: what a matrix's result may and may not owe to the others of its call, and how exact bf16 results of short sides are."""
import ctypes as C
import math

import pytest
import torch

from .test_gpu_ortho import COEF, SHAPES, check, make, plain

pytestmark = pytest.mark.gpu


def _norm_sums(ms):
    """the first matrix's 256 partial sums of squares, as a call of the C entry leaves them: the workspace begins with a table of
    (in, out, byte offset of the buffers, rows, cols), and a matrix's buffers with these sums"""
    from alphazero_amd.engine import load_library

    lib, n = load_library(), len(ms)
    rows, cols = (C.c_int32 * n)(*[m.shape[0] for m in ms]), (C.c_int32 * n)(*[m.shape[1] for m in ms])
    out = [torch.empty_like(m) for m in ms]
    ws = torch.zeros(lib.az_orthogonalize_workspace(0, n, rows, cols), dtype=torch.uint8, device="cuda")
    ptrs = lambda ts: (C.c_void_p * n)(*[t.data_ptr() for t in ts])
    assert lib.az_orthogonalize(0, n, ptrs(ms), ptrs(out), rows, cols, 1, *COEF, 1e-7, ws.data_ptr(), ws.numel(),
                                torch.cuda.current_stream().cuda_stream) == 0
    at = int(ws[16:24].view(torch.int64))
    return ws[at:at + 2048].view(torch.float64).clone()


def test_a_norm_is_summed_in_the_same_order_beside_larger_matrices():
    m, larger = make((100, 200), torch.float32, 1), make((700, 3000), torch.float32, 2)
    alone = _norm_sums([m])
    assert abs(float(alone.sum()) / float((m.double() ** 2).sum()) - 1) < 1e-12
    assert torch.equal(alone, _norm_sums([m, larger]))


def test_a_norm_is_summed_in_the_same_order_at_any_address():
    m = make((100, 203), torch.float32, 3)
    store = torch.empty(m.numel() + 3, device="cuda")
    for off in (1, 2, 3):
        moved = store[off:off + m.numel()].view(m.shape)
        moved.copy_(m)
        assert torch.equal(_norm_sums([moved]), _norm_sums([m]))


@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (7, 1), (20, 700), (32, 768), (33, 32), (768, 33), (64, 64), (64, 576), (64, 769), (2, 3000), (4096, 64)], ids=lambda s: "x".join(map(str, s)))
def test_bf16_results_of_short_sides_are_off_by_their_own_rounding(shape):
    """Factors of 22 bits leave the result x + d before its rounding; |round(x + d) - x| <= |round(x) - x| + 2 |d| entry by entry.  d: four
    times the larger of two runs of the definition whose X, A and B carry errors of that size (as in test_gpu_ortho)"""
    from alphazero_amd import ops

    level = 2.0 ** -22 + 2.0 ** -24 * math.sqrt(max(shape))
    larger = make((100, 900), torch.bfloat16, 77)
    for seed in range(4):
        m = make(shape, torch.bfloat16, seed * 131 + shape[0], 0.01)
        ref = plain(m)
        gen = torch.Generator(device="cuda").manual_seed(1)
        d = 4 * max(float((plain(m, noise=level, gen=gen) - ref).norm()) for _ in range(2))
        own = float((ref.bfloat16().double() - ref).norm())
        for got in (ops.orthogonalize(m), ops.orthogonalize([larger, m])[1]):
            err = float((got.double() - ref).norm())
            assert err <= own + 2 * d + 2.0 ** -24, (err, own, d)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_small_matrices_beside_larger_ones_against_the_definition(dtype):
    """in one call with a larger matrix they take another kernel than alone; both are held to the definition"""
    from alphazero_amd import ops

    small = [make(s, dtype, i, 0.01) for i, s in enumerate(s for s in SHAPES if min(s) <= 64 and max(s) <= 768)]
    assert len(small) > 12
    for larger in (make((100, 900), dtype, 78), make((60, 900), dtype, 79)):
        got = ops.orthogonalize([*small, larger])
        for m, o, alone in zip(small, got, ops.orthogonalize(small)):
            check(m, o)
            check(m, alone)
        assert torch.equal(got[-1], ops.orthogonalize(larger))


@pytest.mark.parametrize("shape", [(64, 100), (100, 200)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("k", [14, 20, 26, 40])
def test_norms_far_below_eps(shape, k):
    """|M| = 2^-k eps: X0 is about 2^-k, every step multiplies it by 3.4445 (its cube is far below it).  Entries of X stand in steps of 2^-38
    (2^-24 over the scale 2^14), so that 2^-39 may be lost at X0 and at each step, and 3.4445^5 (1 + 1 / 3.4445 + ..) = 684 times that in
    all; beside it five times the 2^-22 of the halves and the 2^-23 of f32 arithmetic"""
    from alphazero_amd import ops

    eps = 1e-7
    m = make(shape, torch.float32, 5)
    m = m * float(eps * 2.0 ** -k / m.double().norm())
    ref = plain(m, eps=eps)
    got = ops.orthogonalize(m, eps=eps)
    assert bool(((got.double() - ref).abs() <= 2.0 ** -19 * ref.abs() + 684 * 2.0 ** -39).all()), float((got.double() - ref).abs().max())
    assert k == 40 or float(got.abs().max()) > 0


def test_buffers_that_start_beyond_4_gib():
    """a 4,096 x 65,536 f32 matrix has 3.1 GiB of the workspace (X, two transposes, A, B): the third one's begin past 6 GiB, and its result is the
    same, bit for bit"""
    from alphazero_amd import ops

    m = torch.randn(4096, 65536, device="cuda", generator=torch.Generator(device="cuda").manual_seed(72))
    one = ops.orthogonalize(m, steps=1)
    for o in ops.orthogonalize([m, m, m], steps=1):
        assert torch.equal(o, one)


@pytest.mark.parametrize("dtype,other", [(torch.float32, (1800, 1900)), (torch.float16, (1800, 1900)), (torch.bfloat16, (100, 900)), (torch.bfloat16, (1800, 1900))], ids=str)
def test_small_matrices_beside_those_that_share_no_launch(dtype, other):
    """a larger matrix of another tile size, or of another number of halves, leaves the small ones their own kernel: nothing changes, bit for bit"""
    from alphazero_amd import ops

    small = [make(s, dtype, i, 0.01) for i, s in enumerate(((64, 576), (20, 700), (1, 7), (33, 32), (768, 64)))]
    larger = make(other, dtype, 90)
    got = ops.orthogonalize([small[0], larger, *small[1:]])
    assert torch.equal(got[1], ops.orthogonalize(larger))
    for o, alone in zip([got[0], *got[2:]], ops.orthogonalize(small)):
        assert torch.equal(o, alone)
