"""Refusals of the operators' entry points that need no GPU: they return before anything is launched."""
import ctypes as C

import pytest
import torch


def _lib():
    from alphazero_amd import _build
    from alphazero_amd.engine import load_library

    _build.build()
    return load_library()


def _sample(lib, **kw):
    a = dict(dtype=0, rows=2, n=9, scores=64, stride=9, legal=None, legal_stride=0, u=64, t=None, tv=1.0, k=None, kv=0, p=None, pv=1.0,
             mp=None, mpv=0.0, actions=64, logp=None)
    a.update(kw)
    return lib.az_sample_actions(a["dtype"], a["rows"], a["n"], a["scores"], a["stride"], a["legal"], a["legal_stride"], a["u"], a["t"],
                                 a["tv"], a["k"], a["kv"], a["p"], a["pv"], a["mp"], a["mpv"], a["actions"], a["logp"], None)


@pytest.mark.parametrize("bad", [dict(dtype=3), dict(rows=-1), dict(n=0), dict(n=(1 << 19) + 1), dict(scores=None), dict(u=None), dict(actions=None),
                                 dict(scores=66), dict(dtype=1, scores=65), dict(u=65), dict(actions=66), dict(logp=65), dict(stride=-9),
                                 dict(legal=64, legal_stride=-1), dict(tv=-1.0), dict(tv=float("nan")), dict(pv=-0.1), dict(mpv=1.5),
                                 dict(mpv=float("nan")), dict(t=65), dict(k=66), dict(p=65), dict(mp=65)])
def test_sample_refuses(bad):
    lib = _lib()
    assert _sample(lib, **bad) == -1
    assert lib.az_tower_last_error().startswith(b"sample:")


def test_sample_of_no_rows():
    assert _sample(_lib(), rows=0) == 0


def test_sample_python_refusals():
    from alphazero_amd import ops
    from alphazero_amd.engine import EngineError

    s, u = torch.zeros(2, 9), torch.zeros(2)
    with pytest.raises(EngineError, match="no CPU path"):
        ops.sample_actions(s, u)
    with pytest.raises(EngineError, match="dtype"):
        ops.sample_actions(s.double(), u)
    with pytest.raises(EngineError, match="expected a tensor"):
        ops.sample_actions([1.0], u)


@pytest.mark.gpu
def test_sample_python_refusals_on_the_gpu():
    from alphazero_amd import ops
    from alphazero_amd.engine import EngineError

    s, u = torch.zeros(2, 9, device="cuda"), torch.zeros(2, device="cuda")
    for bad in (lambda: ops.sample_actions(s[0], u), lambda: ops.sample_actions(s, u[:1]), lambda: ops.sample_actions(s, u.half()),
                lambda: ops.sample_actions(s, u.cpu()), lambda: ops.sample_actions(s.t(), torch.zeros(9, device="cuda")),
                lambda: ops.sample_actions(s[:, :0], u), lambda: ops.sample_actions(s, u, legal=torch.ones(2, 9, device="cuda")),
                lambda: ops.sample_actions(s, u, legal=torch.ones(2, 8, device="cuda", dtype=torch.bool)),
                lambda: ops.sample_actions(s, u, temperature=-1.0), lambda: ops.sample_actions(s, u, temperature=float("nan")),
                lambda: ops.sample_actions(s, u, top_k=1.5), lambda: ops.sample_actions(s, u, top_k=float("inf")), lambda: ops.sample_actions(s, u, top_k=-1), lambda: ops.sample_actions(s, u, min_p=1.1),
                lambda: ops.sample_actions(s, u, top_p=torch.ones(3, device="cuda")), lambda: ops.sample_actions(s, u, top_k=torch.ones(2, device="cuda"))):
        with pytest.raises(EngineError):
            bad()


def _norm(lib, backward=False, **kw):
    a = dict(dtype=0, pd=0, n=2, hw=9, c=8, g=2, act=1, eps=1e-5, x=64, r=None, w=None, b=None, dy=64, y=64, stats=64, ws=64, size=1 << 20)
    a.update(kw)
    if backward:
        return lib.az_group_norm_backward(a["dtype"], a["pd"], a["n"], a["hw"], a["c"], a["g"], a["act"], a["x"], a["r"], a["w"], a["b"], a["dy"],
                                          a["stats"], a["y"], None, None, None, a["ws"], a["size"], None)
    return lib.az_group_norm_forward(a["dtype"], a["pd"], a["n"], a["hw"], a["c"], a["g"], a["act"], a["eps"], a["x"], a["r"], a["w"], a["b"], a["y"],
                                     a["stats"], a["ws"], a["size"], None)


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("bad", [dict(dtype=5), dict(pd=1), dict(dtype=1, pd=2), dict(act=3), dict(act=-1), dict(n=-1), dict(hw=-1), dict(c=0), dict(g=0),
                                 dict(g=3), dict(c=16385, g=1), dict(c=2048, g=2048), dict(n=(1 << 28) + 1), dict(hw=(1 << 28) + 1), dict(x=None),
                                 dict(stats=None), dict(ws=None), dict(size=16), dict(x=66), dict(dtype=1, pd=1, w=65), dict(stats=68), dict(r=65)])
def test_norm_refuses(bad, backward):
    lib = _lib()
    assert _norm(lib, backward, **bad) == -1
    assert lib.az_tower_last_error().startswith(b"group norm:")


@pytest.mark.parametrize("backward", [False, True])
def test_norm_refuses_more_workgroups_than_a_launch_holds(backward):
    lib = _lib()
    for n, c, g in ((1 << 24, 1, 1), (1 << 21, 8, 8), ((1 << 14), 1024, 1024)):
        assert _norm(lib, backward, n=n, c=c, g=g, hw=1, size=1 << 60) == -1
        assert b"2^24" in lib.az_tower_last_error()
        assert lib.az_group_norm_workspace(int(backward), n, 1, c, g) == -1


def test_norm_sizes():
    lib = _lib()
    assert _norm(lib, n=0) == 0 and _norm(lib, hw=0) == 0
    assert lib.az_group_norm_workspace(0, 4, 81, 64, 5) == -1
    assert lib.az_group_norm_workspace(0, 0, 81, 64, 8) == 0
    assert lib.az_group_norm_workspace(1, 4, 81, 64, 8) > 0


def test_norm_python_refusals():
    from alphazero_amd import ops
    from alphazero_amd.engine import EngineError
    from alphazero_amd.nets import GomokuNet, GroupNormAct

    with pytest.raises(EngineError, match="no CPU path"):
        ops.group_norm_act(torch.zeros(2, 8, 3, 3), 2)
    with pytest.raises(EngineError, match="no CPU path"):
        GroupNormAct(2, 8)(torch.zeros(2, 8, 3, 3))
    with pytest.raises(EngineError, match="dtype"):
        ops.group_norm_act(torch.zeros(2, 8, 3, 3, dtype=torch.float64), 2)
    with pytest.raises(ValueError):
        GroupNormAct(3, 8)
    with pytest.raises(ValueError):
        GomokuNet(9, 16, 1, norm="layer")


@pytest.mark.gpu
def test_norm_python_refusals_on_the_gpu():
    from alphazero_amd import ops
    from alphazero_amd.engine import EngineError

    x, w = torch.zeros(2, 8, 3, 3, device="cuda"), torch.ones(8, device="cuda")
    for bad in (lambda: ops.group_norm_act(x[0], 2), lambda: ops.group_norm_act(x, 3), lambda: ops.group_norm_act(x, 0), lambda: ops.group_norm_act(x, 2.0),
                lambda: ops.group_norm_act(x, 2, w[:4]), lambda: ops.group_norm_act(x, 2, w, w.half()), lambda: ops.group_norm_act(x.half(), 2, w.bfloat16()),
                lambda: ops.group_norm_act(x, 2, w.cpu()), lambda: ops.group_norm_act(x, 2, activation="gelu"), lambda: ops.group_norm_act(x, 2, eps=-1.0),
                lambda: ops.group_norm_act(x, 2, residual=x.half()), lambda: ops.group_norm_act(x, 2, residual=x[:1]),
                lambda: ops.group_norm_act(x, 2, eps=float("nan"))):
        with pytest.raises(EngineError):
            bad()


def _ortho(lib, **kw):
    a = dict(dtype=0, count=1, ins=[512], outs=[512], rows=[100], cols=[200], steps=5, a=3.4445, b=-4.775, c=2.0315, eps=1e-7, ws=512, size=1 << 24)
    a.update(kw)
    n = len(a["ins"])
    return lib.az_orthogonalize(a["dtype"], a["count"], (C.c_void_p * n)(*a["ins"]), (C.c_void_p * n)(*a["outs"]), (C.c_int32 * n)(*a["rows"]),
                                (C.c_int32 * n)(*a["cols"]), a["steps"], a["a"], a["b"], a["c"], a["eps"], a["ws"], a["size"], None)


@pytest.mark.parametrize("bad", [dict(dtype=7), dict(count=-1), dict(rows=[-1]), dict(cols=[65537]), dict(steps=0), dict(steps=65), dict(eps=-1.0),
                                 dict(eps=float("nan")), dict(a=3.0, b=0.0, c=0.0), dict(a=float("nan")), dict(c=50.0), dict(ins=[None]), dict(outs=[None]),
                                 dict(ins=[514]), dict(dtype=1, outs=[513]), dict(ws=None), dict(ws=128), dict(size=100)])
def test_ortho_refuses(bad):
    lib = _lib()
    assert _ortho(lib, **bad) == -1
    assert lib.az_tower_last_error().startswith(b"orthogonalize:")


def test_ortho_of_nothing():
    lib = _lib()
    assert _ortho(lib, rows=[0]) == 0
    assert lib.az_orthogonalize(0, 0, None, None, None, None, 5, 3.4445, -4.775, 2.0315, 1e-7, None, 0, None) == 0
    assert lib.az_orthogonalize_workspace(0, 1, (C.c_int32 * 1)(-1), (C.c_int32 * 1)(1)) == -1
    assert lib.az_orthogonalize_workspace(0, 1, (C.c_int32 * 1)(0), (C.c_int32 * 1)(9)) == 0


def test_ortho_python_refusals():
    from alphazero_amd import ops
    from alphazero_amd.engine import EngineError
    from alphazero_amd.learner import Muon

    for bad in (torch.zeros(3, 4), [torch.zeros(3, 4)], torch.zeros(3), torch.zeros(2, 2, 2, 2), "m", [1.0], torch.zeros(3, 4, dtype=torch.float64)):
        with pytest.raises(EngineError):
            ops.orthogonalize(bad)
    with pytest.raises(EngineError, match="steps"):
        ops.orthogonalize([], steps=0)
    with pytest.raises(EngineError, match="coefficients"):
        ops.orthogonalize([], coefficients=(1.0, 2.0))
    with pytest.raises(ValueError):
        Muon([torch.nn.Parameter(torch.zeros(2, 2))], momentum=1.0)
    p = torch.nn.Parameter(torch.zeros(2, 2))
    p.grad = torch.ones(2, 2)
    with pytest.raises(EngineError, match="no CPU path"):
        Muon([p]).step()


@pytest.mark.gpu
def test_ortho_python_refusals_on_the_gpu():
    from alphazero_amd import ops
    from alphazero_amd.engine import EngineError

    m = torch.zeros(3, 4, device="cuda")
    for bad in (lambda: ops.orthogonalize([m, m.half()]), lambda: ops.orthogonalize([m, m.cpu()]), lambda: ops.orthogonalize([m[0]]),
                lambda: ops.orthogonalize(m, coefficients=(3.0, 0.0, 0.0)), lambda: ops.orthogonalize(m, eps=-1.0), lambda: ops.orthogonalize(m, steps=2.5)):
        with pytest.raises(EngineError):
            bad()
