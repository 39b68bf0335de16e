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
                lambda: ops.sample_actions(s, u, top_k=1.5), lambda: ops.sample_actions(s, u, top_k=-1), lambda: ops.sample_actions(s, u, min_p=1.1),
                lambda: ops.sample_actions(s, u, top_p=torch.ones(3, device="cuda")), lambda: ops.sample_actions(s, u, top_k=torch.ones(2, device="cuda"))):
        with pytest.raises(EngineError):
            bad()
