"""The package imports where torch has no GPU support at all; its operators then refuse what they are given."""
import subprocess
import sys

from .conftest import ROOT

CODE = """
import torch
for name in [n for n in dir(torch._C) if n.startswith("_cuda_")]:
    delattr(torch._C, name)
import alphazero_amd.match, alphazero_amd.loop, alphazero_amd.nets, alphazero_amd.ops as ops
from alphazero_amd.engine import EngineError
try:
    ops.sample_actions(torch.zeros(1, 9), torch.zeros(1))
except EngineError as e:
    assert "no CPU path" in str(e)
    print("imported and refused")
"""


def test_imports_without_gpu_support_in_torch():
    out = subprocess.run([sys.executable, "-c", CODE], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and "imported and refused" in out.stdout, out.stderr[-2000:]


def test_a_net_saved_whole_before_the_choice_of_norms():
    import torch

    from alphazero_amd.nets import GomokuNet

    net = GomokuNet(9, 8, 1).eval()
    x = torch.zeros(1, 9, 9, 9)
    want = net(x)[0]
    old = GomokuNet.__new__(GomokuNet)  # what unpickling makes of it: the attributes of then
    old.__dict__ = {k: v for k, v in net.__dict__.items() if k != "_channels_last"}
    assert torch.equal(old(x)[0], want)
