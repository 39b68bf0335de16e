"""learner.Muon under DataParallelLearner with two ranks (gloo, CPU; the orthogonalisation is computed plainly, the kernel's place): each step
is the one that a single process takes on the mean of the ranks' gradients, and the ranks hold the same weights, bit for bit."""
import socket
import subprocess
import sys

from .conftest import ROOT

_WORKER = r"""
import sys, torch, torch.distributed as dist
rank, port, root = int(sys.argv[1]), sys.argv[2], sys.argv[3]
sys.path.insert(0, root)
from alphazero_amd import ops
from alphazero_amd.learner import DataParallelLearner, Muon, calculate_loss
from alphazero_amd.nets import TicTacToeNet
def plain(ms, steps=5, a=3.4445, b=-4.7750, c=2.0315, eps=1e-7):
    out = []
    for m in ms:
        x = m.double(); tall = x.shape[0] > x.shape[1]
        x = x.t() if tall else x
        x = x / (x.norm() + eps)
        for _ in range(steps):
            s = x @ x.t()
            x = a * x + (b * s + c * s @ s) @ x
        out.append((x.t() if tall else x).to(m.dtype).contiguous())
    return out
ops.orthogonalize = plain
dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=2)
torch.manual_seed(0)
model, ref = TicTacToeNet(), TicTacToeNet()
ref.load_state_dict(model.state_dict())
g = torch.Generator().manual_seed(7)
def batch():
    return (torch.randint(-1, 2, (16, 9, 3, 3), generator=g).float(), torch.softmax(torch.randn(16, 9, generator=g), 1),
            torch.randint(-1, 2, (16, 1), generator=g).float())
batches = [[batch() for _ in range(2)] for _ in range(3)]  # both ranks know all: rank r trains on the r-th of every step
class Pool:
    def sample(self, n, timeout=None):
        return batches[step][rank]
dp = DataParallelLearner(model, Muon(model.parameters(), weight_decay=0.01), bucket_bytes=64 << 10)
opt = Muon(ref.parameters(), weight_decay=0.01)
ok = len(dp.buckets) > 1
for step in range(3):
    dp.step(Pool(), 16)
    opt.zero_grad()
    ref.train()
    for b in batches[step]:
        (0.5 * calculate_loss(ref, *b)[0]).backward()
    opt.step()
    # the orthogonalisation amplifies roundings of the gradients' smallest directions 3.4-fold a step: 1e-7 * 485 of an update of 0.02
    ok = ok and all(torch.allclose(p, q, rtol=0, atol=1e-5 * (step + 1)) for p, q in zip(model.parameters(), ref.parameters()))
flat = torch.cat([q.detach().reshape(-1) for q in model.parameters()])
other = [torch.empty_like(flat) for _ in range(2)]
dist.all_gather(other, flat)
ok = ok and torch.equal(other[0], other[1])
dist.destroy_process_group()
sys.exit(0 if ok else 3)
"""


def test_two_ranks_take_the_step_of_their_mean_gradient(tmp_path):
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    script = tmp_path / "muon.py"
    script.write_text(_WORKER)
    procs = [subprocess.Popen([sys.executable, str(script), str(r), str(port), ROOT]) for r in range(2)]
    assert [p.wait(timeout=180) for p in procs] == [0, 0]
