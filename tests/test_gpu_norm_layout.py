"""What the norms of a group-norm net are given, on the framework's own paths, lies channels last: none of them copies its sample."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture
def given(monkeypatch):
    from alphazero_amd import ops

    seen, dense = [], ops._dense
    monkeypatch.setattr(ops, "_dense", lambda t: (seen.append(t.is_contiguous(memory_format=torch.channels_last)), dense(t))[1])
    return seen


def test_training_step(given):
    from alphazero_amd.learner import calculate_loss
    from alphazero_amd.nets import GomokuNet

    net = GomokuNet(9, 64, 2, norm="group").cuda()
    x = torch.randint(-1, 2, (16, 9, 9, 9), device="cuda").float()
    loss, _, _ = calculate_loss(net, x, torch.softmax(torch.randn(16, 81, device="cuda"), 1), torch.randn(16, 1, device="cuda").sign())
    loss.backward()
    assert len(given) == 7 + 2 + 7 and all(given[:9])  # x of seven norms, two residuals; then the gradients, as the convolutions leave them


def test_self_play(given):
    from alphazero_amd import Engine
    from alphazero_amd.arena import SelfPlayRunner
    from alphazero_amd.nets import GomokuNet

    net = GomokuNet(9, 64, 2, norm="group").cuda().eval()
    eng = Engine(2, 6, 4, board_size=9, device="cuda:0")
    SelfPlayRunner(eng, net, 4, seed=3).move_round(torch.ones(6, device="cuda"))
    eng.check()
    eng.close()
    assert len(given) and len(given) % 9 == 0 and all(given)
