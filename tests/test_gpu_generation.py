"""The operators together, as a generation of the training loop uses them: self-play and training of a group-norm net with Muon, then a
match with drawn openings between the net before and after."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("norm,optimizer", [("group", "muon"), ("batch", "muon"), ("group", "adam")])
def test_self_play_training_and_a_match(norm, optimizer):
    from alphazero_amd import games
    from alphazero_amd.loop import SelfPlayTrainLoop
    from alphazero_amd.match import play_match
    from alphazero_amd.nets import GomokuNet

    torch.manual_seed(3)
    net = GomokuNet(9, 64, 1, norm=norm)
    before = copy.deepcopy(net)
    dev = torch.device("cuda", 0)
    loop = SelfPlayTrainLoop(net, 2, 9, 24, 8, dev, batch_size=64, train_steps_per_move=2, min_samples=64, nn_dtype=torch.float32,
                             ring_capacity=4096, optimizer=optimizer)
    out = {}
    for _ in range(60):  # until games have ended and steps were taken
        out = loop.run(1)
        if out["train_steps"] >= 6:
            break
    assert out["train_steps"] >= 6
    moved = [k for (k, p), q in zip(net.named_parameters(), before.parameters()) if not torch.equal(p.cpu(), q)]
    assert len(moved) == len(list(net.parameters()))
    assert all(bool(torch.isfinite(p).all()) for p in net.parameters())
    if norm == "group":  # the player's copy follows
        assert all(torch.equal(p, q) for p, q in zip(loop.player.parameters(), loop.master.parameters()))
    res = play_match(games.Gomoku9Game, net, before, 8, num_simulation=8, opening_plies=6, top_p=0.95, min_p=0.05, seed=2, record_moves=True)
    assert res["a_wins"] + res["b_wins"] + res["draws"] == 8
    assert len({tuple(int(m[i]) for m in res["moves"][:6]) for i in range(8)}) > 2


def test_the_loop_refuses_an_unknown_optimizer():
    from alphazero_amd.loop import SelfPlayTrainLoop
    from alphazero_amd.nets import GomokuNet

    with pytest.raises(ValueError):
        SelfPlayTrainLoop(GomokuNet(9, 64, 1), 2, 9, 4, 4, torch.device("cuda", 0), optimizer="sgd")
