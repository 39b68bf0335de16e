"""play_match(opening_plies=...): the first moves drawn from the searches' visit counts (ops.sample_actions)."""
import pytest
import torch

from .helpers import HashNet

pytestmark = pytest.mark.gpu


def _play(n_games, **kw):
    from alphazero_amd import games
    from alphazero_amd.match import play_match

    return play_match(games.DotsAndBoxesGame, HashNet(24, 5.0), HashNet(24, 3.0), n_games, num_simulation=24, record_moves=True, **kw)


def _games(out):
    return torch.stack(out["moves"], 1).tolist()


def test_drawn_openings_make_different_games_and_a_seed_repeats_them():
    plain, drawn = _play(12), _play(12, opening_plies=4, temperature=1.0, seed=7)
    assert len({tuple(g) for g in _games(plain)}) == 2  # who moves first is all that differs
    assert len({tuple(g) for g in _games(drawn)}) > 6
    assert _games(drawn) == _games(_play(12, opening_plies=4, temperature=1.0, seed=7))
    assert _games(drawn) != _games(_play(12, opening_plies=4, temperature=1.0, seed=8))
    assert drawn["a_wins"] + drawn["b_wins"] + drawn["draws"] == 12


def test_openings_cut_to_the_best_move_are_the_deterministic_match():
    plain = _games(_play(6))
    assert _games(_play(6, opening_plies=100, temperature=0.0)) == plain
    assert _games(_play(6, opening_plies=100, top_k=1)) == plain
    assert _games(_play(6, opening_plies=100, top_p=0.0)) == plain
