"""Ranking against 4-bit items where fp32 ranking has rules of its own."""
import numpy as np
import pytest
import torch

from src.evaluation import Evaluator

pytestmark = pytest.mark.gpu


def _both(cuda, users, items, k, seen):
    ptr = np.concatenate([[0], np.cumsum([len(s) for s in seen])]).astype(np.int64)
    col = np.concatenate(seen).astype(np.int32)
    return [Evaluator(device=cuda, item_bits=bits).topk(users, items, list(range(len(users))), k,
                                                        ptr, col) for bits in (32, 4)]


def _exact_items(n, cuda):
    """Items that 4 bits hold exactly (a group's largest value is 6) and whose scores differ."""
    items = torch.zeros(n, 64)
    items[:, 0], items[:, 32] = 6.0, 6.0
    codes = torch.arange(n)
    for j, c in enumerate((1, 2, 3)):
        items[:, c] = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6])[(codes >> (3 * j)) & 7]
    users = torch.zeros(3, 64)
    users[:, 1:4] = torch.tensor([[1.0, 20.0, 400.0], [-1.0, -20.0, -400.0], [400.0, 1.0, 20.0]])
    return users.to(cuda), items.to(cuda)


def test_items_without_a_score_rank_last(cuda):
    users, items = _exact_items(300, cuda)
    items[7, 5], items[40, 33] = float("nan"), float("nan")
    seen = [[3, 200], [], [7, 299]]
    full, four = _both(cuda, users, items, 100, seen)
    assert torch.equal(full, four)
    for r in four:
        assert 7 not in r.tolist() and 40 not in r.tolist()


def test_more_places_than_items(cuda):
    """Places that no item fills hold -1, as in the fp32 ranking."""
    users, items = _exact_items(12, cuda)
    full, four = _both(cuda, users, items, 20, [[3, 5], [], [11]])
    assert four.shape == (3, 20) and torch.equal(full, four)
    assert (four[:, 12:] == -1).all()
