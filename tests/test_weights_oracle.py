"""The oracle of attention weights, of the choice of tokens and of their moving,
against closed forms and cases worked out by hand."""

import numpy as np
import pytest
import torch

from oracle import weights_oracle as W


def test_probabilities_of_equal_scores_are_equal_and_causal():
    k = np.zeros((5, 2, 128))
    q = np.ones((2, 4, 128))
    p = W.probabilities(q, k, np.ones(5, bool), 0.1, [4, 5])
    assert np.allclose(p[0, :, :4], 0.25) and (p[0, :, 4] == 0).all()
    assert np.allclose(p[1], 0.2)
    assert np.allclose(W.by_kv_head(p, 2).sum(), 2 * 4)
    ok = np.array([True, False, True, True, True])
    p = W.probabilities(q, k, ok, 0.1, [2, 0])
    assert np.allclose(p[0, :, 0], 1) and (p[0, :, 1:] == 0).all() and (p[1] == 0).all()


def test_probabilities_are_torch_softmax():
    gen = torch.Generator().manual_seed(0)
    q = torch.randn(3, 6, 128, generator=gen, dtype=torch.float64)
    k = torch.randn(9, 2, 128, generator=gen, dtype=torch.float64)
    p = W.probabilities(q.numpy(), k.numpy(), np.ones(9, bool), 0.3, [7, 8, 9])
    for i in range(3):
        for h in range(6):
            s = k[:7 + i, h // 3] @ q[i, h] * 0.3
            assert np.allclose(p[i, h, :7 + i], torch.softmax(s, -1).numpy(), atol=1e-15)


@pytest.mark.parametrize("budget,recent,start,want", [
    (3, 0, 0, [1, 3, 4]), (3, 1, 0, [1, 3, 5]), (3, 1, 1, [0, 1, 5]), (2, 2, 1, [0, 5]),
    (6, 9, 9, [0, 1, 2, 3, 4, 5]), (4, 0, 0, [1, 2, 3, 4]), (1, 0, 3, [0])])
def test_select_by_hand(budget, recent, start, want):
    weights = np.zeros((2, 1, 4), np.float32)
    weights[1, 0] = [0.5, 9.0, 1.0, 2.0]  # positions 0 to 3
    weights[0, 0, :2] = [2.0, 1.0]        # 4 and 5: a tie with 3, one with 2
    kept, n = W.select(weights, 6, [1, 0], budget, recent, start)
    assert n == min(6, budget) and kept[0, :n].tolist() == want and (kept[0, n:] == -1).all()


def test_evict_by_hand():
    a = np.arange(8, dtype=np.float32).reshape(2, 4, 1)
    W.evict([a], np.array([[1, 2, 5, -1]], np.int32), 3, [1, 0], 4)
    # positions 0 to 3 were 4, 5, 6, 7 and 4, 5 were 0, 1
    assert a[1, :, 0].tolist() == [5, 6, 1, 7] and a[0, :, 0].tolist() == [0, 1, 2, 3]
