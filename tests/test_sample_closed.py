"""Sampling from rows in which a mask closed tokens (logits of -inf), on the host."""
import numpy as np
import pytest

from woolly_b200.engine import (GenerationConfig, last_open, sample_from_distribution, sample_next_token)


class Draw:
    def __init__(self, u):
        self.u = np.float32(u)

    def random(self, dtype=None):
        return self.u


NEAR = float(np.float32(1) - np.float32(2.0 ** -24))  # the largest draw


def closed_rows(seed, rows, V, share):
    """Random rows with `share` of the ids open, never the last id."""
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((rows, V)) * 3).astype(np.float32)
    shut = rng.random((rows, V)) >= share
    shut[:, -1] = True
    shut[np.arange(rows), rng.integers(0, V - 1, rows)] = False
    x[shut] = -np.inf
    return x, shut


@pytest.mark.parametrize("V,share", [(50, 0.1), (32000, 0.5), (1000, 0.003)])
@pytest.mark.parametrize("kw", [dict(temperature=1.0), dict(temperature=0.7, top_p=0.9999999),
                                dict(temperature=0.0, top_p=0.9999999), dict(temperature=1.0, top_k=5, top_p=0.999),
                                dict(temperature=0.0)])
def test_a_closed_token_is_never_picked(V, share, kw):
    x, shut = closed_rows(V, 30, V, share)
    for u in (NEAR, 0.5, 0.0):
        for row, s in zip(x, shut):
            assert not s[sample_next_token(row, GenerationConfig(**kw), Draw(u))]


def test_rows_without_closed_tokens_fall_back_to_the_last_index():
    p = np.zeros(7, np.float32)
    assert sample_from_distribution(p, Draw(0.3)) == 6
    x = np.zeros(7, np.float32)
    # seven equal probabilities sum to less than the draw, and to less than top_p
    assert sample_next_token(x, GenerationConfig(temperature=1.0), Draw(NEAR)) == 6
    assert sample_next_token(x, GenerationConfig(temperature=0.0, top_p=0.99999994), Draw(0)) == 6


def test_rows_that_leave_nothing():
    assert last_open(np.float32([1, -np.inf, 2, -np.inf])) == 2
    assert last_open(np.full(4, -np.inf)) == 3
    for bad in (np.nan, np.inf):
        x = np.float32([0.0, bad, 1.0, -np.inf])
        with np.errstate(invalid="ignore"):
            for t in (0.0, 1.0):
                assert sample_next_token(x, GenerationConfig(temperature=t), Draw(0.5)) == 2
