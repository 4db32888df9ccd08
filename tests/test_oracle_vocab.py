"""Pins of the float64 definitions behind the vocabulary operators (no GPU): closed forms, and
gradients against differences."""
import math

import numpy as np
import pytest

from oracle import vocab_f64


def test_embedding_closed_form():
    x = np.arange(12, dtype=np.float64).reshape(4, 3)
    got = vocab_f64.embedding(x, np.array([[2, -1], [5, 3]]), scale=2.0, first_row=2)
    assert np.array_equal(got, [[[0, 2, 4], [0, 0, 0]], [[18, 20, 22], [6, 8, 10]]] * np.array(1.0))
    ends = np.array([np.iinfo(np.int64).min, np.iinfo(np.int64).max])
    assert not vocab_f64.embedding(x, ends, first_row=7).any()


def test_embedding_dx_is_the_transpose_of_the_lookup():
    rng = np.random.default_rng(1)
    x, ids = rng.normal(size=(7, 4)), rng.integers(-2, 12, (3, 5))
    dy = rng.normal(size=(3, 5, 4))
    dx, size, count = vocab_f64.embedding_dx(dy, ids, 7, scale=1.5, first_row=2)
    assert np.sum(dx * x) == pytest.approx(np.sum(dy * vocab_f64.embedding(x, ids, 1.5, 2)), rel=1e-13)
    assert count.sum() == np.sum((ids >= 2) & (ids < 9)) and (size >= np.abs(dx) - 1e-15).all()
    dx, _, count = vocab_f64.embedding_dx(dy, ids, 7, padding_idx=4, first_row=2)
    assert not dx[2].any() and count[2] == 0


def test_distill_closed_forms():
    # the teacher's one entry: minus log softmax there; a uniform student: log of the vocabulary
    r = vocab_f64.topk_distill(np.zeros((1, 8)), [[3]], [[5.0]])
    assert r["loss"][0] == pytest.approx(math.log(8)) and r["stats"][0, 1] == pytest.approx(math.log(8))
    assert r["dlogits"][0] == pytest.approx(np.full(8, 1 / 8) - np.eye(8)[3])
    # the student equals a teacher that names every column: nothing to learn
    z = np.random.default_rng(2).normal(size=(1, 6))
    r = vocab_f64.topk_distill(z, [list(range(6))], z + 3.0, temperature=2.5)
    assert abs(r["loss"][0]) < 1e-14 and np.abs(r["dlogits"]).max() < 1e-15
    # absent entries, absent label
    r = vocab_f64.topk_distill(z, [[-1, 6]], [[1.0, np.nan]], labels=[-100], hard_weight=1.0)
    assert r["loss"][0] == 0 and not r["dlogits"].any() and not r["stats"].any()


@pytest.mark.parametrize("temperature,soft,hard", [(1.0, 1.0, 0.0), (2.0, 0.7, 0.3), (0.5, 0.0, 1.0), (3.0, 1.0, 2.0)])
def test_distill_gradient_against_differences(temperature, soft, hard):
    rng = np.random.default_rng(3)
    z = rng.normal(size=(3, 9)) * 2
    idx = np.array([[0, 4, 4], [8, -1, 2], [-1, -1, 9]])  # one column twice, absent entries, none at all
    teacher = rng.normal(size=(3, 3))
    labels, dloss = np.array([4, -100, 1]), np.array([0.5, 2.0, 1.0])

    def f(z):
        return np.dot(dloss, vocab_f64.topk_distill(z, idx, teacher, temperature, soft, labels, hard)["loss"])

    grad = vocab_f64.topk_distill(z, idx, teacher, temperature, soft, labels, hard, dloss)["dlogits"]
    h = 1e-6
    for at in np.ndindex(z.shape):
        up, down = z.copy(), z.copy()
        up[at] += h
        down[at] -= h
        assert grad[at] == pytest.approx((f(up) - f(down)) / (2 * h), abs=2e-8), at
