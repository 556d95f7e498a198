"""The token-training operators' float64 restatements (oracle/tokens.py): their gradients against
central differences, and their conventions for tokens without a row, a label or a class left."""
import numpy as np
import pytest

from oracle import tokens as ot


def problem(T, V, C, bias, seed=0):
    rng = np.random.default_rng(seed)
    x, w = rng.standard_normal((T, C)), rng.standard_normal((V, C)) * .5
    b = rng.standard_normal(V) if bias else None
    labels = rng.integers(-2, V + 2, T)
    return rng, x, w, b, labels, rng.standard_normal(T)


@pytest.mark.parametrize('bias', [False, True])
@pytest.mark.parametrize('T,V,C', [(1, 1, 8), (5, 3, 8), (7, 11, 16)])
def test_xent_gradients_are_the_losses_differences(T, V, C, bias):
    rng, x, w, b, labels, dloss = problem(T, V, C, bias)
    dx, dw, db, _, _ = ot.linear_xent_bwd(x, w, labels, dloss, b)

    def value(x, w, b):
        return float((ot.linear_xent(x, w, labels, b)[0] * dloss).sum())

    h = 1e-5
    for i, got in ((0, dx), (1, dw), (2, db)):
        if i == 2 and b is None:
            continue
        step = rng.standard_normal(got.shape)
        ends = []
        for sign in (1, -1):
            args = [x, w, b]
            args[i] = args[i] + sign * h * step
            ends.append(value(*args))
        # central differences: error h^2 times the third derivative (below 1e-7 here) and the
        # values' rounding over h (below 1e-9)
        assert abs((ends[0] - ends[1]) / (2 * h) - float((got * step).sum())) < 1e-6


def test_xent_rows_without_a_label_or_a_class():
    _, x, w, _, _, dloss = problem(4, 3, 8, False)
    labels = np.array([0, -100, 3, 2])
    x[1] = np.nan
    loss, lse = ot.linear_xent(x, w, labels)
    dx, dw, _, _, rows = ot.linear_xent_bwd(x, w, labels, dloss)
    assert list(rows) == [0, 3] and np.isfinite(dw).all()
    assert (loss[[1, 2]] == 0).all() and (lse[[1, 2]] == -np.inf).all() and (dx[[1, 2]] == 0).all()
    loss, lse = ot.linear_xent(x, w, labels, np.full(3, -np.inf))
    assert (loss == 0).all() and (lse == -np.inf).all()


def test_embed_gradient_is_the_lookups_difference():
    rng = np.random.default_rng(1)
    table, ids = rng.standard_normal((5, 4)), np.array([0, 4, 4, -1, 5, 2])
    dout, step = rng.standard_normal((6, 4)), rng.standard_normal((5, 4))
    # linear: the difference is exact up to rounding
    diff = ((ot.embed(ids, table + step, 3.) - ot.embed(ids, table, 3.)) * dout).sum()
    assert abs(diff - (ot.embed_bwd(ids, dout, 5, 3.) * step).sum()) < 1e-12
    assert (ot.embed(ids, table, 3.)[[3, 4]] == 0).all()


def test_clip_bounds_the_norm():
    grads = [np.array([3., 0.]), np.zeros((0,)), np.array([[4.]])]
    norm, out = ot.clip(grads, 1.0, scale=2.0, eps=0.0)
    assert norm == 10.0 and np.allclose(np.sqrt(sum((o * o).sum() for o in out)), 1.0)
    norm, out = ot.clip(grads, 100.0)
    assert norm == 5.0 and all((a == b).all() for a, b in zip(out, grads))
