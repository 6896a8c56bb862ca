"""tests/routing_gradient.py, the oracle of gradients whose definition's differences cancel, against that definition in 400
decimal digits, and against tests/routing.py where float64 is enough."""
from decimal import Decimal, getcontext

import numpy as np
import pytest

from tests import routing as Q
from tests import routing_gradient as G


def definition(x, scoring, ids, dw, renorm):
    """One token's gradient: the weights' Jacobian, term by term."""
    getcontext().prec = 400
    x = [Decimal(float(v)) for v in x]
    if scoring == "sigmoid":
        p = [1 / (1 + (-v).exp()) for v in x]
    else:
        e = [(v - max(x)).exp() for v in x]
        p = [v / sum(e) for v in e]
    total = sum(p[e] for e in ids) if renorm else Decimal(1)
    dp = [Decimal(0)] * len(x)
    for s, e in enumerate(ids):  # w_s = p_e / total
        d = Decimal(float(dw[s]))
        dp[e] += d / total
        if renorm:
            for o in ids:
                dp[o] -= d * p[e] / total ** 2
    if scoring == "sigmoid":
        return [float(a * b * (1 - b)) for a, b in zip(dp, p)]
    inner = sum(a * b for a, b in zip(dp, p))
    return [float(b * (a - inner)) for a, b in zip(dp, p)]


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [0, 1])
@pytest.mark.parametrize("level,ahead", [(0.0, 0.0), (0.0, 12.0), (0.0, 40.0), (0.0, 100.0), (-90.0, 0.0), (-300.0, 30.0), (60.0, 20.0)])
def test_against_the_definition(scoring, renorm, level, ahead):
    rng = np.random.default_rng(0)
    x = level + rng.standard_normal((3, 6))
    x[:, 2] += ahead
    ids = np.array([[2, 0, 4], [1, 2, 5], [0, 3, 0]], np.int32)  # the largest among them, not among them, one twice
    dw = rng.standard_normal((3, 3))
    got, size = G.grad(x, scoring, ids, dw, renorm)
    want = np.array([definition(x[t], scoring, ids[t], dw[t], renorm) for t in range(3)])
    # an exponential of a logarithm of up to 400 is off by 400 * 2^-53; some factors and terms
    assert (np.abs(got - want) <= 2.0 ** -40 * size + 1e-320).all()
    assert (np.abs(got) <= size * (1 + 2.0 ** -40)).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [0, 1])
def test_against_the_plain_oracle(scoring, renorm):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((20, 10))
    x[0], x[1, 2:] = -np.inf, -np.inf
    ids = rng.integers(-1, 11, (20, 4)).astype(np.int32)
    dw = rng.standard_normal((20, 4))
    want = Q.grad(x, scoring, ids, dw, renorm, 2.5)
    assert (np.abs(G.grad(x, scoring, ids, dw, renorm, 2.5)[0] - want) <= 1e-13).all()
