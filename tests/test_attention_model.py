"""The 2-norm bar of attention over the INT8 cache, on the CPU: a model of the kernel's arithmetic keeps it, and
models that lose a plane of digits, or scale the weights by keys that a row does not see, do not."""
import numpy as np
import pytest

import attention_model as A

SIZES = [(1, 128), (5, 64), (128, 128), (129, 64), (545, 128), (3001, 128)]


def shares(kind, n, hd, hide=0, **kw):
    """Error over bar for four rows; the last `hide` keys are not seen."""
    r = []
    for s in range(4):
        h = A.history(np.random.default_rng(1000 * s + n + hd), kind, n, hd)
        see = np.arange(n) < n - hide
        o, bar = A.exact(*h, hd ** -0.5, see)
        r.append(np.linalg.norm(A.model(*h, hd ** -0.5, see, **kw) - o) / bar)
    return np.array(r)


@pytest.mark.parametrize("n,hd", SIZES)
@pytest.mark.parametrize("kind", ["plain", "peaked", "sink0", "sink1", "sink2", "sink6", "last3", "outlier2",
                                  "outlier3"])
def test_the_arithmetic_keeps_the_bar(kind, n, hd):
    assert (shares(kind, n, hd) < 1).all()


@pytest.mark.parametrize("n,hd", SIZES[1:])
@pytest.mark.parametrize("lose", ["q", "w"])
def test_a_lost_plane_of_digits_does_not(lose, n, hd):
    assert (shares("plain", n, hd, lose=lose) > 1).all()


@pytest.mark.parametrize("n,hd", [(5, 64), (128, 128), (545, 128), (3001, 128)])  # the hidden key shares a tile
@pytest.mark.parametrize("kind", ["last3", "last6", "last9"])
def test_hidden_keys_do_not_count(kind, n, hd):
    assert (shares(kind, n, hd, hide=1) < 1).all()
    assert (shares(kind, n, hd, hide=1, per_row=False) > 1).any()


@pytest.mark.parametrize("n,hd", SIZES[2:])
@pytest.mark.parametrize("kind", ["sink2", "sink6", "outlier3"])
def test_weight_and_value_scale_of_different_keys(kind, n, hd):
    """The largest weight and the largest value scale, each for itself, are no scale for their product."""
    assert (shares(kind, n, hd, per_row=False) > 1).any()


def test_nothing_seen_is_zero():
    h = A.history(np.random.default_rng(1), "plain", 130, 64)
    see = np.zeros(130, bool)
    o, bar = A.exact(*h, 0.125, see)
    assert bar == 0 and not o.any() and not A.model(*h, 0.125, see).any()
