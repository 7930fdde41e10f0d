"""The operands and bounds by which the GPU tests tell whether a plane product
of an F32 product is missing, against a model with one left out."""
import numpy as np
import pytest
from nn_planes import TERMS, carried_by, planes, product


def test_planes_are_the_number():
    r = np.random.default_rng(1)
    x = (r.standard_normal(10000) * 2.0 ** r.integers(-60, 60, 10000)).astype(np.float32)
    assert np.array_equal(sum(p.astype(np.float64) for p in planes(x)), x.astype(np.float64))


@pytest.mark.parametrize("k", [64, 72, 264, 1000])
def test_a_missing_term_shows_norm_wise(k):
    r = np.random.default_rng(k)
    x, w = r.standard_normal((64, k)).astype(np.float32), r.standard_normal((k, 64)).astype(np.float32)
    want = x.astype(np.float64) @ w.astype(np.float64)
    off = lambda terms: np.linalg.norm(product(x, w, terms) - want) / np.linalg.norm(want)  # noqa: E731
    assert off(TERMS) <= 2e-7
    for t in TERMS:
        assert off([u for u in TERMS if u != t]) >= 4e-6


@pytest.mark.parametrize("term", TERMS)
def test_one_pair_carries_the_result(term):
    x, w = carried_by(term, 50, 203, 40, 2)
    want = x.astype(np.float64) @ w.astype(np.float64)
    assert want.min() >= 2.0**-16 and (np.abs(x).astype(np.float64).max() * np.abs(w).max()) <= 4
    # of the result's size: the pair alone gives it, all others nothing
    assert np.allclose(product(x, w, [term]), want, rtol=2.0**-6, atol=0)
    assert np.abs(product(x, w, [t for t in TERMS if t != term])).max() <= 2.0**-6 * want.max()
