"""The references of tests/block_ref.py, which the operators are tested against, on examples worked by hand."""
import numpy as np
import pytest

import block_examples as X
import block_ref as R

# 64-bit arithmetic on logits that are logarithms rounded to 64 bits
TOL = dict(rtol=1e-13, atol=1e-15)


@pytest.mark.parametrize("logits, K, rule, ids, w", X.ROUTE)
def test_route(logits, K, rule, ids, w):
    got = R.route([logits], K, **rule)
    assert got[0][0].tolist() == ids
    np.testing.assert_allclose(got[1][0], w, **TOL)


@pytest.mark.parametrize("x, rows, gate, rule, y, r", X.NORM)
def test_block_norm(x, rows, gate, rule, y, r):
    got = R.block_norm([x], None if rows is None else [rows], gate, eps=0.0, **rule)
    np.testing.assert_allclose(got[0][0], y, **TOL)
    np.testing.assert_allclose(got[1][0], x if r is None else r, **TOL)


@pytest.mark.parametrize("logits, u, rule, token, prob", X.SAMPLE)
def test_sample(logits, u, rule, token, prob):
    got = R.sample([logits], [u], **rule)
    assert got[0][0] == token
    np.testing.assert_allclose(got[1][0], prob, **TOL)
