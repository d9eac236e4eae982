"""The limits of attention_precision.py notice each product of terms, and each digit, that is left out."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import attention_precision as near  # noqa: E402

LENGTHS = [16, 100, 1000, 4000]


def _rows(n, kind, **kw):
    rng = np.random.default_rng(n)
    got, want = [], []
    for _ in range(12):
        q = (2.0 * rng.standard_normal(64)).astype(np.float32)
        if kind == "q8":
            k, v = (rng.integers(-127, 128, (n, 64)) for _ in range(2))
            ks, vs = ((0.2 + rng.random(n)).astype(np.float32).astype(np.float64) / 70 for _ in range(2))
            got.append(near.row_q8(q, k, ks, v, vs, 0.125, **kw))
            want.append(near.exact(q, k * ks[:, None], v * vs[:, None], 0.125))
            continue
        k, v = (rng.standard_normal((n, 64)).astype(np.float32) for _ in range(2))
        if kind == "bf16":
            k, v = (near.terms(x)[0].astype(np.float32) for x in (k, v))
        got.append(near.row(q, k, v, 0.125, **kw))
        want.append(near.exact(q, k, v, 0.125))
    return np.stack(got), np.stack(want)


@pytest.mark.parametrize("n", LENGTHS)
@pytest.mark.parametrize("kind", ["f32", "bf16", "q8"])
def test_all_products_are_near(kind, n):
    kw = {} if kind == "q8" else dict(scores=near.PRODUCTS[kind], values=near.PRODUCTS[kind])
    assert near.near(*_rows(n, kind, **kw)), near.off(*_rows(n, kind, **kw))


@pytest.mark.parametrize("n", LENGTHS)
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("which", ["scores", "values"])
def test_a_product_left_out_is_not(kind, n, which):
    for missing in near.PRODUCTS[kind][1:]:
        kw = dict(scores=near.PRODUCTS[kind], values=near.PRODUCTS[kind])
        kw[which] = [p for p in kw[which] if p != missing]
        assert not near.near(*_rows(n, kind, **kw)), (missing, near.off(*_rows(n, kind, **kw)))


@pytest.mark.parametrize("n", LENGTHS)
@pytest.mark.parametrize("bits", [dict(q_bits=16), dict(w_bits=15)])
def test_a_digit_left_out_is_not(n, bits):
    assert not near.near(*_rows(n, "q8", **bits)), near.off(*_rows(n, "q8", **bits))
