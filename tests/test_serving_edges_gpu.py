"""Products with 4-bit weights at the ends of fp32 and of the sizes that one kernel takes, against their definition in
64 bits; rows that are alone."""
import os
import sys

import numpy as np
import pytest

from tie_b200 import ops

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import serving_oracle as ref  # noqa: E402
from test_serving_ops_gpu import _f, _np  # noqa: E402

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24


def _bound(x, w, group):
    """How far a product may be from x w^T.

    An element is an integer of a unit that is 2^-29 of the largest of its 128 columns at most (and 2^-127 at least),
    rounded to the nearest: off by half of that, and by nothing where it is zero or, having 24 bits, within 2^-6 of the
    largest. Sums of digits over a group are exact; joining them rounds five times, a group's product with its scale and
    its addition once, 16 warps' parts of a row and the digits of one or two rows add 16 and 4 more. Nothing below 2^-149
    is held of an fp32 sum."""
    k = x.shape[1]
    wide = np.zeros((len(x), -(-k // 128) * 128))
    wide[:, :k] = np.abs(x)
    top = np.repeat(wide.reshape(len(x), -1, 128).max(-1), 128, 1)[:, :k]
    near = (x == 0) | ((np.abs(x) >= top * 2.0 ** -6) & (top >= 2.0 ** -97))
    held = np.where(near, 0.0, np.maximum(top * 2.0 ** -30, 2.0 ** -128))
    adds = -(-k // group) + 5 + 16 + 4
    return (np.abs(x) @ np.abs(w).T) * adds * EPS + held @ np.abs(w).T + adds * 2.0 ** -149


def _weights(rng, n, k, group, scale, zero=()):
    """packed and scales on the device, and the weights in 64 bits; the columns `zero` have level 0."""
    q = rng.integers(-7, 8, (n, k))
    q[:, list(zero)] = 0
    s = ref.bf16((scale * (1.0 + rng.random((n, -(-k // group))))).astype(np.float32))
    return torch.tensor(ref.pack_q4(q), device="cuda"), torch.tensor(s, device="cuda").to(torch.bfloat16), ref.weights(q, s, group)


def _product(x, packed, scales, group):
    y = torch.empty(len(x), packed.shape[0], device="cuda")
    ops.matvec_q4(_f(x.astype(np.float32)), packed, scales, group, y)
    return _np(y).astype(np.float64)


GROUPS = pytest.mark.parametrize("group", [32, 64, 128])
ROWS = pytest.mark.parametrize("rows", [1, 2, 3, 8])


@GROUPS
@ROWS
@pytest.mark.parametrize("size,scale", [(1e-30, 1.375 * 2.0 ** -20), (1e-36, 1e-3), (1e-20, 1e-22), (1e-37, 1e30), (1e-38, 2.0 ** 120),
                                        (1.0, 2.0 ** -125), (1e30, 2.0 ** -130), (1e-25, 2.0 ** -60)])
def test_small_products_keep_their_bits(group, rows, size, scale):
    """Activations and scales whose product with the smallest unit is no normal number, though the result may be."""
    rng = np.random.default_rng(rows)
    packed, scales, w = _weights(rng, 37, 256, group, scale)
    x = (size * rng.standard_normal((rows, 256))).astype(np.float32).astype(np.float64)
    want = x @ w.T
    assert (np.abs(_product(x, packed, scales, group) - want) <= _bound(x, w, group)).all()


@GROUPS
@ROWS
@pytest.mark.parametrize("scale", [64.0, 2.0 ** 40, 2.0 ** 100, 2.0 ** 126])
def test_a_large_activation_that_meets_nothing(group, rows, scale):
    """3e38 in a column whose levels are 0: the result is the other columns', whatever the scales are."""
    rng = np.random.default_rng(rows)
    packed, scales, w = _weights(rng, 37, 256, group, scale, zero=[5])
    x = np.zeros((rows, 256))
    x[:, 5] = np.float32(3e38)
    x[:, 128:] = (rng.standard_normal((rows, 128)) * min(1.0, 2.0 ** 100 / scale)).astype(np.float32)
    want = x @ w.T
    got = _product(x, packed, scales, group)
    assert np.isfinite(got).all() and (np.abs(got - want) <= _bound(x, w, group)).all()


@GROUPS
@ROWS
def test_large_activations(group, rows):
    """Sums of levels times activations beyond fp32, with scales that bring them back."""
    rng = np.random.default_rng(rows)
    packed, scales, w = _weights(rng, 37, 256, group, 1e-4)
    x = (1e38 * (2.0 * rng.random((rows, 256)) + 1.0)).astype(np.float32).astype(np.float64)
    want = x @ w.T
    assert (np.abs(_product(x, packed, scales, group) - want) <= _bound(x, w, group)).all()


@GROUPS
@pytest.mark.parametrize("rows", [2, 3])
def test_a_large_row_leaves_the_rows_beside_it(group, rows):
    rng = np.random.default_rng(rows)
    packed, scales, w = _weights(rng, 37, 256, group, 2.0 ** -20)
    x = 1e-30 * rng.standard_normal((rows, 256))
    before = _product(x, packed, scales, group)
    x[1] = 3e38
    got = _product(x, packed, scales, group)
    keep = np.arange(rows) != 1
    assert np.array_equal(got[keep], before[keep])


@ROWS
def test_what_is_held_of_small_elements(rows):
    """Beside a largest element of 1, others are held to 2^-30: half of a unit of 2^-29."""
    rng = np.random.default_rng(rows)
    packed, scales, w = _weights(rng, 37, 128, 128, 0.01)
    x = np.zeros((rows, 128))
    x[:, 3] = 1.0
    x[:, 70] = [np.float32(2.0 ** -30 * f) for f in (0.999, 1.001, 2.9, 0.5, 1.5, 0.999, 4.1, 1000.5)][:rows]
    want = x @ w.T
    # (the sum of two products is rounded to 2^-24 of it, which hides the second: so without the first as well)
    off = np.abs(_product(x, packed, scales, 128) - want)
    assert (off <= _bound(x, w, 128)).all()
    held = np.rint(x[:, 70] * 2.0 ** 29) * 2.0 ** -29
    q = np.zeros((37, 128), np.int64)
    q[:, 70] = 1
    packed = torch.tensor(ref.pack_q4(q), device="cuda")
    one = torch.ones(37, 1, dtype=torch.bfloat16, device="cuda")
    got = _product(x, packed, one, 128)
    assert np.array_equal(got, np.repeat(held[:, None], 37, 1)) and (np.abs(got[:, 0] - x[:, 70]) <= 2.0 ** -30).all()


@pytest.mark.parametrize("group,k", [(32, 6400), (32, 6401), (64, 6784), (64, 6785), (128, 6912), (128, 6913)])
def test_the_longest_rows_that_are_taken_by_eight(group, k):
    """The length where eight rows' digits fill shared memory, and one column more: two rows at a time."""
    rng = np.random.default_rng(k)
    packed, scales, w = _weights(rng, 37, k, group, 0.01)
    x = rng.standard_normal((8, k)).astype(np.float32).astype(np.float64)
    got = _product(x, packed, scales, group)
    assert (np.abs(got - x @ w.T) <= _bound(x, w, group)).all()
    # by two, a row does not depend on the rows beside it, nor on how many there are
    for lo in (0, 6):
        alone = _product(x[lo:lo + 2], packed, scales, group)
        assert np.array_equal(alone, got[lo:lo + 2]) == (k % 128 == 1)


@pytest.mark.parametrize("kind", ["f32", "q8"])
def test_a_row_alone_may_have_any_stride(kind):
    """There is no next row, so strides that two tensors do not share, or that are not whole groups of 4, mean nothing."""
    rng = np.random.default_rng(1)
    w = 2 * 64
    k, v, q = (rng.standard_normal((1, w)).astype(np.float32) for _ in range(3))

    def wide(x, extra):
        t = torch.zeros(1, w + extra, device="cuda")
        if x is not None:
            t[:, :w] = _f(x)
        return t[:, :w]

    def i(*x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    dtype = torch.int8 if kind == "q8" else torch.float32
    pages = [torch.zeros(3, 16, w, dtype=dtype, device="cuda") for _ in range(2)]
    scales = [torch.zeros(3, 2, 16, device="cuda") for _ in range(2)] if kind == "q8" else [None, None]
    if kind == "q8":
        ops.kv_store_q8(wide(k, 64), wide(v, 3), i(17), *pages, *scales)
    else:
        ops.kv_store(wide(k, 64), wide(v, 3), i(17), *pages)
    out = [wide(None, 7), wide(None, 128)]
    ops.kv_load(i(17), *pages, *out, *scales)
    for x, o in zip((k, v), out):
        # (levels are within half of a step of 1 / 127 of the largest)
        assert np.abs(_np(o) - x).max() <= (np.abs(x).max() / 253 if kind == "q8" else 0.0)
    # a sequence of one position: the row of values
    got = wide(None, 5)
    ws = torch.empty(ops.attention_shared_workspace(1, 2), dtype=torch.uint8, device="cuda")
    table, start, ctx = i(1).view(1, 1), i(0, 1), i(0)
    ops.kv_store_q8(wide(k, 1), wide(v, 2), i(16), *pages, *scales) if kind == "q8" else ops.kv_store(wide(k, 1), wide(v, 2), i(16), *pages)
    ops.attention_shared(wide(q, 3), *pages, table, start, ctx, 1, got, ws, *scales)
    assert np.abs(_np(got) - _np(out[1])).max() <= 4 * EPS * np.abs(v).max()
