"""Attention over shared positions where its tensor-core kernel has the most to do (CTAs with several parts of several
steps each) or gives up, and how near to their 64-bit definitions (serving_oracle.py) all its kernels come."""
import os
import sys

import numpy as np
import pytest

import tie_b200
from tie_b200 import ops

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import attention_precision as precision  # noqa: E402
import ops_oracle as paged  # noqa: E402
import serving_oracle as ref  # noqa: E402
from test_serving_ops_gpu import KINDS, Batch, _i, _f, _long, _np  # noqa: E402

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _parts(shared, tiles_heads, ctas):
    """Steps of the parts that each CTA has of groups of `shared` positions with that many items each: a line of
    items, a place for each step of 64 positions and one before them, in equal stretches."""
    line = [(n - 1) // 64 + 2 for n in shared for _ in range(tiles_heads)]
    share = -(-sum(line) // ctas)
    out, x = [[] for _ in range(ctas)], 0
    for places in line:
        for c in range(x // share, (x + places - 1) // share + 1):
            lo, hi = max(x, c * share) - x, min(x + places, (c + 1) * share) - x
            if hi - 1 > max(lo - 1, 0):
                out[c].append(hi - 1 - max(lo - 1, 0))
        x += places
    return out


def _some(b, chosen):
    """The definition's rows of the chosen sequences (new tokens: one each), and how far fp32 may be from them."""
    rows = b.start[chosen]
    starts = np.searchsorted(chosen, b.groups)
    o, vmax, smax = ref.attention(b.q[rows], b.kn, b.vn, b.table[chosen], np.arange(len(chosen) + 1), b.ctx[chosen], b.heads,
                                  b.scale, np.zeros((len(chosen), b.q.shape[1])), 1, b.ksn, b.vsn, prefix_table=b.ptable,
                                  prefix_lens=b.shared, group_start=starts)
    return rows, o, paged.attention_bound(vmax, smax, int(b.shared.max() + b.ctx.max()) + 1)


@pytest.mark.parametrize("kind", KINDS)
def test_ctas_with_several_parts_of_several_steps(kind):
    """32 prompts of a few hundred positions with 128 answers each: some answers of each are as the definition has them,
    all of them the same whenever they are computed."""
    rng = np.random.default_rng(31)
    n, groups, heads, kv_heads = 4096, 32, 12, 4
    shared = rng.integers(270, 400, groups)
    ctas = 2 * torch.cuda.get_device_properties(0).multi_processor_count
    many = [p for p in _parts(shared, n // groups * (heads // kv_heads) // 128 * kv_heads, ctas) if sum(m >= 2 for m in p) >= 2]
    assert len(many) > ctas // 2
    b = Batch(4, rng.integers(0, 9, n).tolist(), [1] * n, heads, kv_heads, kind, tuple(range(0, n + 1, n // groups)), tuple(shared))
    assert b.rows * heads * b.ptable.shape[1] * 16 >= 8_000_000          # the tensor-core kernel's, over every format
    first = b.call()
    got = _np(first).astype(np.float64)
    chosen = np.sort(np.concatenate([np.arange(groups) * (n // groups) + at for at in (0, 77)]))
    rows, o, bound = _some(b, chosen)
    assert (np.abs(got[rows] - o) <= bound).all()
    for _ in range(6):
        assert torch.equal(b.call(), first)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("held", [0x00, 0x3f, 0x7f, 0xff])
def test_a_wait_that_runs_out(kind, held):
    """Whatever the workspace held: rows that were not finished are NaN as a whole head, the others are right, the status
    says so, and the next call is as if nothing had been."""
    rng = np.random.default_rng(2)
    n, groups, heads = 4096, 32, 12
    b = _long(2, rng.integers(0, 9, n).tolist(), [1] * n, heads, 4, kind, tuple(range(0, n + 1, n // groups)),
              tuple(rng.integers(20, 190, groups)))
    rows, o, bound = _some(b, np.sort(rng.choice(n, 150, replace=False)))
    want = b.call()
    out, ws = torch.full_like(want, -3.0), torch.empty(ops.attention_shared_workspace(b.rows, b.heads), dtype=torch.uint8, device="cuda")
    ws.fill_(held)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def call():
        ops.attention_shared(_f(b.q), b.k, b.v, _i(b.table), _i(b.start), _i(b.ctx), 1, out, ws, k_scales=b.ks, v_scales=b.vs,
                             prefix_table=_i(b.ptable), prefix_lens=_i(b.shared), group_start=_i(b.groups), status=status)

    ops.attention_shared_wait_drill(5_000_000)
    call()
    assert status.item() == tie_b200.MODEL_STATUS.index("MODEL_ERR_DEVICE")
    got = _np(out).reshape(n, heads, 64)
    lost = np.isnan(got)
    assert np.array_equal(lost.any(-1), lost.all(-1)) and lost.any() and not lost.all()
    kept = ~lost.any(-1)
    assert np.array_equal(got[kept], _np(want).reshape(got.shape)[kept])
    kept = kept[rows]
    assert kept.any() and not kept.all()
    assert (np.abs(got[rows] - o.reshape(-1, heads, 64)) <= bound.reshape(-1, heads, 64))[kept].all()
    status.zero_()
    call()
    assert status.item() == 0 and torch.equal(out, want)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv_heads", [(3, 3), (8, 2), (16, 1)])
@pytest.mark.parametrize("ctx,new,groups,shared", [
    ([15], [1], (), ()), ([700], [1], (), ()), ([3000, 40, 333], [1, 1, 1], (), ()), ([500, 90], [9, 40], (), ()),
    ([20, 100, 3, 60], [1, 2, 1, 5], (0, 4), (900,)), ([30] * 24, [1] * 24, (0, 10, 24), (200, 77)),
])
def test_rows_are_near_the_definition(kind, heads, kv_heads, ctx, new, groups, shared):
    b = Batch(41, ctx, new, heads, kv_heads, kind, groups, shared)
    got, want = _np(b.call()), b.want()[0]
    shape = (b.rows * heads, 64)
    assert precision.near(got.reshape(shape), want.reshape(shape)), precision.off(got.reshape(shape), want.reshape(shape))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,new,heads,kv_heads,groups,shared", [
    (130, 1, 2, 2, (0, 130), (70,)), (64, 2, 8, 2, (0, 64), (1000,)), (100, 1, 12, 1, (0, 40, 100), (333, 2000)),
])
def test_rows_of_long_prefixes_are_near_the_definition(kind, n, new, heads, kv_heads, groups, shared):
    b = _long(43, np.random.default_rng(n).integers(0, 50, n).tolist(), [new] * n, heads, kv_heads, kind, groups, shared)
    got, want = _np(b.call()), b.want()[0]
    shape = (b.rows * heads, 64)
    assert precision.near(got.reshape(shape), want.reshape(shape)), precision.off(got.reshape(shape), want.reshape(shape))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv_heads,new", [(1024, 1024, 1), (8192, 1024, 1), (1024, 1024, 5)])
def test_as_many_heads_as_there_may_be(kind, heads, kv_heads, new):
    """One team of warps, or not even a second one, on the GPU."""
    b = Batch(47, [20, 3], [new, 1], heads, kv_heads, kind, (0, 2), (18,))
    b.check()


@pytest.mark.parametrize("kind", KINDS)
def test_long_prefixes_of_many_heads(kind):
    b = _long(49, [2] * 64, [1] * 64, 256, 256, kind, (0, 64), (130,))
    got = _np(b.call()).astype(np.float64)
    rows, o, bound = _some(b, np.array([0, 33, 63]))
    assert (np.abs(got[rows] - o) <= bound).all()


@pytest.mark.parametrize("kind", KINDS)
def test_as_many_groups_as_sequences_and_any_bound_of_new_tokens(kind):
    """4096 groups of a sequence each; max_new is a bound, however far off."""
    rng = np.random.default_rng(51)
    n = 4096
    b = Batch(51, rng.integers(0, 9, n).tolist(), rng.integers(0, 2, n).tolist(), 1, 1, kind, tuple(range(n + 1)),
              tuple(rng.integers(1, 40, n).tolist()))
    b.check()
    b.max_new = 2 ** 31 - 1
    b.check()
