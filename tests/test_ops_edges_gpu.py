"""The operators over the paged cache at the edges of the number range and of their arguments, on the GPU."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
torch = pytest.importorskip("torch")
import ops_oracle as ref  # noqa: E402
from test_ops_gpu import KV, _attend, _batch, _check_plan, _i, _workspace  # noqa: E402
from tie_b200 import ops  # noqa: E402

pytestmark = pytest.mark.gpu
PAGE, D = 16, 64


def _positions(b, s):
    """Pages and rows of sequence s's positions, cached and new."""
    pos = np.arange(b["ctx"][s] + b["start"][s + 1] - b["start"][s])
    return torch.from_numpy(b["table"][s][pos // PAGE]).cuda(), torch.from_numpy(pos % PAGE).cuda()


# ------------------------------------------------------------------ values of very different sizes

# exponents of the value rows by position (None: a row of zeros)
SIZES = {
    "zeros, then large": lambda pos, n: np.where(pos < n // 2, np.nan, 70),
    "large, then zeros": lambda pos, n: np.where(pos < n // 2, 70, np.nan),
    "tiny, then huge": lambda pos, n: np.where(pos < n // 2, -60, 100),
    "huge, then tiny": lambda pos, n: np.where(pos < n // 2, 100, -60),
    "ones and huge by pages": lambda pos, n: np.where(pos // PAGE % 2, 100, 0),
    "zeros and huge by rows": lambda pos, n: np.where(pos % 2, 100, np.nan),
    "zeros and huge by steps": lambda pos, n: np.where(pos // 128 % 2, 100, np.nan),
    "huge at last": lambda pos, n: np.where(pos < n - 5, np.nan, 100),
    "rising": lambda pos, n: -100 + 200 * pos // n,
    "falling": lambda pos, n: 100 - 200 * pos // n,
}


@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("n_seq,kv_heads,group,ctx,new", [
    (1, 1, 1, 700, 1), (1, 1, 1, 0, 150), (1, 1, 2, 700, 9), (1, 2, 1, 650, 150), (1, 1, 1, 3000, 40), (80, 4, 1, 300, 12)])
def test_attention_counts_keys_whatever_their_values(kv, sizes, n_seq, kv_heads, group, ctx, new):
    """A key's weight does not depend on how large its value is beside the others': the row sum keeps keys whose
    values are zero or tiny when others' are huge. The bound is attention_bound's, in units of the largest value,
    and 2^-106 for values below 2^-67, which are multiplied by 2^81 and not more: a second fp16 term of
    subnormal size is rounded by at most 2^-25 then, 2^-106 of the value, and the weights of a row add up to 1."""
    b = _batch(np.random.default_rng(ctx + new), [ctx] * n_seq, [new] * n_seq, kv_heads * group, kv_heads, kv)
    for s in range(n_seq):
        page, row = _positions(b, s)
        e = SIZES[sizes](np.arange(ctx + new), ctx + new)
        size = torch.from_numpy(np.where(np.isnan(e), 0.0, np.exp2(np.nan_to_num(e)))).cuda()[:, None]
        b["v"][page, row] = (b["v"][page, row].double() * size).to(kv)
    status = _i([0])
    got = _attend(b, status=status).cpu().numpy().astype(np.float64)
    want, vmax, smax = ref.attention(b["q"].cpu().numpy().astype(np.float64), b["k"].cpu().double().numpy(),
                                     b["v"].cpu().double().numpy(), b["table"], b["start"], b["ctx"], kv_heads * group,
                                     kv_heads, 0.125, np.zeros(got.shape))
    assert int(status[0]) == 0
    bad = ~(np.abs(got - want) <= ref.attention_bound(vmax, smax, ctx + new) + 2.0 ** -106)
    assert not bad.any(), (bad.sum(), np.argwhere(bad)[:4], got[bad][:4], want[bad][:4])


@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("n_seq,kv_heads,ctx,new", [
    (1, 1, 0, 1), (1, 1, 900, 1), (1, 12, 1900, 2), (1, 1, 20011, 1), (1, 1, 20011, 4), (160, 2, 300, 1), (1, 1, 700, 9),
    (80, 4, 300, 12), (1, 1, 5000, 40)])
def test_attention_of_the_largest_values_is_finite(kv, n_seq, kv_heads, ctx, new):
    """The mean of finite values is finite, also where their sum is not."""
    b = _batch(np.random.default_rng(ctx), [ctx] * n_seq, [new] * n_seq, kv_heads, kv_heads, kv)
    b["v"].copy_((b["v"].double().abs().clamp(max=1.0) * 0.5 + 0.4) * 2.0 ** 127)       # 0.4 to 0.9 of 2^127
    got = _attend(b).cpu().numpy().astype(np.float64)
    want, vmax, smax = ref.attention(b["q"].cpu().numpy().astype(np.float64), b["k"].cpu().double().numpy(),
                                     b["v"].cpu().double().numpy(), b["table"], b["start"], b["ctx"], kv_heads, kv_heads,
                                     0.125, np.zeros(got.shape))
    assert (np.abs(got - want) <= ref.attention_bound(vmax, smax, ctx + new)).all()


# ------------------------------------------------------------------ values that are not finite

# positions that score far below the others
LOW = {
    "one position": lambda pos, n: pos == n // 2,
    "one warp's pages": lambda pos, n: pos // PAGE % 8 == 3,
    "one CTA's pages": lambda pos, n: pos // 128 % 8 == 1,
    "the first half": lambda pos, n: pos < n // 2,
    "the second half": lambda pos, n: (pos >= n // 2) & (pos < n - 60),
}


@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("odd", [float("inf"), float("nan")])
@pytest.mark.parametrize("low", LOW)
@pytest.mark.parametrize("n_seq,kv_heads,ctx,new", [
    (1, 1, 240, 1), (1, 1, 900, 1), (1, 12, 1900, 2), (1, 1, 20011, 1), (1, 1, 20011, 4), (160, 2, 300, 1), (1, 1, 700, 9),
    (1, 2, 300, 60), (80, 4, 300, 12), (1, 1, 5000, 40)])
def test_attention_values_that_are_not_finite_reach_the_rows_that_see_them(kv, odd, low, n_seq, kv_heads, ctx, new):
    """However small its probability, and whoever read it (the maximum's warp, CTA or part, or another): a value
    that is not finite makes its dimension of every row that sees it not finite, and nothing else."""
    n = ctx + new
    b = _batch(np.random.default_rng(ctx), [ctx] * n_seq, [new] * n_seq, kv_heads, kv_heads, kv)
    b["q"].mul_(0.01)
    b["q"][:, ::D] = 1.0
    b["k"][..., ::D] = 0.0
    lows = LOW[low](np.arange(n), n)
    at = int(np.flatnonzero(lows)[lows.sum() // 2])
    for s in range(n_seq):
        page, row = _positions(b, s)
        where = torch.from_numpy(lows).cuda()
        b["k"][page[where], row[where], ::D] = -400.0        # the others score about 0
        b["v"][page[at], row[at], 5::D] = odd
    got = _attend(b, scale=1.0).view(n_seq, new, kv_heads, D)
    sees = torch.arange(new, device="cuda") + ctx >= at
    assert not bool(got[:, sees][..., 5].isfinite().any())
    got[:, sees, :, 5] = 0.0
    assert bool(got.isfinite().all())


# ------------------------------------------------------------------ nothing to do

@pytest.mark.parametrize("kv", KV)
def test_steps_without_rows(kv):
    """Tensors without elements: no rows to store or to attend with, no free page."""
    b = _batch(np.random.default_rng(1), [20, 3], [0, 0], 4, 2, kv)
    none = torch.empty(0, 2 * D, device="cuda")
    before = b["k"].clone()
    ops.kv_store(none, none.clone(), torch.empty(0, dtype=torch.int32, device="cuda"), b["k"], b["v"])
    assert torch.equal(b["k"], before)
    q = torch.empty(0, 4 * D, device="cuda")
    for max_new in (0, 5):
        ops.attention_paged(q, b["k"], b["v"], _i(b["table"]), _i([0, 0, 0]), _i(b["ctx"]), max_new, q.clone(), _workspace())
    torch.cuda.synchronize()


@pytest.mark.parametrize("new,status", [([1, 2], ref.OK), ([1, 13], ref.OK), ([1, 14], ref.CAPACITY), ([0, 0], ref.OK)])
def test_plan_with_an_empty_free_list(new, status):
    """Rows that fit the pages there are; or, without a page to give, nothing."""
    table = np.array([[4, 7], [2, 9]])
    got = _check_plan([20, 3], new, table, 10, 16, free=np.empty(0, np.int64), n_free=0)
    assert got[-1] == status


# ------------------------------------------------------------------ the same slot twice

@pytest.mark.parametrize("kv", KV)
def test_store_of_two_rows_with_one_slot(kv):
    """Every element is one of the rows', in the keys and in the values, and no other slot is touched."""
    rows, w, n_pages = 4000, 3 * D, 5
    g = torch.Generator(device="cuda").manual_seed(7)
    k, v = torch.randn(2, rows, w, generator=g, device="cuda")
    slots = torch.randint(0, n_pages * PAGE // 2, (rows,), generator=g, device="cuda").to(torch.int32) * 2
    pages = [torch.full((n_pages, PAGE, w), 9.0, device="cuda", dtype=kv) for _ in range(2)]
    ops.kv_store(k, v, slots, *pages)
    for p, x in zip(pages, (k, v)):
        flat = p.view(-1, w)
        for slot in range(n_pages * PAGE):
            mine = x[slots == slot].to(kv)
            if slot % 2:
                assert bool((flat[slot] == 9.0).all())
            else:
                assert len(mine) > 1 and bool((mine == flat[slot]).any(0).all())


# ------------------------------------------------------------------ very long contexts

def test_attention_of_tiles_that_take_longer_than_a_wait():
    """A tile of 72 million positions takes its CTA over 2 s, and more tiles than the CTA describes in advance stand
    behind it. The positions are those of 64 pages again and again, so the exact result is a weighted mean over these.

    A row sum is added up over half a million steps and the running output over a quarter of them, each addition
    off by 2^-24 of the sum at worst."""
    n, new, small = 72 << 20, 148 * 256, 20
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = torch.randn(2, 64, PAGE, D, generator=g, device="cuda").to(torch.bfloat16)
    width = ref.pages_of(n + new)
    table = (torch.arange(width, dtype=torch.int32, device="cuda") % 64).repeat(1 + small, 1)
    rows = new + 9 * small
    q = torch.randn(rows, D, generator=g, device="cuda")
    start = _i([0] + [new + 9 * s for s in range(small + 1)])
    out, status = torch.full((rows, D), 7.0, device="cuda"), _i([0])
    ops.attention_paged(q, k, v, table, start, _i([n] + [0] * small), new, out, _workspace(), status=status)
    torch.cuda.synchronize()
    assert int(status[0]) == 0
    kd, vd = k.double().view(-1, D), v.double().view(-1, D)
    pick = torch.cat([torch.arange(0, new, 997, device="cuda"), torch.arange(new, rows, device="cuda")])
    seen = torch.where(pick < new, n + pick + 1, (pick - new) % 9 + 1)[:, None]
    count = (seen // len(kd) + (torch.arange(len(kd), device="cuda") < seen % len(kd))).double()
    p = torch.exp(0.125 * q[pick].double() @ kd.T) * count
    want = p / p.sum(1, keepdim=True) @ vd
    bound = 2 * (seen / 128 + 100 + 96) * 2.0 ** -24 * vd.abs().max()
    assert bool(((out[pick].double() - want).abs() <= bound).all())


# ------------------------------------------------------------------ queries and keys of very different sizes

@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("power", [112, 60, -60, -105])
@pytest.mark.parametrize("ctx,new", [(70, 1), (70, 9), (0, 150), (300, 40)])
def test_attention_of_queries_and_keys_whose_products_are_ordinary(kv, power, ctx, new):
    """Queries of 2^power and keys of 2^-power: their products are as ever, and so are the results."""
    b = _batch(np.random.default_rng(new), [ctx], [new], 4, 2, kv)
    b["q"].mul_(2.0 ** power)
    b["k"].copy_((b["k"].double() * 2.0 ** -power).to(kv))
    status = _i([0])
    got = _attend(b, status=status).cpu().numpy().astype(np.float64)
    want, vmax, smax = ref.attention(b["q"].cpu().numpy().astype(np.float64), b["k"].cpu().double().numpy(),
                                     b["v"].cpu().double().numpy(), b["table"], b["start"], b["ctx"], 4, 2, 0.125,
                                     np.zeros(got.shape))
    assert int(status[0]) == 0 and (np.abs(got - want) <= ref.attention_bound(vmax, smax, ctx + new)).all()


# ------------------------------------------------------------------ streams of a tile that end far apart

@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("rows", [136, 160, 200, 256, 300])
@pytest.mark.parametrize("odd", [2.0 ** 100, float("inf")])
def test_attention_of_tiles_whose_halves_end_far_apart(kv, rows, odd):
    """Tiles of two halves, of which the second has a long way out (its rows see a value that their row sums, or their
    results, have to be completed for), each in front of tiles of one short step: the others' O is left in time, and
    no signal for a tile comes before the last one for the tile before it."""
    rng = np.random.default_rng(rows)
    n, kv_heads = 24, 6
    ctx = [v for _ in range(n) for v in (int(rng.integers(300, 700)), int(rng.integers(0, 90)), 10)]
    new = [v for _ in range(n) for v in (rows, int(rng.integers(9, 30)), 9)]
    b = _batch(rng, ctx, new, kv_heads, kv_heads, kv)
    late = min(rows - 1, 130)
    for s in range(0, 3 * n, 3):
        page, row = _positions(b, s)
        b["v"][page[ctx[s] + late], row[ctx[s] + late]] = odd
    outs = [_attend(b) for _ in range(4)]
    assert all(torch.equal(torch.nan_to_num(o), torch.nan_to_num(outs[0])) for o in outs)
    got, start = outs[0].cpu().numpy().astype(np.float64), b["start"]
    for s in (0, 1, 2, 33, 34, 35):
        lo, hi = start[s], start[s + 1]
        one = [x.cpu().double().numpy() for x in (b["q"][lo:hi], b["k"], b["v"])]
        with np.errstate(all="ignore"):
            want, vmax, smax = ref.attention(*one, b["table"][s:s + 1], [0, hi - lo], [ctx[s]], kv_heads, kv_heads, 0.125,
                                             np.zeros((hi - lo, kv_heads * D)))
        sees = s % 3 == 0 and not np.isfinite(odd)
        live = np.arange(hi - lo) < (late if sees else hi - lo)
        near = np.abs(got[lo:hi][live] - want[live]) <= ref.attention_bound(vmax, smax, ctx[s] + new[s])[live]
        assert near.all()
        assert not np.isfinite(got[lo:hi][~live]).any()
