"""The operators over the paged cache on the GPU against their 64-bit definitions (ops_oracle.py)."""
import os
import sys

import numpy as np
import pytest

import tie_b200
from tie_b200 import ops

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import ops_oracle as ref  # noqa: E402

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
PAGE, D = 16, 64
I32 = torch.int32


def _i(v):
    return torch.tensor(np.asarray(v), dtype=I32, device="cuda")


def _out(n, dtype=I32, fill=-77):
    return torch.full((n,), fill, dtype=dtype, device="cuda")


# ------------------------------------------------------------------ page plan

def _plan(ctx, new, table, n_pages, max_rows, free=None, n_free=0, in_place=True):
    n = len(ctx)
    t = _i(table)
    o = dict(row_start=_out(n + 1), seq_of=_out(max_rows), pos_of=_out(max_rows), slot_of=_out(max_rows), status=_out(1))
    kw = {}
    if free is not None:
        nf = _i([n_free])
        kw = dict(free_pages=_i(free), n_free=nf, n_free_out=nf if in_place else _out(1))
    ops.page_plan(_i(ctx), _i(new), t, n_pages, **o, **kw)
    torch.cuda.synchronize()
    left = int(kw["n_free_out"][0]) if kw else 0
    return [t.cpu().numpy(), left] + [o[k].cpu().numpy() for k in ("row_start", "seq_of", "pos_of", "slot_of")] + [int(o["status"][0])]


def _check_plan(*a, **kw):
    got = _plan(*a, **kw)
    kw.pop("in_place", None)
    want = ref.plan(*a, **kw)
    for g, w in zip(got, want):
        assert np.array_equal(g, w)
    return got


def _pool_tables(rng, ctx, new, width, spare):
    have = [ref.pages_of(c) for c in ctx]
    need = sum(ref.pages_of(c + m) for c, m in zip(ctx, new)) - sum(have)
    n_pages = sum(have) + need + spare
    perm = rng.permutation(n_pages)
    table = np.full((len(ctx), width), n_pages, np.int64)
    at = 0
    for s, h in enumerate(have):
        table[s, :h] = perm[at:at + h]
        at += h
    return table, n_pages, perm[at:]


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("n_seq,ctx_max,new_max,pad", [
    (1, 0, 1, 0), (1, 15, 1, 0), (1, 16, 1, 3), (1, 100, 300, 0), (3, 40, 0, 2), (7, 64, 33, 5), (256, 1023, 1, 1),
    (1023, 200, 40, 100), (1025, 50, 3, 0), (4096, 30, 20, 9)])
def test_plan_matches_the_host_allocators_order(n_seq, ctx_max, new_max, pad, in_place):
    rng = np.random.default_rng(n_seq + ctx_max)
    ctx, new = rng.integers(0, ctx_max + 1, n_seq).tolist(), rng.integers(0, new_max + 1, n_seq).tolist()
    ctx[-1], new[0] = ctx_max, new_max
    width = max(max(ref.pages_of(c + m) for c, m in zip(ctx, new)), 1)
    table, n_pages, free = _pool_tables(rng, ctx, new, width, 3)
    rows = max(1, sum(new) + pad)
    got = _check_plan(ctx, new, table, n_pages, rows, free=free, n_free=len(free), in_place=in_place)
    assert got[-1] == ref.OK and got[1] == 3


def test_plan_without_a_free_list_reads_the_table():
    ctx, new = [5, 0, 31], [30, 2, 1]
    table = np.array([[3, 9, -1], [0, 1, 2], [7, 4, 99]])     # -1 and 99 are no pages of 10
    got = _check_plan(ctx, new, table, 10, 40)
    assert got[-1] == ref.OK and (got[5][:33] == -1).sum() == 3


@pytest.mark.parametrize("case", ["pages", "width", "rows", "negative", "n_free"])
def test_plan_assigns_nothing_when_it_cannot_assign_all(case):
    rng = np.random.default_rng(5)
    ctx, new = [20, 16, 3], [10, 40, 0]
    table, n_pages, free = _pool_tables(rng, ctx, new, 4, 0)
    rows, n_free = 60, len(free)
    if case == "pages":
        n_free -= 1
    if case == "width":
        new[1] = 49
    if case == "rows":
        rows = 49
    if case == "negative":
        new[2] = -1
    if case == "n_free":
        n_free = len(free) + 1
    got = _check_plan(ctx, new, table, n_pages, rows, free=free, n_free=n_free)
    assert got[-1] == (ref.ARG if case in ("negative", "n_free") else ref.CAPACITY)
    assert np.array_equal(got[0], table) and got[1] == n_free and not got[2].any()


def test_plan_of_lengths_beyond_32_bits_is_refused():
    big = 2 ** 31 - 1
    got = _check_plan([big, big, 0], [big, 1, 1], np.zeros((3, 2), int), 4, 8, free=[1, 2], n_free=2)
    assert got[-1] == ref.CAPACITY


# ------------------------------------------------------------------ row store

@pytest.mark.parametrize("kv", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,heads,ld_extra", [(1, 1, 0), (3, 2, 4), (257, 12, 12 * 64 * 2), (1000, 25, 0)])
def test_store_rounds_to_nearest_and_leaves_the_rest(kv, rows, heads, ld_extra):
    g = torch.Generator(device="cuda").manual_seed(rows)
    w, n_pages = heads * D, ref.pages_of(rows) + 3
    src = torch.randn(2, rows, w + ld_extra, generator=g, device="cuda")
    src[0, 0, :4] = torch.tensor([float("inf"), float("-inf"), float("nan"), -0.0])
    k, v = src[0, :, ld_extra:], src[1, :, ld_extra:]
    pages = [torch.randn(n_pages, PAGE, w, generator=g, device="cuda").to(kv) for _ in range(2)]
    want = [p.clone() for p in pages]
    slots = torch.randperm(n_pages * PAGE, generator=g, device="cuda")[:rows].to(I32)
    if rows > 3:
        slots[1], slots[2], slots[3] = -1, n_pages * PAGE, 2 ** 31 - 1     # nothing is stored
    ok = (slots >= 0) & (slots < n_pages * PAGE)
    for p, x in zip(want, (k, v)):
        p.view(-1, w)[slots[ok].long()] = x[ok].to(kv)
    ops.kv_store(k, v, slots, *pages)
    for p, x in zip(pages, want):
        bits = torch.int32 if kv == torch.float32 else torch.int16
        a, b = p.view(bits), x.view(bits)
        same = (a == b) | (p.isnan() & x.isnan())
        assert bool(same.all())


# ------------------------------------------------------------------ attention

def _batch(rng, ctx, new, heads, kv_heads, kv, extra_rows=0, ldq_extra=0, spare=2):
    counts = [ref.pages_of(c + m) for c, m in zip(ctx, new)]
    width, n_pages, w = max(max(counts), 1), sum(counts) + spare, kv_heads * D
    table = np.full((len(ctx), width), -1, np.int64)
    perm, at = rng.permutation(n_pages), 0
    for s, n in enumerate(counts):
        table[s, :n] = perm[at:at + n]
        at += n
    rows = sum(new) + extra_rows
    start = np.concatenate([[0], np.cumsum(new)])
    k, v = (rng.standard_normal((n_pages, PAGE, w)).astype(np.float32) for _ in range(2))
    q = (2 * rng.standard_normal((rows, heads * D + ldq_extra))).astype(np.float32)
    dev = lambda x: torch.from_numpy(x).cuda()  # noqa: E731
    return dict(ctx=ctx, start=start, table=table, heads=heads, kv_heads=kv_heads, q=dev(q)[:, :heads * D],
                k=dev(k).to(kv), v=dev(v).to(kv), max_new=max(new), rows=rows)


def _workspace():
    return torch.empty(ops.attention_paged_workspace(), dtype=torch.uint8, device="cuda")


def _attend(b, scale=None, out=None, workspace=None, max_new=None, status=None):
    out = torch.full((b["rows"], b["heads"] * D), 7.0, device="cuda") if out is None else out
    ops.attention_paged(b["q"], b["k"], b["v"], _i(b["table"]), _i(b["start"]), _i(b["ctx"]),
                        b["max_new"] if max_new is None else max_new, out, _workspace() if workspace is None else workspace,
                        scale=scale, status=status)
    return out


def _check_attention(b, scale=None, skip=()):
    status = _i([0])
    got = _attend(b, scale, status=status).cpu().numpy().astype(np.float64)
    start = np.array(b["start"])
    want, vmax, smax = ref.attention(b["q"].cpu().numpy().astype(np.float64), b["k"].cpu().double().numpy(),
                                     b["v"].cpu().double().numpy(), b["table"], start, b["ctx"], b["heads"], b["kv_heads"],
                                     0.125 if scale is None else scale, np.full(got.shape, 7.0))
    assert int(status[0]) == 0
    length = max(b["ctx"]) + b["max_new"]
    bound = ref.attention_bound(vmax, smax, length)
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], bound[bad][:5])
    live = vmax > 0
    # and in the whole: fp32 results, not results of fewer bits
    if live.any():
        assert np.linalg.norm((got - want)[live]) <= 2e-6 * np.linalg.norm(want[live]) * max(1.0, smax.max() / 16)
    return got


KV = [torch.float32, torch.bfloat16]


@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("heads,kv_heads", [(12, 12), (25, 25), (2, 1), (6, 2), (8, 1), (32, 2), (9, 1)])
@pytest.mark.parametrize("ctx,new", [
    ([0], [1]), ([15], [1]), ([16], [1]), ([300], [1]), ([4, 17, 0, 130], [1, 1, 1, 1]), ([250, 3], [2, 1])])
def test_attention_few_tokens(kv, heads, kv_heads, ctx, new):
    _check_attention(_batch(np.random.default_rng(len(ctx) + heads), ctx, new, heads, kv_heads, kv))


@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("heads,kv_heads", [(3, 3), (4, 2), (5, 1)])
@pytest.mark.parametrize("ctx,new", [
    ([0], [9]), ([0], [127]), ([0], [128]), ([1], [129]), ([200], [60]), ([127, 0, 640], [130, 257, 40]),
    ([100, 0, 33, 5, 700], [0, 1, 90, 3, 1])])
def test_attention_chunks_and_mixed(kv, heads, kv_heads, ctx, new):
    _check_attention(_batch(np.random.default_rng(sum(ctx) + heads), ctx, new, heads, kv_heads, kv))


@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("ctx,new", [
    ([5000], [1]), ([4097], [3]), ([3900], [70]), ([17000], [1]), ([20011], [4]), ([30, 17500, 0, 9000], [1, 2, 1, 3]),
    ([5000, 8, 2100], [2, 30, 1]), ([9000], [12])])
def test_attention_long_contexts_split(kv, ctx, new):
    _check_attention(_batch(np.random.default_rng(7), ctx, new, 2, 1, kv))


@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("n_seq", [40, 300])
def test_attention_of_many_sequences(kv, n_seq):
    """Batches that fill the GPU with one and two CTAs per sequence and head."""
    rng = np.random.default_rng(n_seq)
    _check_attention(_batch(rng, rng.integers(0, 300, n_seq).tolist(), rng.integers(0, 3, n_seq).tolist(), 4, 4, kv))


@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("heads,kv_heads", [(25, 25), (36, 18)])
def test_attention_of_more_tiles_than_buffers(kv, heads, kv_heads):
    """Chunks and decoding sequences whose tiles are many more than the SMs and what each keeps of them."""
    rng = np.random.default_rng(heads)
    _check_attention(_batch(rng, rng.integers(0, 300, 80).tolist(), rng.integers(0, 40, 80).tolist(), heads, kv_heads, kv))


@pytest.mark.parametrize("scale", [0.125, 0.01, -0.3, 0.0, 1.0])
def test_attention_scale_and_row_strides(scale):
    _check_attention(_batch(np.random.default_rng(3), [70, 9], [3, 40], 4, 2, torch.float32, ldq_extra=2 * 4 * D), scale)


def test_attention_leaves_padding_and_bad_sequences_alone():
    rng = np.random.default_rng(11)
    b = _batch(rng, [30, 50, 20], [2, 20, 1], 4, 2, torch.float32, extra_rows=6)
    got = _check_attention(b)
    assert (got[23:] == 7.0).all()
    # the second sequence has more new tokens than the call allows, or a length beyond its table
    out = _attend(b, max_new=10).cpu().numpy()
    assert (out[2:22] == 7.0).all() and np.array_equal(out[:2], got[:2].astype(np.float32))
    for ctx in (-1, 10 ** 6, 2 ** 31 - 1):
        c = dict(b, ctx=[30, ctx, 20])
        out = _attend(c).cpu().numpy()
        assert (out[2:22] == 7.0).all() and (out[:2] != 7.0).all() and (out[22] != 7.0).all()
    c = dict(b, start=np.array([0, 2, 40, 41]))                 # rows that do not exist
    out = _attend(c).cpu().numpy()
    assert (out[:2] != 7.0).all() and (out[2:] == 7.0).all()


@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("new", [1, 2, 40])
def test_attention_unmapped_pages_hold_no_positions(kv, new):
    b = _batch(np.random.default_rng(13), [60, 200], [new, new], 4, 2, kv)
    b["table"][0, :] = -1                                       # nothing left: zeros
    b["table"][1, [0, 3, 4]] = [b["k"].shape[0], -5, 2 ** 31 - 1]
    got = _check_attention(b)
    assert (got[:new] == 0.0).all()


@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("new", [1, 3, 40, 150])
@pytest.mark.parametrize("junk", [float("nan"), float("inf"), -3e38, 1e30])
def test_attention_rows_do_not_see_what_is_masked(kv, new, junk):
    """Stale rows behind the context, and later tokens of the chunk itself, hold anything."""
    rng = np.random.default_rng(17)
    b = _batch(rng, [75], [new], 4, 2, kv, spare=1)
    clean = _attend(b).cpu().numpy()
    last, n = ref.pages_of(75 + new) - 1, 75 + new
    for x in (b["k"], b["v"]):
        page = int(b["table"][0, last])
        x[page, (n - 1) % PAGE + 1:] = junk                      # behind the context
        x[[p for p in range(x.shape[0]) if p not in b["table"][0]]] = junk
    assert np.array_equal(_attend(b).cpu().numpy(), clean)
    if new > 1:
        pos = 75 + new // 2                                      # one of the chunk's own tokens
        for x in (b["k"], b["v"]):
            x[int(b["table"][0, pos // PAGE]), pos % PAGE] = junk
        got = _attend(b).cpu().numpy()
        assert np.array_equal(got[:new // 2], clean[:new // 2])  # rows before it
        if not np.isfinite(junk):
            assert not np.isfinite(got[new // 2:]).any()


@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("new", [1, 40])
def test_attention_of_values_far_apart(kv, new):
    """Keys, queries and values of very different sizes keep fp32's relative error."""
    rng = np.random.default_rng(19)
    b = _batch(rng, [140], [new], 2, 1, kv)
    size = torch.from_numpy(np.exp2(rng.integers(-20, 20, (b["v"].shape[0], PAGE, 1))).astype(np.float32)).cuda()
    b["v"] = (b["v"].float() * size).to(kv)
    b["k"] = (b["k"].float() * size.flip(0).clamp(2.0 ** -20, 1.0)).to(kv)
    b["q"] = b["q"] * torch.from_numpy(np.exp2(rng.integers(-30, 1, (b["rows"], 1))).astype(np.float32)).cuda()
    status = _i([0])
    got = _attend(b, status=status).cpu().numpy().astype(np.float64)
    want, vmax, smax = ref.attention(b["q"].cpu().numpy().astype(np.float64), b["k"].cpu().double().numpy(),
                                     b["v"].cpu().double().numpy(), b["table"], b["start"], b["ctx"], 2, 1, 0.125,
                                     np.zeros(got.shape))
    assert (np.abs(got - want) <= ref.attention_bound(vmax, smax, 180)).all()


def test_attention_is_the_same_each_time_in_graphs_and_on_other_streams():
    rng = np.random.default_rng(23)
    b = _batch(rng, [900, 40, 2000], [1, 60, 2], 4, 4, torch.float32)
    ws, table, start, ctx = _workspace(), _i(b["table"]), _i(b["start"]), _i(b["ctx"])
    want = _attend(b, workspace=ws)
    assert torch.equal(_attend(b, workspace=ws), want)
    out = torch.zeros_like(want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.attention_paged(b["q"], b["k"], b["v"], table, start, ctx, 60, out, ws)
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attention_paged(b["q"], b["k"], b["v"], table, start, ctx, 60, out, ws)
    other = _batch(np.random.default_rng(29), [900, 40, 2000], [1, 60, 2], 4, 4, torch.float32)
    for x in ("q", "k", "v"):                                    # new inputs and shorter contexts, the same graph
        b[x].copy_(other[x])
    b["ctx"] = [130, 7, 1500]
    ctx.copy_(_i(b["ctx"]))
    out.fill_(0.0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, _attend(b, workspace=ws))


def test_attention_refuses_a_small_workspace():
    b = _batch(np.random.default_rng(2), [3], [1], 1, 1, torch.float32)
    with pytest.raises(tie_b200.ModelError) as e:
        _attend(b, workspace=torch.empty(1024, dtype=torch.uint8, device="cuda"))
    assert e.value.status == ref.CAPACITY


@pytest.mark.parametrize("new", [1, 33])
def test_attention_and_store_beyond_32_bit_offsets(new):
    """The pool's last pages start behind 2^31 elements."""
    heads, n_pages = 8, (1 << 31) // (PAGE * 8 * D) + 5
    k, v = (torch.empty(n_pages, PAGE, heads * D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    rng = np.random.default_rng(31)
    table = np.array([[n_pages - 1, 3, n_pages - 2, n_pages - 4, 0, n_pages - 3]])
    ctx, rows = 60, 60 + new
    src = torch.from_numpy(rng.standard_normal((rows, 3 * heads * D)).astype(np.float32)).cuda()
    q, kk, vv = src.split(heads * D, 1)
    o = dict(row_start=_out(2), seq_of=_out(rows), pos_of=_out(rows), slot_of=_out(rows), status=_out(1))
    ops.page_plan(_i([0]), _i([rows]), _i(table), n_pages, **o)
    ops.kv_store(kk, vv, o["slot_of"], k, v)
    out = torch.empty(new, heads * D, device="cuda")
    ops.attention_paged(q[ctx:], k, v, _i(table), _i([0, new]), _i([ctx]), new, out, _workspace())
    kd, vd = kk.to(torch.bfloat16).cpu().double().numpy(), vv.to(torch.bfloat16).cpu().double().numpy()
    pad = np.zeros((96 - rows, heads * D))
    want, vmax, smax = ref.attention(q[ctx:].cpu().double().numpy(), np.concatenate([kd, pad]).reshape(6, PAGE, -1),
                                     np.concatenate([vd, pad]).reshape(6, PAGE, -1), np.arange(6)[None], [0, new], [ctx],
                                     heads, heads, 0.125, np.zeros((new, heads * D)))
    assert (np.abs(out.cpu().numpy() - want) <= ref.attention_bound(vmax, smax, rows)).all()


def _long(kv, ctx, new, heads, scores, unmapped=0):
    """One sequence, one K/V head, values around 1; (got, want) of some of its rows, want in 64 bits.

    scores(position) is added to what every row scores the position, in units of the score."""
    total, rng = ctx + new, np.random.default_rng(ctx + heads)
    n_pages = ref.pages_of(total)
    table = rng.permutation(n_pages)
    q, k, v = rng.standard_normal((new, heads * D)), rng.standard_normal((total, D)), 1 + rng.standard_normal((total, D))
    q, k = 0.02 * q.reshape(new, heads, D), 0.1 * k
    q[..., 0], k[:, 0] = 1.0, scores(np.arange(total))
    dev = lambda x: torch.from_numpy(x.astype(np.float32)).cuda()  # noqa: E731
    q, pools = dev(q.reshape(new, -1)), []
    for x in (k, v):
        pool = torch.zeros(n_pages, PAGE, D, device="cuda")
        pool[torch.from_numpy(table).cuda()] = torch.nn.functional.pad(dev(x), (0, 0, 0, -total % PAGE)).view(n_pages, PAGE, D)
        pools.append(pool.to(kv))
    mapped = np.where(np.arange(n_pages) < unmapped // PAGE, -1, table)
    out = torch.full((new, heads * D), 7.0, device="cuda")
    ops.attention_paged(q, *pools, _i(mapped[None]), _i([0, new]), _i([ctx]), new, out, _workspace(), scale=1.0)
    pick = torch.from_numpy(np.unique(np.linspace(0, new - 1, 24).astype(int))).cuda()
    kd, vd = (x[torch.from_numpy(table).cuda()].view(-1, D)[:total].double() for x in pools)
    s = q.view(new, heads, D)[pick].double() @ kd.T
    pos = torch.arange(total, device="cuda")
    s.masked_fill_((pos > ctx + pick[:, None, None]) | (pos < unmapped), -torch.inf)
    return out.view(new, heads, D)[pick].double(), s.softmax(-1) @ vd


@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("heads,new", [(16, 1024), (4, 16)])
def test_attention_of_many_keys_keeps_32_bits(kv, heads, new):
    """30,000 keys of about the same weight: what each step cuts off its sums must not add up.

    Relative bounds, each at its worst: an O of at most 64 MMAs, each of which cuts off at most one unit in
    the last place of a sum that grows evenly, 32 x 2^-23; the split of q, k, p and v, 4 x 2^-22; scores of
    |s| < 0.5 from 12 MMAs that cut off likewise, 12 x 2^-24; 2^x, 2^-22; 1 in 128 of the additions to the row
    sum one after the other (240 steps, in two streams or by two CTAs or more), 120 x 2^-24. In all
    2^-24 (64 + 16 + 12 + 4 + 120) = 1.3e-5."""
    got, want = _long(kv, 30000, new, heads, lambda pos: 0.0 * pos)
    assert torch.linalg.vector_norm(got - want) <= 1.3e-5 * torch.linalg.vector_norm(want)
    # a sum that loses always in one direction shows in the mean: half of the first bound, of 64 MMAs (the rest
    # is rounded, which has no direction, or belongs to a row's sum: 8 x 2^-24 in the mean of the rows)
    assert abs(float((got / want)[want > 0.5].mean()) - 1) <= (32 + 8) * 2.0 ** -24


@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("ramp", [300.0, -300.0, 20.0])
@pytest.mark.parametrize("unmapped", [0, 2064])
def test_attention_of_maxima_that_move(kv, ramp, unmapped):
    """Scores that rise or fall along the context by far more than a running sum can hold at one scale.

    The bound of attention_bound, with the largest sum |q||k| of a row for its scores (the ramp, and 0.02 x 0.1
    x 64 products of at most 5 deviations each way) and the values of the data."""
    n = 6000
    got, want = _long(kv, n, 700, 16, lambda pos: ramp * pos / n, unmapped)
    bound = ref.attention_bound(6.0, abs(ramp) * 1.2 + 1.0, n + 700)
    assert float((got - want).abs().max()) <= bound


def test_binding_reads_tensors_as_they_are():
    """Parameters, views with an offset, single rows of any stride, streams by number; refusals with the GPU's tensors."""
    rng = np.random.default_rng(2)
    b = _batch(rng, [20, 3], [1, 2], 2, 1, torch.float32)
    want = _attend(b)
    wide = torch.full((4, 200), 5.0, device="cuda")
    out = wide[1:, 8:136]
    got = _attend(dict(b, q=torch.nn.Parameter(b["q"].clone())), out=out)
    assert got is out and torch.equal(out, want) and bool((wide[:, :8] == 5).all()) and bool((wide[0] == 5).all())
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    again = torch.zeros_like(want)
    ops.attention_paged(b["q"], b["k"], b["v"], _i(b["table"]), _i(b["start"]), _i(b["ctx"]), 2, again, _workspace(),
                        stream=stream.cuda_stream)
    stream.synchronize()
    assert torch.equal(again, want)
    k1 = torch.arange(64.0, device="cuda")[None].expand(1, 64)
    ops.kv_store(k1, k1.clone(), _i([3]), b["k"], b["v"])
    assert torch.equal(b["k"][0, 3], k1[0]) and torch.equal(b["v"][0, 3], k1[0])
    for bad in (dict(q=b["q"].cpu()), dict(q=b["q"].double()), dict(k=b["k"].cpu()), dict(v=b["v"].bfloat16()),
                dict(k=b["k"][:, :8], v=b["v"][:, :8]), dict(max_new=1 << 32), dict(q=b["q"].T), dict(q=b["q"][0]),
                dict(q=b["q"].cpu().numpy())):
        with pytest.raises(ValueError):
            _attend(dict(b, **bad), out=want)
    with pytest.raises(TypeError):
        _attend(b, scale="large")
    with pytest.raises(ValueError):
        ops.kv_store(k1, k1.clone(), torch.zeros(1, device="cuda"), b["k"], b["v"])


def test_calls_of_many_sequences_on_two_threads():
    """Numbers of sequences that ask for different amounts of shared memory, side by side."""
    import threading
    failed = []

    def calls(n_seq, seed):
        try:
            rng = np.random.default_rng(seed)
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                b = _batch(rng, [3] * n_seq, [2] + [1] * (n_seq - 1), 4, 1, torch.float32)
                b["max_new"] = 9          # not all sequences have few rows, as far as the call knows
                first, ws = _attend(b), _workspace()
                for _ in range(40):
                    o = dict(row_start=_out(n_seq + 1), seq_of=_out(n_seq + 1), pos_of=_out(n_seq + 1),
                             slot_of=_out(n_seq + 1), status=_out(1))
                    ops.page_plan(_i([3] * n_seq), _i([1] * n_seq), _i(b["table"]), 2 * n_seq + 8, **o)
                    again = _attend(b, workspace=ws)
                stream.synchronize()
                assert torch.equal(first, again) and int(o["status"][0]) == 0
                assert o["row_start"].tolist() == list(range(n_seq + 1))
        except Exception as e:                                     # noqa: BLE001
            failed.append((n_seq, repr(e)))

    threads = [threading.Thread(target=calls, args=(n, n)) for n in (4096, 3950)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not failed


# ------------------------------------------------------------------ beam selection

def _select(logits, scores, beams, done=None, eos=-1, alias=False):
    n, vocab = logits.shape
    ws = torch.empty(max(16, ops.beam_select_workspace(n // beams, beams, vocab)), dtype=torch.uint8, device="cuda")
    sc = torch.from_numpy(np.asarray(scores, np.float32)).cuda()
    dn = None if done is None else _i(done)
    so = sc if alias else _out(n, torch.float32)
    do = dn if alias or done is None else _out(n)
    nxt, par = _out(n), _out(n)
    ops.beam_select(logits, sc, beams, nxt, par, so, ws, done=dn, done_out=do, eos_id=eos)
    return [x.cpu().numpy() if x is not None else np.zeros(n, np.int64) for x in (nxt, par, so, do)]


def _check_select(logits, scores, beams, done=None, eos=-1, alias=False):
    """Equal choices; scores within a float's half step of totals that fp32 exponentials put at most 2^-21 off
    (the logarithm of a sum whose terms are each 2^-22 + 2^-23 off), and the score itself rounded."""
    got = _select(logits, scores, beams, done, eos, alias)
    want = ref.beam_select(logits.cpu().numpy(), np.asarray(scores, np.float32), done, beams, eos)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    if done is not None:
        assert np.array_equal(got[3], want[3])
    fin = np.isfinite(want[2])
    assert np.array_equal(got[2][~fin], want[2][~fin].astype(np.float32))
    assert (np.abs(got[2][fin] - want[2][fin]) <= 2.0 ** -21 + 2.0 ** -24 * np.abs(want[2][fin])).all()
    return got


@pytest.mark.parametrize("n_req,beams,vocab", [
    (1, 1, 1), (1, 4, 1), (2, 3, 2), (1, 4, 50257), (3, 5, 50257), (40, 2, 1000), (2, 16, 5003), (700, 1, 257), (5, 16, 16), (3, 7, 4099)])
def test_select_matches_the_definition(n_req, beams, vocab):
    rng = np.random.default_rng(vocab + beams)
    n = n_req * beams
    logits = torch.from_numpy((3 * rng.standard_normal((n, vocab))).astype(np.float32)).cuda()
    _check_select(logits, -10 * rng.random(n), beams)
    _check_select(logits, -10 * rng.random(n), beams, (rng.random(n) < 0.3).astype(np.int64), vocab - 1, alias=True)
    _check_select(logits, np.where(rng.random(n) < 0.5, -np.inf, -1.0), beams, np.zeros(n, np.int64), 0)


def test_select_ties_go_to_the_lowest_index_whatever_the_rows_alignment():
    """Equal beams on rows at every alignment: real ties, in the order of beam * vocab + token."""
    rng = np.random.default_rng(1)
    vocab, beams = 9001, 4
    row = (2 * rng.standard_normal(vocab)).astype(np.float32)
    row[[17, 4000, 8999]] = row.max() + 1
    logits = torch.from_numpy(np.tile(row, (2 * beams, 1))).cuda()          # odd row length: four alignments
    got = _check_select(logits, np.zeros(2 * beams), beams)
    # ranks: beam 0's three best tokens, then beam 1's first; beam 0 keeps its place
    assert list(got[0][:4]) == [17, 17, 4000, 8999] and list(got[1][:4]) == [0, 1, 0, 0]
    _check_select(torch.zeros(2 * beams, 70, device="cuda"), np.zeros(2 * beams), beams)


def test_select_of_rows_without_a_normaliser():
    vocab, beams = 3000, 3
    rng = np.random.default_rng(4)
    base = rng.standard_normal((beams, vocab)).astype(np.float32)
    for bad in ("nan", "-inf", "inf", "mostly"):
        x = base.copy()
        if bad == "nan":
            x[1, 5:900] = np.nan
        elif bad == "mostly":
            x[:, 2:] = -np.inf                                    # two candidates a beam: -inf fills nothing here
            x[1] = -np.inf
            x[2] = -np.inf
        else:
            x[1, :] = -np.inf
            if bad == "inf":
                x[1, 77] = np.inf
        _check_select(torch.from_numpy(x).cuda(), np.array([-3.0, -0.5, -2.0]), beams)
    x = np.full((beams, vocab), np.nan, np.float32)
    _check_select(torch.from_numpy(x).cuda(), np.zeros(beams), beams)
    _check_select(torch.from_numpy(base).cuda(), np.array([np.nan, -np.inf, np.nan]), beams)


def test_select_row_stride_and_many_rows():
    rng = np.random.default_rng(6)
    x = torch.from_numpy(rng.standard_normal((1200, 601)).astype(np.float32)).cuda()
    _check_select(x[:, 1:600], -rng.random(1200), 4)


# ------------------------------------------------------------------ reorder

@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("layers,n_req,beams,heads", [(1, 1, 2, 1), (3, 2, 4, 2), (2, 9, 5, 3), (12, 1, 16, 1), (2, 300, 3, 1)])
def test_reorder_any_parents(kv, layers, n_req, beams, heads):
    rng = np.random.default_rng(beams + n_req)
    n, width = n_req * beams, 5
    n_pages = n * width + 1
    table = rng.permutation(n_pages)[:n * width].reshape(n, width)
    first, length = rng.integers(0, 60, n_req), rng.integers(0, 81, n_req)
    first[0], length[0] = 17, 80
    parent = np.concatenate([r * beams + rng.integers(0, beams, beams) for r in range(n_req)])
    parent[:beams] = np.roll(np.arange(beams), 1)                # a cycle: every beam moves
    pages = [torch.from_numpy(rng.standard_normal((layers, n_pages, PAGE, heads * D)).astype(np.float32)).cuda().to(kv)
             for _ in range(2)]
    want = [ref.reorder(p.float().cpu().numpy(), table, parent, first, length, beams) for p in pages]
    ops.kv_reorder(*pages, _i(table), _i(parent), _i(first), _i(length), beams)
    for p, x in zip(pages, want):
        assert np.array_equal(p.float().cpu().numpy(), x)


def test_reorder_moves_nothing_it_should_not():
    rng = np.random.default_rng(8)
    table = np.arange(12).reshape(4, 3)
    table[1, 0] = table[0, 0]                                    # a shared page
    table[3, 1], table[2, 2] = -1, 12                            # unmapped
    pages = [torch.from_numpy(rng.standard_normal((12, PAGE, D)).astype(np.float32)).cuda() for _ in range(2)]
    for parent, first, length in (([1, 0, 3, 2], [0, 0], [48, 48]), ([2, 0, 0, 3], [5, 5], [40, 40]), ([0, 1, 2, 3], [0, 0], [48, 48]),
                                  ([-1, 9, 2 ** 31 - 1, -2 ** 31], [0, 0], [48, 48]), ([1, 1, 3, 3], [-4, 20], [10 ** 9, 20])):
        # beams 0 and 1 never both write the shared page: an entry equal to the parent's moves nothing
        want = [ref.reorder(p.cpu().numpy()[None], table, parent, first, length, 2)[0] for p in pages]
        ops.kv_reorder(*pages, _i(table), _i(parent), _i(first), _i(length), 2)
        for p, x in zip(pages, want):
            assert np.array_equal(p.cpu().numpy(), x)


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("kv", KV)
def test_a_beam_search_over_the_pool(kv):
    """Plan, store, attend, select, reorder, step after step, as a caller would run them: the attention of
    each beam equals attention over that beam's own history, kept in 64 bits on the side."""
    rng = np.random.default_rng(41)
    n_req, beams, heads, vocab, prompt, steps = 2, 3, 2, 500, 21, 14
    n, w = n_req * beams, heads * D
    width = ref.pages_of(prompt + steps)
    n_pages = n * width + 2
    k, v = (torch.zeros(n_pages, PAGE, w, device="cuda", dtype=kv) for _ in range(2))
    table, free, n_free = _i(np.full((n, width), n_pages)), _i(rng.permutation(n_pages)), _i([n_pages])
    ws, ws2 = _workspace(), torch.empty(ops.beam_select_workspace(n_req, beams, vocab), dtype=torch.uint8, device="cuda")
    emb = rng.standard_normal((vocab, 3 * w)).astype(np.float32)       # a token's query, key and value
    head = torch.from_numpy((rng.standard_normal((w, vocab)) * 0.7).astype(np.float32)).cuda()
    emb_d = torch.from_numpy(emb).cuda()
    lens = _i([0] * n)
    prompts = rng.integers(0, vocab, (n_req, prompt)).repeat(beams, 0)
    hist = [list(p) for p in prompts]
    tokens, new = torch.from_numpy(prompts.reshape(-1)).cuda(), prompt
    scores = torch.full((n,), float("-inf"), device="cuda")
    scores[::beams] = 0.0
    done, first, nxt, par = _i([0] * n), _i([prompt] * n_req), _out(n), _out(n)
    for step in range(steps):
        rows = n * new
        o = dict(row_start=_out(n + 1), seq_of=_out(rows), pos_of=_out(rows), slot_of=_out(rows), status=_out(1))
        ops.page_plan(lens, _i([new] * n), table, n_pages, **o, free_pages=free, n_free=n_free, n_free_out=n_free)
        assert int(o["status"][0]) == ref.OK
        qkv = emb_d[tokens.long()]
        ops.kv_store(qkv[:, w:2 * w], qkv[:, 2 * w:], o["slot_of"], k, v)
        out = torch.empty(rows, w, device="cuda")
        ops.attention_paged(qkv[:, :w], k, v, table, o["row_start"], lens, new, out, ws)
        last = out.view(n, new, w)[:, -1]
        got = last.cpu().numpy().astype(np.float64)
        for s in range(n):
            h = emb[np.array(hist[s])]
            hk, hv = (torch.from_numpy(h[:, c * w:(c + 1) * w]).to(kv).double().numpy() for c in (1, 2))
            pad = np.zeros((-len(h) % PAGE, w))
            want, vmax, smax = ref.attention(h[-1:, :w].astype(np.float64), np.concatenate([hk, pad]).reshape(-1, PAGE, w),
                                             np.concatenate([hv, pad]).reshape(-1, PAGE, w), np.arange(width)[None], [0, 1],
                                             [len(h) - 1], heads, heads, 0.125, np.zeros((1, w)))
            assert (np.abs(got[s] - want[0]) <= ref.attention_bound(vmax, smax, len(h))[0]).all(), (step, s)
        lens += new
        logits = last @ head
        want = ref.beam_select(logits.cpu().numpy(), scores.cpu().numpy(), done.cpu().numpy(), beams, 3)
        ops.beam_select(logits, scores, beams, nxt, par, scores, ws2, done=done, done_out=done, eos_id=3)
        assert np.array_equal(nxt.cpu().numpy(), want[0]) and np.array_equal(par.cpu().numpy(), want[1])
        # the rows cached so far: positions first .. lens - 1
        ops.kv_reorder(k, v, table, par, first, lens[::beams].contiguous(), beams)
        hist = [hist[p] + [int(t)] for p, t in zip(par.tolist(), nxt.tolist())]
        tokens, new = nxt, 1
