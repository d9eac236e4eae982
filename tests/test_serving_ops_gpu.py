"""The 8-bit cache, attention over shared positions and the 4-bit weights on the GPU against their 64-bit definitions
(serving_oracle.py)."""
import os
import sys

import numpy as np
import pytest

import tie_b200
from tie_b200 import ops

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import ops_oracle as paged  # noqa: E402
import serving_oracle as ref  # noqa: E402

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
PAGE, D, EPS = 16, 64, 2.0 ** -24
I32 = torch.int32


def _i(v):
    return torch.tensor(np.asarray(v), dtype=I32, device="cuda")


def _f(v):
    return torch.tensor(np.asarray(v), dtype=torch.float32, device="cuda")


def _np(t):
    return t.float().cpu().numpy() if t.dtype == torch.bfloat16 else t.cpu().numpy()


# ------------------------------------------------------------------ the cache in 8 bits

def _check_store(k, v, slots, heads, n_pages, stride=0):
    """Stores rows and reads them back; levels, scales and values equal the definition's, the rest is as it was."""
    rows, w = len(k), heads * D
    rng = np.random.default_rng(rows)
    pages = [rng.integers(-127, 128, (n_pages, PAGE, w)).astype(np.int8) for _ in range(2)]
    scales = [rng.random((n_pages, heads, PAGE)).astype(np.float32) for _ in range(2)]
    wide = torch.zeros(rows, 2 * w + stride, device="cuda")
    wide[:, :w], wide[:, w:2 * w] = _f(k), _f(v)
    dp, ds = [torch.tensor(p, device="cuda") for p in pages], [_f(s) for s in scales]
    ops.kv_store_q8(wide[:, :w], wide[:, w:2 * w], _i(slots), dp[0], dp[1], ds[0], ds[1])
    got = torch.full((rows, 2 * w + stride), -5.0, device="cuda")
    ops.kv_load(_i(slots), dp[0], dp[1], got[:, :w], got[:, w:2 * w], ds[0], ds[1])
    got = got.cpu().numpy()
    assert (got[:, 2 * w:] == -5.0).all()
    for i, x in enumerate((k, v)):
        p, s = ref.store_q8(x, slots, pages[i], scales[i])
        assert np.array_equal(_np(dp[i]), p)
        assert np.array_equal(_np(ds[i]), s, equal_nan=True)
        for r, slot in enumerate(slots):
            mine = got[r, i * w:(i + 1) * w]
            if 0 <= slot < n_pages * PAGE:
                with np.errstate(invalid="ignore", over="ignore"):
                    want = p[slot // PAGE, slot % PAGE].reshape(heads, D).astype(np.float32) * s[slot // PAGE, :, slot % PAGE, None]
                assert np.array_equal(mine, want.reshape(-1), equal_nan=True)
            else:
                assert (mine == -5.0).all()


@pytest.mark.parametrize("rows,heads,stride", [(1, 1, 0), (3, 2, 4), (33, 5, 0), (257, 12, 64), (1000, 3, 8)])
def test_rows_are_stored_in_8_bits_and_read_back(rows, heads, stride):
    rng = np.random.default_rng(rows * heads)
    n_pages = rows // PAGE + 3
    slots = rng.permutation(n_pages * PAGE)[:rows]
    slots[rng.random(rows) < 0.1] = -1
    slots[rng.random(rows) < 0.05] = n_pages * PAGE
    k, v = (rng.standard_normal((rows, heads * D)).astype(np.float32) for _ in range(2))
    _check_store(k, v, slots, heads, n_pages, stride)


def test_levels_next_to_their_borders():
    """Quotients that are ties, next to ties, next to the ends; rows of zeros, of the smallest and largest numbers, of
    none that are finite."""
    f = np.float32
    rng = np.random.default_rng(1)
    rows = []
    for scale in (1.0, 2.0 ** -20, 2.0 ** 100, 0.3, 1e-3, 7.77, 2.0 ** -126, 2.0 ** -130, 1e-44):
        half = (np.arange(-32, 32) + 0.5).astype(f) * f(scale)
        for x in (half, np.nextafter(half, f(np.inf)), np.nextafter(half, f(-np.inf)), (4 * half).astype(f)):
            x = x.copy()
            x[0] = f(127.0) * f(scale)
            rows.append(x)
    rows += [np.zeros(D, f), np.full(D, f(-1e-45)), np.full(D, f(3.4028235e38)), np.full(D, f(-3.4028235e38))]
    rows += [rng.standard_normal(D).astype(f) * f(10.0 ** e) for e in (-44, -40, -38, -37, -30, 30, 37)]
    for bad in (np.inf, -np.inf, np.nan):
        x = rng.standard_normal(D).astype(f)
        x[rng.integers(D)] = bad
        rows.append(x)
    x = np.stack(rows)
    _check_store(x, x[::-1].copy(), rng.permutation(len(x) + 7)[:len(x)], 1, (len(x) + 7) // PAGE + 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_other_pools_are_read_back(dtype):
    """As they are; a slot may be read by many rows."""
    rng = np.random.default_rng(3)
    heads, n_pages, rows = 3, 5, 211
    pages = [_f(rng.standard_normal((n_pages, PAGE, heads * D))).to(dtype) for _ in range(2)]
    slots = rng.integers(-2, n_pages * PAGE + 2, rows)
    out = [torch.full((rows, heads * D), 9.0, device="cuda") for _ in range(2)]
    ops.kv_load(_i(slots), pages[0], pages[1], out[0], out[1])
    for p, o in zip(pages, out):
        want = np.full((rows, heads * D), 9.0, np.float32)
        ok = (slots >= 0) & (slots < n_pages * PAGE)
        want[ok] = _np(p).reshape(-1, heads * D)[slots[ok]]
        assert np.array_equal(_np(o), want)


# ------------------------------------------------------------------ attention

KINDS = ["f32", "bf16", "q8"]


def _pool(rng, n_pages, heads, kind, spread=1.0):
    """Pages and scales on the device, and as numpy arrays for the definition."""
    out = []
    for _ in range(2):
        if kind == "q8":
            p = torch.tensor(rng.integers(-127, 128, (n_pages, PAGE, heads * D)).astype(np.int8), device="cuda")
            s = _f((0.2 + rng.random((n_pages, heads, PAGE))) * spread / 70)
            out.append((p, s, p.cpu().numpy(), s.cpu().numpy()))
        else:
            p = _f(rng.standard_normal((n_pages, PAGE, heads * D)) * spread)
            p = p.to(torch.bfloat16) if kind == "bf16" else p
            out.append((p, None, _np(p), None))
    return out


class Batch:
    """A batch over a pool in random pages: groups of sequences with shared first positions."""

    def __init__(self, seed, ctx, new, heads, kv_heads, kind, groups=(), shared=(), pad_rows=0, spread=1.0, q_spread=2.0,
                 unmapped=0.0):
        rng = self.rng = np.random.default_rng(seed)
        self.heads, self.kv_heads, self.kind = heads, kv_heads, kind
        need = [-(-(c + n) // PAGE) for c, n in zip(ctx, new)]
        first = [-(-n // PAGE) for n in shared]
        n_pages = self.n_pages = sum(need) + sum(first) + 2
        perm = rng.permutation(n_pages)
        at = 0

        def table(of):
            nonlocal at
            t = np.full((len(of), max(max(of), 1)), n_pages, np.int64)
            for i, m in enumerate(of):
                t[i, :m] = perm[at:at + m]
                at += m
            t[rng.random(t.shape) < unmapped] = -1
            return t

        self.table = table(need)
        self.ctx, self.new = np.array(ctx), np.array(new)
        self.start = np.concatenate([[0], np.cumsum(new)])
        self.rows = int(self.start[-1]) + pad_rows
        self.groups, self.shared = np.array(groups, np.int64), np.array(shared, np.int64)
        self.ptable = table(first) if len(shared) else None
        self.max_new = max(new) if len(new) else 0
        (self.k, self.ks, self.kn, self.ksn), (self.v, self.vs, self.vn, self.vsn) = _pool(rng, n_pages, kv_heads, kind, spread)
        self.q = (q_spread * rng.standard_normal((self.rows, heads * D))).astype(np.float32)
        self.scale = 0.125

    def sync_pool(self):
        """The arrays' values to the device's tensors."""
        for t, a in ((self.k, self.kn), (self.v, self.vn), (self.ks, self.ksn), (self.vs, self.vsn)):
            if t is not None:
                t.copy_(torch.tensor(a, device="cuda").to(t.dtype))

    def call(self, out=None, stream=None, ws=None, q=None):
        if out is None:
            out = torch.full((self.rows, self.heads * D), -3.0, device="cuda")
        if ws is None:
            ws = torch.empty(ops.attention_shared_workspace(self.rows, self.heads), dtype=torch.uint8, device="cuda")
            ws.fill_(0xff)                 # what a workspace holds is nothing to a call
        kw = {}
        if self.ptable is not None:
            kw = dict(prefix_table=_i(self.ptable), prefix_lens=_i(self.shared), group_start=_i(self.groups))
        ops.attention_shared(_f(self.q) if q is None else q, self.k, self.v, _i(self.table), _i(self.start), _i(self.ctx),
                             self.max_new, out, ws, k_scales=self.ks, v_scales=self.vs, scale=self.scale, stream=stream, **kw)
        return out

    def want(self):
        kw = {}
        if self.ptable is not None:
            kw = dict(prefix_table=self.ptable, prefix_lens=self.shared, group_start=self.groups)
        out = np.full((self.rows, self.heads * D), -3.0)
        o, vmax, smax = ref.attention(self.q, self.kn, self.vn, self.table, self.start, self.ctx, self.heads, self.scale, out,
                                      self.max_new, self.ksn, self.vsn, **kw)
        length = int(max(self.ctx + self.new)) + (int(self.shared.max()) if len(self.shared) else 0)
        return o, paged.attention_bound(vmax, smax, length)

    def check(self, **kw):
        got = _np(self.call(**kw)).astype(np.float64)
        o, bound = self.want()
        assert np.array_equal(np.isnan(got), np.isnan(o))
        off = np.abs(got - o)
        worst = np.nanmax(off - bound) if off.size else 0.0
        assert not (off > bound).any(), (worst, np.argwhere(off > bound)[:3].tolist())
        return got


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (8, 2), (6, 1), (16, 2)])
@pytest.mark.parametrize("ctx,new,groups,shared", [
    ([0], [1], (), ()), ([15], [1], (), ()), ([16], [1], (), ()), ([130], [3], (), ()),
    ([0, 0], [1, 1], (0, 2), (1,)), ([3, 20], [1, 1], (0, 2), (16,)), ([0, 7, 40], [1, 1, 1], (0, 3), (63,)),
    ([5, 0, 33, 90], [1, 2, 0, 4], (0, 2, 4), (50, 129)), ([9, 9, 9, 200, 1], [1, 1, 1, 1, 1], (1, 3, 3, 4), (70, 20, 5)),
])
def test_attention_matches_the_definition(kind, heads, kv_heads, ctx, new, groups, shared):
    Batch(len(ctx) + heads, ctx, new, heads, kv_heads, kind, groups, shared, pad_rows=2).check()


@pytest.mark.parametrize("kind", KINDS)
def test_attention_of_many_rows(kind):
    """Items of 8, 16 and 32 rows and more than one of them: chunks behind a cache, many sequences behind one text."""
    Batch(1, [30, 0], [37, 9], 2, 1, kind).check()
    Batch(2, [30, 0, 4], [10, 1, 13], 3, 3, kind, (0, 3), (100,)).check()
    rng = np.random.default_rng(5)
    Batch(3, rng.integers(0, 40, 70).tolist(), [1] * 70, 2, 2, kind, (0, 70), (333,)).check()
    Batch(4, rng.integers(0, 40, 30).tolist(), rng.integers(0, 3, 30).tolist(), 4, 1, kind, (0, 10, 11, 30), (40, 100, 77)).check()


@pytest.mark.parametrize("kind", KINDS)
def test_attention_over_long_texts(kind):
    """Long enough that every warp's stretch cuts items, and that a row has hundreds of parts."""
    Batch(1, [9000], [1], 1, 1, kind).check()
    Batch(2, [100, 0, 2500], [1, 1, 1], 2, 1, kind, (0, 3), (7001,)).check()


def test_attention_of_many_sequences():
    rng = np.random.default_rng(9)
    n = 4096
    b = Batch(1, rng.integers(0, 9, n).tolist(), rng.integers(0, 2, n).tolist(), 1, 1, "f32",
              tuple(range(0, n + 1, 2)), tuple(rng.integers(1, 30, n // 2).tolist()))
    b.check()


@pytest.mark.parametrize("kind", KINDS)
def test_pages_that_are_not_mapped_hold_nothing(kind):
    """Also where that leaves a row nothing: zeros."""
    Batch(7, [50, 3, 90], [1, 2, 1], 4, 2, kind, (0, 2, 3), (60, 20), unmapped=0.4).check()
    b = Batch(8, [50, 3], [1, 2], 4, 2, kind, (0, 2), (60,), unmapped=1.0)
    assert (b.check() == 0.0).all()
    b = Batch(8, [50, 3], [1, 2], 4, 2, kind, unmapped=1.0)
    assert (b.check() == 0.0).all()


@pytest.mark.parametrize("kind", KINDS)
def test_sequences_that_are_left_out_keep_their_rows(kind):
    """No new tokens, more than max_new, beyond the table; groups whose range or length has no meaning; rows behind
    the last sequence."""
    b = Batch(3, [20, 5, 40, 8], [1, 5, 2, 1], 2, 1, kind, (0, 2, 4), (33, 20), pad_rows=3)
    b.max_new = 2
    assert (b.check()[1:6] == -3.0).all()
    b.ctx[2] = 10 ** 6
    assert (b.check()[6:8] == -3.0).all()
    b.ctx[2], b.ctx[3] = 40, -1
    b.check()
    for groups, shared in (((-1, 2, 4), (33, 20)), ((0, 2, 5), (33, 20)), ((3, 2, 4), (33, 20)), ((0, 2, 4), (-5, 20)),
                           ((0, 2, 4), (0, 0)), ((0, 2, 4), (33, 10 ** 8))):
        b = Batch(3, [20, 5, 40, 8], [1, 2, 2, 1], 2, 1, kind, (0, 2, 4), (33, 20))
        b.groups, b.shared = np.array(groups), np.array(shared)
        b.check()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_what_no_row_sees_changes_nothing(kind, bad):
    """Anything in the rest of the last pages, in pages of nobody, and in positions that earlier rows do not see."""
    b = Batch(11, [21, 3], [1, 6], 4, 2, kind, (0, 2), (40,))
    before = b.check()
    lens = np.concatenate([b.ctx + b.new, b.shared])
    used = np.zeros((b.n_pages, PAGE), bool)
    for entries, n in zip(list(b.table) + list(b.ptable), lens):
        for p in range(n):
            used[entries[p // PAGE], p % PAGE] = True
    for values in ([b.ksn, b.vsn] if kind == "q8" else [b.kn, b.vn]):
        if kind == "q8":
            np.moveaxis(values, 1, 2)[~used] = bad
        else:
            values[~used] = bad
    b.sync_pool()
    assert np.array_equal(b.check(), before)
    # a value of sequence 1's last position: its last row is not finite, the others are as they were
    p = b.ctx[1] + b.new[1] - 1
    if kind == "q8":
        b.vsn[b.table[1, p // PAGE], :, p % PAGE] = bad
    else:
        b.vn[b.table[1, p // PAGE], p % PAGE] = bad
    b.sync_pool()
    got = _np(b.call())
    assert np.array_equal(got[:-1], before[:-1].astype(np.float32)) and not np.isfinite(got[-1]).any()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_largest_and_smallest_numbers(kind):
    """Values near the ends of the range, beside one another; scores that a softmax in fp32 can only just hold apart."""
    b = Batch(13, [300, 20], [1, 2], 4, 2, kind, (0, 2), (120,))
    big = 3.3895314e38                                     # bf16's largest number
    b.vn[:] = np.where(b.rng.random(b.vn.shape) < 0.5, big, np.float32(1e-38))
    b.sync_pool()
    got = b.check()
    assert np.isfinite(got).all()
    b = Batch(14, [300, 20], [1, 2], 4, 2, kind, (0, 2), (120,), q_spread=40.0)
    b.check()
    b = Batch(15, [30], [1], 1, 1, kind)
    b.kn *= 0.0                                            # equal scores: the mean of what is seen
    b.sync_pool()
    b.check()


def test_strides_and_scale():
    b = Batch(17, [40, 9], [2, 1], 4, 2, "f32", (0, 2), (20,))
    b.scale = -0.031
    wide_q = torch.zeros(b.rows, 5 * D, device="cuda")
    wide_q[:, :4 * D] = _f(b.q)
    wide_out = torch.full((b.rows, 4 * D + 12), -3.0, device="cuda")
    b.call(out=wide_out[:, :4 * D], q=wide_q[:, :4 * D])
    o, bound = b.want()
    got = _np(wide_out)
    assert (np.abs(got[:, :4 * D] - o) <= bound).all() and (got[:, 4 * D:] == -3.0).all()


def test_the_same_call_gives_the_same_bits():
    b = Batch(19, [700, 20, 333, 4, 90], [1, 1, 1, 1, 1], 8, 4, "bf16", (0, 5), (2000,))
    first = b.call()
    for _ in range(3):
        assert torch.equal(b.call(), first)


@pytest.mark.parametrize("kind", KINDS)
def test_streams_and_graphs(kind):
    """Two calls at once with a workspace each, and a captured call that is replayed for other lengths."""
    b, c = Batch(21, [400, 20], [1, 1], 4, 2, kind, (0, 2), (500,)), Batch(22, [30] * 40, [1] * 40, 4, 2, kind, (0, 40), (100,))
    want = [_np(b.call()), _np(c.call())]
    torch.cuda.synchronize()
    ws = [torch.empty(ops.attention_shared_workspace(x.rows, x.heads), dtype=torch.uint8, device="cuda") for x in (b, c)]
    outs = [[], []]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for i, x in enumerate((b, c)):
            with torch.cuda.stream(streams[i]):
                outs[i].append(x.call(ws=ws[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(np.array_equal(_np(o), want[i]) for o in outs[i])
    # the graph
    q, table, start, ctx = _f(b.q), _i(b.table), _i(b.start), _i(b.ctx)
    pt, pl, gs = _i(b.ptable), _i(b.shared), _i(b.groups)
    out = torch.full((b.rows, 4 * D), -3.0, device="cuda")
    args = dict(k_scales=b.ks, v_scales=b.vs, prefix_table=pt, prefix_lens=pl, group_start=gs)
    ops.attention_shared(q, b.k, b.v, table, start, ctx, 1, out, ws[0], **args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attention_shared(q, b.k, b.v, table, start, ctx, 1, out, ws[0], **args)
    for lens, n in (([400, 20], 500), ([17, 0], 499), ([0, 19], 1)):
        b.ctx, b.shared = np.array(lens), np.array([n])
        ctx.copy_(_i(lens))
        pl.copy_(_i([n]))
        graph.replay()
        torch.cuda.synchronize()
        o, bound = b.want()
        assert (np.abs(_np(out) - o) <= bound).all()


def test_a_pool_beyond_32_bits():
    """Pages whose elements lie behind 2^31 of them."""
    heads, n_pages = 16, 140000
    k = torch.empty(n_pages, PAGE, heads * D, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    assert k.numel() > 2 ** 31
    b = Batch(23, [40], [1], heads, heads, "bf16", (0, 1), (30,))
    far = n_pages - 1 - np.arange(b.n_pages)
    k[torch.tensor(far, device="cuda")], v[torch.tensor(far, device="cuda")] = b.k, b.v
    o, bound = b.want()
    b.table, b.ptable = np.where(b.table < b.n_pages, n_pages - 1 - b.table, -1), n_pages - 1 - b.ptable
    b.k, b.v = k, v
    assert (np.abs(_np(b.call()) - o) <= bound).all()
    rows = [torch.zeros(3, heads * D, device="cuda") for _ in range(2)]
    ops.kv_load(_i((n_pages - 1) * PAGE + np.arange(3)), k, v, rows[0], rows[1])
    assert torch.equal(rows[0], k[-1, :3].float()) and torch.equal(rows[1], v[-1, :3].float())


def test_without_groups_it_is_the_paged_attention():
    b = Batch(25, [300, 5, 77], [1, 4, 2], 8, 2, "f32")
    got = b.check()
    out = torch.full((b.rows, b.heads * D), -3.0, device="cuda")
    ws = torch.empty(ops.attention_paged_workspace(), dtype=torch.uint8, device="cuda")
    ops.attention_paged(_f(b.q), b.k, b.v, _i(b.table), _i(b.start), _i(b.ctx), b.max_new, out, ws)
    _, bound = b.want()
    assert (np.abs(_np(out) - got) <= 2 * bound).all()


def test_attention_refuses_a_small_workspace():
    b = Batch(27, [3], [1], 2, 1, "f32")
    n = ops.attention_shared_workspace(b.rows, b.heads)
    with pytest.raises(tie_b200.ModelError):
        b.call(ws=torch.empty(n - 16, dtype=torch.uint8, device="cuda"))


# ---- prefixes on the tensor cores

SCORES = 8_000_000                                         # from here on all formats' long prefixes go there


def _long(seed, ctx, new, heads, kv_heads, kind, groups, shared, **kw):
    """A batch whose prefixes go to the tensor cores: rows and the tables' width decide, not the positions there are."""
    b = Batch(seed, ctx, new, heads, kv_heads, kind, groups, shared, **kw)
    width = max(b.ptable.shape[1], -(-SCORES // (b.rows * heads * PAGE)))
    t = np.full((len(b.ptable), width), b.n_pages, np.int64)
    t[:, :b.ptable.shape[1]] = b.ptable
    b.ptable = t
    assert b.rows * heads // kv_heads >= 64 * len(b.ptable)
    return b


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 4), (8, 2), (6, 1)])
@pytest.mark.parametrize("n,new,groups,shared", [
    (64, 1, (0, 64), (1,)), (64, 1, (0, 64), (15,)), (65, 1, (0, 65), (64,)), (128, 1, (0, 128), (65,)), (43, 3, (0, 43), (700,)),
    (129, 1, (0, 129), (333,)), (150, 2, (0, 70, 150), (190, 127)), (200, 1, (3, 70, 70, 199), (16, 200, 129)),
])
def test_long_prefixes_match_the_definition(kind, heads, kv_heads, n, new, groups, shared):
    rng = np.random.default_rng(n + heads)
    _long(n, rng.integers(0, 20, n).tolist(), [new] * n, heads, kv_heads, kind, groups, shared, pad_rows=2).check()


@pytest.mark.parametrize("kind", KINDS)
def test_long_prefixes_of_many_steps(kind):
    """Items that several CTAs share, and CTAs that have several."""
    rng = np.random.default_rng(3)
    _long(1, [3] * 140, [1] * 140, 2, 2, kind, (0, 140), (12345,)).check()
    _long(2, rng.integers(0, 9, 700).tolist(), [1] * 700, 2, 1, kind, (0, 100, 310, 700), (900, 40, 1500)).check()


@pytest.mark.parametrize("kind", KINDS)
def test_long_prefixes_of_as_many_sequences_as_there_may_be(kind):
    """Lengths that leave shared memory for one CTA an SM, and groups of 64 to 192 rows."""
    rng = np.random.default_rng(6)
    cuts = np.sort(rng.choice(np.arange(1, 64), 31, replace=False)) * 64
    b = _long(3, rng.integers(0, 3, 4096).tolist(), [1] * 4096, 1, 1, kind, tuple([0] + cuts.tolist() + [4096]),
              tuple(rng.integers(0, 90, 32).tolist()))
    b.check()


@pytest.mark.parametrize("kind", KINDS)
def test_long_prefixes_with_holes(kind):
    """Pages that are not mapped, all of them, and lengths without meaning."""
    b = _long(5, [5] * 90, [1] * 90, 4, 2, kind, (0, 50, 90), (400, 77), unmapped=0.4)
    b.check()
    b.shared = np.array([0, 77])
    b.check()
    b.shared = np.array([400, 10 ** 8])
    b.check()
    b.shared, b.ctx = np.array([400, 77]), np.where(np.arange(90) % 7 == 0, 10 ** 6, b.ctx)
    b.check()
    b = _long(6, [0] * 70, [1] * 70, 4, 2, kind, (0, 70), (90,), unmapped=1.0)
    assert (b.check() == 0.0).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_long_prefixes_and_what_is_not_finite(kind, bad):
    """The rest of a last page, and pages of nobody, change nothing; a shared value makes its group's rows not finite."""
    n = 130
    b = _long(7, [2] * n, [1] * n, 2, 1, kind, (0, 65, n), (70, 33))
    before = b.check()
    used = np.zeros((b.n_pages, PAGE), bool)
    for entries, m in zip(list(b.table) + list(b.ptable), np.concatenate([b.ctx + b.new, b.shared])):
        for p in range(m):
            used[entries[p // PAGE], p % PAGE] = True
    for values in ([b.ksn, b.vsn] if kind == "q8" else [b.kn, b.vn]):
        if kind == "q8":
            np.moveaxis(values, 1, 2)[~used] = bad
        else:
            values[~used] = bad
    b.sync_pool()
    assert np.array_equal(b.check(), before)
    if kind == "q8":
        b.vsn[b.ptable[1, 2], :, 0] = bad
    else:
        b.vn[b.ptable[1, 2], 0] = bad
    b.sync_pool()
    got = _np(b.call())
    assert np.array_equal(got[:65], before[:65].astype(np.float32)) and not np.isfinite(got[65:]).any()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_long_prefixes_of_large_numbers(kind):
    b = _long(13, [4] * 70, [1] * 70, 4, 2, kind, (0, 70), (120,))
    b.vn[:] = np.where(b.rng.random(b.vn.shape) < 0.5, 3.3895314e38, np.float32(1e-38))
    b.sync_pool()
    assert np.isfinite(b.check()).all()
    _long(14, [4] * 70, [1] * 70, 4, 2, kind, (0, 70), (500,), q_spread=40.0).check()


@pytest.mark.parametrize("kind", KINDS)
def test_long_prefixes_captured(kind):
    """The same bits again, and a captured call that is replayed for other lengths; its status stays clear."""
    b = _long(15, [9] * 80, [1] * 80, 4, 2, kind, (0, 80), (1500,))
    first = b.call()
    assert torch.equal(b.call(), first)
    q, table, start, ctx = _f(b.q), _i(b.table), _i(b.start), _i(b.ctx)
    pt, pl, gs, status = _i(b.ptable), _i(b.shared), _i(b.groups), _i([0])
    out = torch.full((b.rows, 4 * D), -3.0, device="cuda")
    ws = torch.empty(ops.attention_shared_workspace(b.rows, 4), dtype=torch.uint8, device="cuda")
    args = dict(k_scales=b.ks, v_scales=b.vs, prefix_table=pt, prefix_lens=pl, group_start=gs, status=status)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attention_shared(q, b.k, b.v, table, start, ctx, 1, out, ws, **args)
        ops.attention_shared(q, b.k, b.v, table, start, ctx, 1, out, ws, **args)
    for n, c in ((1500, 9), (64, 3), (1, 0), (1499, 15)):
        b.shared, b.ctx = np.array([n]), np.full(80, c)
        pl.copy_(_i([n]))
        ctx.copy_(_i(b.ctx))
        graph.replay()
        torch.cuda.synchronize()
        o, bound = b.want()
        assert (np.abs(_np(out) - o) <= bound).all()
    assert int(status[0]) == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("long", [False, True])
def test_calls_one_after_another_see_each_others_results(kind, long):
    """Calls whose query is the result of the call before, with lengths that a copy changes between them, and one
    workspace: launched without a pause they give what they give one by one."""
    b = (_long(17, [9] * 70, [1] * 70, 4, 2, kind, (0, 70), (600,)) if long
         else Batch(18, [300, 20, 5], [1, 1, 1], 4, 2, kind, (0, 3), (90,)))
    lens = [b.shared - i for i in range(6)]

    def run(pause):
        rows = [_f(b.q)] + [torch.empty(b.rows, 4 * D, device="cuda") for _ in lens]
        table, start, ctx, pt, pl, gs = (_i(x) for x in (b.table, b.start, b.ctx, b.ptable, b.shared, b.groups))
        news = [_i(n) for n in lens]
        ws = torch.empty(ops.attention_shared_workspace(b.rows, 4), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        for i, n in enumerate(news):
            pl.copy_(n)
            ops.attention_shared(rows[i], b.k, b.v, table, start, ctx, 1, rows[i + 1], ws, k_scales=b.ks, v_scales=b.vs,
                                 prefix_table=pt, prefix_lens=pl, group_start=gs, scale=4.0)
            if pause:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        return rows[-1]

    one_by_one = run(True)
    for _ in range(4):
        assert torch.equal(run(False), one_by_one)


# ------------------------------------------------------------------ 4-bit weights

def _make(w, group):
    """packed, scales on the device."""
    n, k = w.shape
    (a, b), c = ops.q4_shapes(n, k, group)
    packed = torch.full((a, b), 0x5a, dtype=torch.uint8, device="cuda")
    scales = torch.full(c, 9.0, dtype=torch.bfloat16, device="cuda")
    ops.quantize_q4(w, packed, scales, group)
    return packed, scales


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,k,pad", [(1, 1, 0), (1, 128, 0), (3, 31, 1), (5, 33, 2), (17, 127, 0), (16, 129, 3), (33, 640, 0),
                                     (70, 1600, 4)])
def test_weights_are_made_and_read_back(group, n, k, pad):
    rng = np.random.default_rng(n * k + group)
    w = (0.02 * rng.standard_normal((n, k))).astype(np.float32)
    w[rng.random((n, k)) < 0.1] = 0.0
    wide = torch.full((n, k + pad), 7.0, device="cuda")
    wide[:, :k] = _f(w)
    packed, scales = _make(wide[:, :k], group)
    q, s = ref.quantize_q4(w, group)
    assert np.array_equal(_np(scales), s)
    assert np.array_equal(packed.cpu().numpy(), ref.pack_q4(q))
    back = torch.full((n, k + pad), 7.0, device="cuda")
    ops.dequantize_q4(packed, scales, group, back[:, :k])
    back = back.cpu().numpy()
    assert np.array_equal(back[:, :k], ref.weights(q, s, group).astype(np.float32)) and (back[:, k:] == 7.0).all()


def test_four_bit_levels_next_to_their_borders():
    f = np.float32
    rows = []
    for scale in (1.0, 2.0 ** -20, 2.0 ** 90, 0.3, 1e-3, 2.0 ** -126, 2.0 ** -130, 1e-44):
        half = np.tile((np.arange(-7, 9) - 0.5).astype(f), 2) * f(scale)
        for x in (half, np.nextafter(half, f(np.inf)), np.nextafter(half, f(-np.inf))):
            x = np.clip(x, -7 * f(scale), 7 * f(scale)).astype(f)
            x[3] = 7 * f(scale)
            rows.append(x)
    rows += [np.zeros(32, f), np.full(32, f(3.4028235e38)), np.full(32, f(-1e-45))]
    for bad in (np.inf, -np.inf, np.nan):
        x = np.ones(32, f)
        x[5] = bad
        rows.append(x)
    w = np.stack(rows)
    packed, scales = _make(_f(w), 32)
    q, s = ref.quantize_q4(w, 32)
    assert np.array_equal(_np(scales), s, equal_nan=True)
    assert np.array_equal(packed.cpu().numpy(), ref.pack_q4(q))


def _weights_of(rng, n, k, group):
    q = rng.integers(-7, 8, (n, k))
    s = ref.bf16(((0.5 + rng.random((n, -(-k // group)))) * 0.01).astype(np.float32))
    return (torch.tensor(ref.pack_q4(q), device="cuda"), torch.tensor(s, device="cuda").to(torch.bfloat16),
            ref.weights(q, s, group))


def _check_matvec(rng, rows, n, k, group, bias=False, residual=None, act=False, pad=0, offset=0):
    packed, scales, w = _weights_of(rng, n, k, group)
    x = rng.standard_normal((rows, k)).astype(np.float32)
    xd = torch.full((rows, offset + k + pad), float("nan"), device="cuda")    # what is not x is not read
    xd[:, offset:offset + k] = _f(x)
    b = (0.1 * rng.standard_normal(n)).astype(np.float32) if bias else None
    r = rng.standard_normal((rows, n)).astype(np.float32) if residual else None
    y = torch.full((rows, n + 3), -3.0, device="cuda")
    if residual == "in place":
        y[:, :n] = _f(r)
    rd = y[:, :n] if residual == "in place" else _f(r) if residual else None
    ops.matvec_q4(xd[:, offset:offset + k], packed, scales, group, y[:, :n], bias=None if b is None else _f(b), residual=rd,
                  gelu=act)
    want, bound = ref.matvec(x, w, b, r, act)
    got = y.cpu().numpy()
    assert (got[:, n:] == -3.0).all()
    off = np.abs(got[:, :n] - want)
    assert not (off > bound).any(), (off - bound).max()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows", [1, 2, 3, 7, 8, 9, 17])
@pytest.mark.parametrize("n,k", [(1, 1), (15, 33), (17, 128), (100, 129), (33, 1000), (40, 2100)])
def test_matvec_matches_the_definition(group, rows, n, k):
    _check_matvec(np.random.default_rng(rows + n), rows, n, k, group)


@pytest.mark.parametrize("rows", [1, 5])
@pytest.mark.parametrize("n,k", [(2500, 260), (5000, 130), (20000, 65)])
def test_matvec_of_many_outputs(rows, n, k):
    _check_matvec(np.random.default_rng(n), rows, n, k, 64)


@pytest.mark.parametrize("rows", [2, 6])
@pytest.mark.parametrize("epilogue", [dict(bias=True), dict(bias=True, act=True), dict(bias=True, residual="beside"),
                                      dict(bias=True, residual="in place"), dict(residual="beside", act=True)])
def test_matvec_epilogues(rows, epilogue):
    _check_matvec(np.random.default_rng(5), rows, 77, 300, 32, **epilogue)


@pytest.mark.parametrize("pad,offset", [(1, 0), (4, 0), (0, 1), (3, 4), (2, 2)])
def test_matvec_of_rows_that_lie_anywhere(pad, offset):
    _check_matvec(np.random.default_rng(6), 3, 40, 161, 64, pad=pad, offset=offset)
    _check_matvec(np.random.default_rng(7), 1, 40, 161, 64, pad=pad, offset=offset)


@pytest.mark.parametrize("rows", [2, 4])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_a_row_that_is_not_finite_is_so_alone(rows, bad):
    rng = np.random.default_rng(8)
    packed, scales, w = _weights_of(rng, 50, 200, 64)
    x = rng.standard_normal((rows, 200)).astype(np.float32)
    y = torch.empty(rows, 50, device="cuda")
    ops.matvec_q4(_f(x), packed, scales, 64, y)
    before = _np(y)
    x[1, 77] = bad
    ops.matvec_q4(_f(x), packed, scales, 64, y)
    got = _np(y)
    keep = np.arange(rows) != 1
    assert np.array_equal(got[keep], before[keep])
    assert not np.isfinite(got[1]).any()


def test_extreme_activations():
    """Sums of numbers of any size: the largest, the smallest, and both in a row."""
    rng = np.random.default_rng(9)
    packed, scales, w = _weights_of(rng, 30, 256, 128)
    for lo, hi in ((30, 37), (-36, -30), (-20, 20)):
        x = (rng.standard_normal((3, 256)) * 10.0 ** rng.uniform(lo, hi, (3, 256))).astype(np.float32)
        y = torch.empty(3, 30, device="cuda")
        ops.matvec_q4(_f(x), packed, scales, 128, y)
        want, bound = ref.matvec(x, w)
        assert (np.abs(_np(y) - want) <= bound + 1e-42).all()


@pytest.mark.parametrize("rows,k", [(8, 6016), (8, 6200), (3, 16384), (9, 16384)])
def test_matvec_of_long_rows(rows, k):
    """On both sides of the length from which two rows are taken at a time, and the longest."""
    _check_matvec(np.random.default_rng(k), rows, 37, k, 128, bias=True)


def test_matvec_limits():
    """As many rows as there may be; one more, or a longer row, is refused."""
    rng = np.random.default_rng(3)
    packed, scales, w = _weights_of(rng, 2, 5, 32)
    x = _f(rng.standard_normal((131070, 5)))
    y = torch.empty(131070, 2, device="cuda")
    ops.matvec_q4(x, packed, scales, 32, y)
    want, bound = ref.matvec(_np(x), w)
    assert (np.abs(_np(y) - want) <= bound).all()
    with pytest.raises(tie_b200.ModelError):
        ops.matvec_q4(torch.zeros(131071, 5, device="cuda"), packed, scales, 32, torch.empty(131071, 2, device="cuda"))
    packed, scales, _ = _weights_of(rng, 2, 16385, 64)
    with pytest.raises(tie_b200.ModelError):
        ops.matvec_q4(torch.zeros(1, 16385, device="cuda"), packed, scales, 64, torch.empty(1, 2, device="cuda"))


def test_products_one_after_another():
    """A chain of products, each of the result of the one before, and weights made between them: without a pause as
    one by one; on two streams at once as on one."""
    rng = np.random.default_rng(4)
    n = 384
    ws = [_f(0.05 * rng.standard_normal((n, n))) for _ in range(5)]
    x0 = _f(rng.standard_normal((4, n)))

    def run(pause, stream=None):
        x, packed, scales = x0, torch.empty(n, n // 2, dtype=torch.uint8, device="cuda"), torch.empty(n, n // 64, dtype=torch.bfloat16, device="cuda")
        ys = [torch.empty(4, n, device="cuda") for _ in ws]
        for w, y in zip(ws, ys):
            ops.quantize_q4(w, packed, scales, 64, stream=stream)
            ops.matvec_q4(x, packed, scales, 64, y, residual=x, gelu=True, stream=stream)
            x = y
            if pause:
                torch.cuda.synchronize()
        return x

    want = run(True)
    torch.cuda.synchronize()
    for _ in range(4):
        assert torch.equal(run(False), want)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(4):
        for st in streams:
            with torch.cuda.stream(st):
                outs.append(run(False))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("rows", [3, 12])
def test_a_decode_layer_of_answers_to_one_prompt(rows):
    """The attention half of a decode step: 4-bit projection, the new rows into the 8-bit cache by the page plan, attention
    over the shared prompt and the answers' own pages, 4-bit projection added to the residual stream. Each step's
    result is held to the definition applied to what the step before it gave."""
    rng = np.random.default_rng(rows)
    heads, E, shared = 4, 256, 75
    ctx = rng.integers(0, 50, rows)
    need = [-(-(c + 1) // PAGE) for c in ctx]
    have = [-(-c // PAGE) for c in ctx]
    first = -(-shared // PAGE)
    n_pages = sum(need) + first + 3
    perm = rng.permutation(n_pages)
    table = np.full((rows, max(need) + 1), -1, np.int64)
    at = first
    for s, m in enumerate(have):
        table[s, :m] = perm[at:at + m]
        at += m
    free = perm[at:]
    (k, ks, kn, ksn), (v, vs, vn, vsn) = _pool(rng, n_pages, heads, "q8")
    wq = _make(_f(0.05 * rng.standard_normal((3 * E, E))), 64)
    wp = _make(_f(0.05 * rng.standard_normal((E, E))), 32)
    bq, bp = (_f(0.1 * rng.standard_normal(m)) for m in (3 * E, E))
    x = _f(rng.standard_normal((rows, E)))
    resid = _f(rng.standard_normal((rows, E)))
    qkv, out = torch.empty(rows, 3 * E, device="cuda"), torch.empty(rows, E, device="cuda")
    y = resid.clone()
    t, start = _i(table), torch.empty(rows + 1, dtype=I32, device="cuda")
    seq_of, pos_of, slots, status = (torch.empty(m, dtype=I32, device="cuda") for m in (rows, rows, rows, 1))
    n_free = _i([len(free)])
    ws = torch.empty(ops.attention_shared_workspace(rows, heads), dtype=torch.uint8, device="cuda")
    ops.page_plan(_i(ctx), _i([1] * rows), t, n_pages, start, seq_of, pos_of, slots, status, free_pages=_i(free),
                  n_free=n_free, n_free_out=n_free)
    ops.matvec_q4(x, *wq, 64, qkv, bias=bq)
    ops.kv_store_q8(qkv[:, E:2 * E], qkv[:, 2 * E:], slots, k, v, ks, vs)
    ops.attention_shared(qkv[:, :E], k, v, t, start, _i(ctx), 1, out, ws, k_scales=ks, v_scales=vs,
                         prefix_table=_i(perm[None, :first]), prefix_lens=_i([shared]), group_start=_i([0, rows]))
    ops.matvec_q4(out, *wp, 32, y, bias=bp, residual=y)
    torch.cuda.synchronize()
    assert int(status[0]) == 0

    def back(packed, scales, group, n, kk):
        w = torch.empty(n, kk, device="cuda")
        ops.dequantize_q4(packed, scales, group, w)
        return _np(w).astype(np.float64)

    want, bound = ref.matvec(_np(x), back(*wq, 64, 3 * E, E), _np(bq).astype(np.float64))
    assert (np.abs(_np(qkv) - want) <= bound).all()
    slot = _np(slots)
    new = _np(qkv)
    kn, ksn = ref.store_q8(new[:, E:2 * E], slot, kn, ksn)
    vn, vsn = ref.store_q8(new[:, 2 * E:], slot, vn, vsn)
    assert np.array_equal(_np(k), kn) and np.array_equal(_np(vs), vsn)
    o, vmax, smax = ref.attention(new[:, :E], kn, vn, _np(t), _np(start), ctx, heads, 0.125, np.zeros((rows, E)), 1, ksn, vsn,
                                  perm[None, :first], [shared], [0, rows])
    assert (np.abs(_np(out) - o) <= paged.attention_bound(vmax, smax, shared + 51)).all()
    want, bound = ref.matvec(_np(out), back(*wp, 32, E, E), _np(bp).astype(np.float64), _np(resid).astype(np.float64))
    assert (np.abs(_np(y) - want) <= bound).all()


def test_operators_run_on_the_stream_given():
    """On a side stream behind work that is still running there, without waiting for it."""
    rng = np.random.default_rng(31)
    packed, scales, w = _weights_of(rng, 64, 128, 64)
    x = rng.standard_normal((2, 128)).astype(np.float32)
    xd, y = torch.zeros(2, 128, device="cuda"), torch.empty(2, 64, device="cuda")
    src = _f(x)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        torch.cuda._sleep(10 ** 7)
        xd.copy_(src)
    ops.matvec_q4(xd, packed, scales, 64, y, stream=st.cuda_stream)
    st.synchronize()
    want, bound = ref.matvec(x, w)
    assert (np.abs(_np(y) - want) <= bound).all()


@pytest.mark.parametrize("rows", [1, 9])
def test_a_captured_decode_step(rows):
    """Projection, store, attention and projection in one graph, replayed over new rows and lengths: as the calls one by one."""
    rng = np.random.default_rng(rows)
    heads, E, steps = 2, 128, 20
    pages = -(-steps // PAGE) * rows
    (k, ks, _, _), (v, vs, _, _) = _pool(rng, pages, heads, "q8")
    pools = [k, ks, v, vs]
    wq, wp = _make(_f(0.05 * rng.standard_normal((3 * E, E))), 64), _make(_f(0.05 * rng.standard_normal((E, E))), 32)
    table, start = _i(np.arange(pages).reshape(rows, -1)), _i(np.arange(rows + 1))
    base = _i(np.arange(rows) * (pages // rows) * PAGE)
    ctx = torch.zeros(rows, dtype=I32, device="cuda")
    x = torch.zeros(rows, E, device="cuda")
    qkv, out, y = torch.empty(rows, 3 * E, device="cuda"), torch.empty(rows, E, device="cuda"), torch.empty(rows, E, device="cuda")
    slots = torch.empty(rows, dtype=I32, device="cuda")
    ws = torch.empty(ops.attention_shared_workspace(rows, heads), dtype=torch.uint8, device="cuda")

    def step(pause):
        calls = [lambda: torch.add(base, ctx, out=slots), lambda: ops.matvec_q4(x, *wq, 64, qkv),
                 lambda: ops.kv_store_q8(qkv[:, E:2 * E], qkv[:, 2 * E:], slots, k, v, ks, vs),
                 lambda: ops.attention_shared(qkv[:, :E], k, v, table, start, ctx, 1, out, ws, k_scales=ks, v_scales=vs),
                 lambda: ops.matvec_q4(out, *wp, 32, y, residual=x), lambda: x.copy_(y), lambda: ctx.add_(1)]
        for call in calls:
            call()
            if pause:
                torch.cuda.synchronize()

    first = _f(rng.standard_normal((rows, E)))
    at_start = [p.clone() for p in pools]

    def reset():
        for p, q in zip(pools, at_start):
            p.copy_(q)
        x.copy_(first)
        ctx.zero_()

    reset()
    want = []
    for _ in range(steps):
        step(True)
        want.append(y.clone())
    kept = [p.clone() for p in pools]
    reset()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(False)
    reset()
    for i in range(steps):
        graph.replay()
        assert torch.equal(y, want[i])
    assert all(torch.equal(p, q) for p, q in zip(pools, kept))


def test_calls_of_two_threads():
    """Attention and products from two threads at once, each on a stream of its own, with one set of pages and weights."""
    import threading
    rng = np.random.default_rng(33)
    b = [Batch(34, [400, 20], [1, 1], 4, 2, "q8", (0, 2), (500,)), _long(35, [9] * 70, [1] * 70, 4, 2, "f32", (0, 70), (300,))]
    packed, scales, _ = _weights_of(rng, 500, 256, 64)
    want = []
    for x in b:
        o = x.call()
        y = torch.empty(x.rows, 500, device="cuda")
        ops.matvec_q4(o, packed, scales, 64, y)
        want.append(y)
    torch.cuda.synchronize()
    wrong = []

    def work(x, y0):
        st = torch.cuda.Stream()
        try:
            with torch.cuda.stream(st):
                for _ in range(20):
                    o, y = x.call(), torch.empty(x.rows, 500, device="cuda")
                    ops.matvec_q4(o, packed, scales, 64, y)
                    st.synchronize()
                    if not torch.equal(y, y0):
                        wrong.append(x.kind)
        except Exception as e:                 # noqa: BLE001
            wrong.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(b, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[:3]
