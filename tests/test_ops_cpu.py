"""What the operators over device memory refuse before any device work (no GPU needed), and the
checks of their Python binding."""
import pytest

import tie_b200
from tie_b200 import ops

L = tie_b200.library()
OK, CAPACITY, ARG, DEVICE = (tie_b200.MODEL_STATUS.index(s) for s in
                             ("MODEL_OK", "MODEL_ERR_CAPACITY", "MODEL_ERR_ARG", "MODEL_ERR_DEVICE"))
P = 0x10000000   # an address that nothing here follows: every call below ends before device work
BAD = P + 4      # not 16-byte aligned


def _call(fn, order, **changed):
    a = dict(order)
    assert set(changed) <= set(a)
    a.update(changed)
    return fn(*a.values())


PLAN = dict(ctx=P, new=P, n_seq=2, table=P, width=4, n_pages=8, free=P, max_free=8, n_free=P, n_free_out=P, row_start=P,
            seq_of=P, pos_of=P, slot_of=P, max_rows=16, status=P, stream=None)
STORE = dict(k=P, v=P, ld=128, slots=P, rows=3, k_pages=P, v_pages=P, fmt=0, n_pages=8, kv_heads=2, stream=None)
ATTN = dict(q=P, ldq=256, heads=4, k=P, v=P, fmt=0, n_pages=8, kv_heads=2, table=P, width=4, row_start=P, ctx=P, n_seq=2,
            max_new=3, rows=5, scale=0.125, out=P, ldo=256, ws=P, ws_bytes=1 << 30, status=None, stream=None)
SELECT = dict(logits=P, ldl=100, scores=P, done=P, n_req=2, beams=4, vocab=100, eos=7, next=P, parent=P, scores_out=P,
              done_out=P, ws=P, ws_bytes=1 << 30, stream=None)
REORDER = dict(k=P, v=P, fmt=0, layers=2, stride=8 * 16 * 128, n_pages=8, kv_heads=2, table=P, width=4, parent=P, first=P,
               length=P, n_req=2, beams=4, stream=None)


@pytest.mark.parametrize("changed", [
    {k: None} for k in ("ctx", "new", "table", "row_start", "seq_of", "pos_of", "slot_of", "status", "n_free", "n_free_out")
] + [dict(n_seq=0), dict(width=0), dict(n_pages=0), dict(max_rows=0), dict(max_free=-1), dict(free=None)])
def test_plan_refuses(changed):
    assert _call(L.tie_page_plan, PLAN, **changed) == ARG


@pytest.mark.parametrize("changed", [dict(n_seq=4097), dict(n_pages=(1 << 27) + 1), dict(width=1 << 27)])
def test_plan_limits(changed):
    assert _call(L.tie_page_plan, PLAN, **changed) == CAPACITY


@pytest.mark.parametrize("changed", [{k: None} for k in ("k", "v", "slots", "k_pages", "v_pages")] + [
    {k: BAD} for k in ("k", "v", "k_pages", "v_pages")] + [
    dict(ld=124), dict(ld=130), dict(rows=-1), dict(fmt=2), dict(fmt=-1), dict(n_pages=0), dict(kv_heads=0),
    dict(kv_heads=1025), dict(n_pages=(1 << 27) + 1)])
def test_store_refuses(changed):
    assert _call(L.tie_kv_store, STORE, **changed) == ARG


def test_no_rows_is_no_work():
    assert _call(L.tie_kv_store, STORE, rows=0) == OK
    assert _call(L.tie_attention_paged, ATTN, rows=0) == OK
    assert _call(L.tie_attention_paged, ATTN, max_new=0) == OK
    assert _call(L.tie_kv_reorder, REORDER, beams=1) == OK


@pytest.mark.parametrize("changed", [{k: None} for k in ("q", "k", "v", "table", "row_start", "ctx", "out", "ws")] + [
    {k: BAD} for k in ("q", "k", "v", "out", "ws")] + [
    dict(heads=3), dict(heads=0), dict(heads=8196, kv_heads=4, ldq=8196 * 64, ldo=8196 * 64), dict(ldq=252), dict(ldo=252),
    dict(ldq=258), dict(ldo=258), dict(width=0), dict(n_seq=0), dict(max_new=-1), dict(rows=-1), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(fmt=2), dict(n_pages=0), dict(kv_heads=0)])
def test_attention_refuses(changed):
    assert _call(L.tie_attention_paged, ATTN, **changed) == ARG


@pytest.mark.parametrize("changed", [dict(n_seq=4097), dict(width=1 << 27), dict(rows=(1 << 30) // 4)])
def test_attention_limits(changed):
    assert _call(L.tie_attention_paged, ATTN, **changed) == CAPACITY


@pytest.mark.parametrize("changed", [{k: None} for k in ("logits", "scores", "next", "parent", "scores_out", "ws")] + [
    dict(n_req=0), dict(beams=0), dict(vocab=0), dict(ldl=99), dict(eos=100), dict(eos=-1), dict(eos=-1, done=None), dict(ws=BAD)])
def test_select_refuses(changed):
    assert _call(L.tie_beam_select, SELECT, **changed) == ARG


@pytest.mark.parametrize("changed", [dict(beams=17), dict(n_req=4097), dict(vocab=(1 << 30) + 1, ldl=(1 << 30) + 1)])
def test_select_limits(changed):
    assert _call(L.tie_beam_select, SELECT, **changed) == CAPACITY
    assert L.tie_beam_select_workspace(1, 17, 100) == 0 and L.tie_beam_select_workspace(0, 4, 100) == 0


@pytest.mark.parametrize("changed", [{k: None} for k in ("k", "v", "table", "parent", "first", "length")] + [
    dict(k=BAD), dict(v=BAD), dict(fmt=3), dict(layers=0), dict(n_pages=0), dict(kv_heads=0), dict(width=0), dict(n_req=0),
    dict(beams=0), dict(stride=8 * 16 * 128 - 4), dict(stride=8 * 16 * 128 + 1)])
def test_reorder_refuses(changed):
    assert _call(L.tie_kv_reorder, REORDER, **changed) == ARG


@pytest.mark.parametrize("changed", [dict(beams=17), dict(n_req=4097), dict(width=1 << 27), dict(n_req=4096, width=1 << 20)])
def test_reorder_limits(changed):
    assert _call(L.tie_kv_reorder, REORDER, **changed) == CAPACITY


def test_binding_checks_shapes_and_types():
    """What the C entry points cannot see (tensors on the CPU: refused before any call)."""
    import torch
    pages = torch.zeros(4, 16, 128)
    ints = torch.zeros(8, dtype=torch.int32)
    table = torch.zeros(2, 2, dtype=torch.int32)
    rows = torch.zeros(5, 128)
    with pytest.raises(ValueError):
        ops.kv_store(rows, rows, ints, pages, pages[:, :8])                    # not whole pages
    with pytest.raises(ValueError):
        ops.kv_store(rows, rows, ints, pages.double(), pages.double())         # no such format
    with pytest.raises(ValueError):
        ops.kv_store(rows, rows.half(), ints, pages, pages)
    with pytest.raises(ValueError):
        ops.kv_store(rows, rows[:4], ints, pages, pages)
    with pytest.raises(ValueError):
        ops.kv_store(rows, rows, ints[:4], pages, pages)                       # fewer slots than rows
    with pytest.raises(ValueError):
        ops.kv_store(rows, rows, ints.long(), pages, pages)
    with pytest.raises(ValueError):
        ops.attention_paged(rows, pages, pages, table.T, ints, ints, 1, rows.clone(), rows)
    with pytest.raises(ValueError):
        ops.attention_paged(rows, pages, pages, table, ints[:2], ints, 1, rows.clone(), rows)
    with pytest.raises(ValueError):
        ops.attention_paged(rows.T, pages, pages, table, ints, ints, 1, rows.T, rows)
    with pytest.raises(ValueError):
        ops.beam_select(rows, ints.float(), 2, ints, ints, ints.float(), rows)  # 5 rows are not pairs
    with pytest.raises(ValueError):
        ops.kv_reorder(pages, pages.clone(), torch.zeros(3, 2, dtype=torch.int32), ints, ints, ints, 2)
    with pytest.raises(ValueError):
        ops.page_plan(ints, ints, table, 4, ints[:2], ints, ints, ints, ints)
    with pytest.raises(ValueError):                                            # all well but for the device
        ops.kv_store(rows, rows, ints, pages, pages.clone())
    with pytest.raises(ValueError):
        ops.page_plan(ints, ints, table, 4, ints, ints, ints, ints, ints)


def test_host_memory_is_refused():
    """Without a device the call reports that; with one, memory the device does not own is refused."""
    import torch
    t = torch.zeros(4, 16, 128)
    slots = torch.zeros(2, dtype=torch.int32)
    rc = L.tie_kv_store(t.data_ptr(), t.data_ptr(), 128, slots.data_ptr(), 2, t.data_ptr(), t.data_ptr(), 0, 4, 2, 0)
    assert rc == (ARG if torch.cuda.is_available() else DEVICE)
