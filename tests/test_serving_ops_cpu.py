"""What the 8-bit cache, attention over shared positions and the 4-bit weights refuse before any device work (no GPU
needed), the checks of their Python binding, and the layout of packed weights."""
import os
import sys

import numpy as np
import pytest

import tie_b200
from tie_b200 import ops

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import serving_oracle as ref  # noqa: E402

L = tie_b200.library()
OK, CAPACITY, ARG, DEVICE = (tie_b200.MODEL_STATUS.index(s) for s in
                             ("MODEL_OK", "MODEL_ERR_CAPACITY", "MODEL_ERR_ARG", "MODEL_ERR_DEVICE"))
P = 0x10000000   # an address that nothing here follows: every call below ends before device work
BAD = P + 4      # not 16-byte aligned
INT8 = 2


def _call(fn, order, **changed):
    a = dict(order)
    assert set(changed) <= set(a)
    a.update(changed)
    return fn(*a.values())


STORE = dict(k=P, v=P, ld=128, slots=P, rows=3, k_pages=P, v_pages=P, k_scales=P, v_scales=P, n_pages=8, kv_heads=2,
             stream=None)
LOAD = dict(slots=P, rows=3, k_pages=P, v_pages=P, k_scales=P, v_scales=P, fmt=INT8, n_pages=8, kv_heads=2, k=P, v=P, ld=128,
            stream=None)
ATTN = dict(q=P, ldq=256, heads=4, k=P, v=P, k_scales=P, v_scales=P, fmt=INT8, n_pages=8, kv_heads=2, table=P, width=4,
            row_start=P, ctx=P, n_seq=2, max_new=3, rows=5, ptable=P, pwidth=3, plen=P, gstart=P, n_group=1, scale=0.125,
            out=P, ldo=256, ws=P, ws_bytes=1 << 40, status=None, stream=None)
MAKE = dict(w=P, ldw=100, n=7, k=100, group=64, packed=P, scales=P, stream=None)
BACK = dict(packed=P, scales=P, n=7, k=100, group=64, w=P, ldw=100, stream=None)
MATVEC = dict(x=P, ldx=100, rows=2, packed=P, scales=P, n=7, k=100, group=64, bias=P, residual=P, ldr=7, gelu=0, y=P, ldy=7,
              stream=None)


@pytest.mark.parametrize("changed", [{k: None} for k in ("k", "v", "slots", "k_pages", "v_pages", "k_scales", "v_scales")] + [
    {k: BAD} for k in ("k", "v", "k_pages", "v_pages", "k_scales", "v_scales")] + [
    dict(ld=124), dict(ld=130), dict(rows=-1), dict(n_pages=0), dict(kv_heads=0), dict(kv_heads=1025),
    dict(n_pages=(1 << 27) + 1)])
def test_store_refuses(changed):
    assert _call(L.tie_kv_store_q8, STORE, **changed) == ARG


@pytest.mark.parametrize("changed", [{k: None} for k in ("k", "v", "slots", "k_pages", "v_pages", "k_scales", "v_scales")] + [
    {k: BAD} for k in ("k", "v", "k_pages", "v_pages", "k_scales", "v_scales")] + [
    dict(ld=124), dict(ld=130), dict(rows=-1), dict(fmt=3), dict(fmt=-1), dict(fmt=0), dict(fmt=1, k_scales=None),
    dict(n_pages=0), dict(kv_heads=0)])
def test_load_refuses(changed):
    assert _call(L.tie_kv_load, LOAD, **changed) == ARG


@pytest.mark.parametrize("changed", [{k: None} for k in ("q", "k", "v", "k_scales", "v_scales", "table", "row_start", "ctx", "out",
                                                         "ws", "ptable", "plen", "gstart")] + [
    {k: BAD} for k in ("q", "k", "v", "k_scales", "v_scales", "out", "ws")] + [
    dict(k=P + 16), dict(heads=3), dict(heads=0), dict(heads=8196, kv_heads=4, ldq=8196 * 64, ldo=8196 * 64), dict(ldq=252),
    dict(ldo=252), dict(ldq=258), dict(ldo=258), dict(width=0), dict(n_seq=0), dict(max_new=-1), dict(rows=-1),
    dict(scale=float("nan")), dict(scale=float("inf")), dict(fmt=3), dict(fmt=0), dict(fmt=1, v_scales=None), dict(n_pages=0),
    dict(kv_heads=0), dict(n_group=-1), dict(n_group=0), dict(pwidth=0)])
def test_attention_refuses(changed):
    assert _call(L.tie_attention_shared, ATTN, **changed) == ARG


@pytest.mark.parametrize("changed", [dict(n_seq=4097), dict(n_group=4097), dict(width=1 << 27), dict(pwidth=1 << 27),
                                     dict(rows=(1 << 30) // 4)])
def test_attention_limits(changed):
    assert _call(L.tie_attention_shared, ATTN, **changed) == CAPACITY
    assert L.tie_attention_shared_workspace(-1, 4) == 0 and L.tie_attention_shared_workspace(3, 0) == 0


@pytest.mark.parametrize("changed", [{k: None} for k in ("w", "packed", "scales")] + [
    dict(w=P + 2), dict(packed=BAD), dict(scales=P + 1), dict(n=0), dict(k=0), dict(group=16), dict(group=100), dict(ldw=99)])
def test_four_bit_weights_refuse(changed):
    assert _call(L.tie_quantize_q4, MAKE, **changed) == ARG
    assert _call(L.tie_dequantize_q4, BACK, **changed) == ARG


@pytest.mark.parametrize("changed", [{k: None} for k in ("x", "y", "packed", "scales")] + [
    {k: P + 2} for k in ("x", "y", "bias", "residual")] + [
    dict(packed=BAD), dict(scales=P + 1), dict(n=0), dict(k=0), dict(group=48), dict(ldx=99), dict(ldy=6), dict(ldr=6),
    dict(rows=-1), dict(gelu=2)])
def test_matvec_refuses(changed):
    assert _call(L.tie_matvec_q4, MATVEC, **changed) == ARG


def test_limits_of_four_bit_weights():
    big = (1 << 24) + 1
    assert _call(L.tie_quantize_q4, MAKE, k=big, ldw=big) == CAPACITY
    assert _call(L.tie_dequantize_q4, BACK, n=2 ** 31 - 1, k=1 << 20, ldw=1 << 20) == CAPACITY
    assert _call(L.tie_matvec_q4, MATVEC, k=big, ldx=big) == CAPACITY
    assert _call(L.tie_matvec_q4, MATVEC, rows=8 * 65535 + 1) == CAPACITY
    assert L.tie_q4_bytes(3, 128) == 192 and L.tie_q4_bytes(3, 129) == 384 and L.tie_q4_bytes(50257, 1600) == 50257 * 13 * 64
    assert L.tie_q4_bytes(0, 5) == 0 and L.tie_q4_bytes(5, 0) == 0 and L.tie_q4_bytes(2 ** 31 - 1, 2 ** 31 - 1) == (2 ** 31 - 1) * 2 ** 30


def test_no_rows_is_no_work():
    assert _call(L.tie_kv_store_q8, STORE, rows=0, k=None, v=None, slots=None) == OK
    assert _call(L.tie_kv_load, LOAD, rows=0, k=None, v=None, slots=None) == OK
    assert _call(L.tie_attention_shared, ATTN, rows=0, q=None, out=None) == OK
    assert _call(L.tie_attention_shared, ATTN, max_new=0) == OK
    assert _call(L.tie_matvec_q4, MATVEC, rows=0, x=None, y=None) == OK


def test_binding_checks_shapes_and_types():
    """What the C entry points cannot see (tensors on the CPU: refused before any call)."""
    import torch
    pages, levels = torch.zeros(4, 16, 128), torch.zeros(4, 16, 128, dtype=torch.int8)
    scales = torch.zeros(4, 2, 16)
    ints = torch.zeros(8, dtype=torch.int32)
    table = torch.zeros(2, 2, dtype=torch.int32)
    rows = torch.zeros(5, 128)
    w, packed, ws = torch.zeros(5, 100), torch.zeros(5, 64, dtype=torch.uint8), torch.zeros(5, 2, dtype=torch.bfloat16)
    bad = [
        lambda: ops.kv_store_q8(rows, rows, ints, pages, pages, scales, scales),
        lambda: ops.kv_store_q8(rows, rows, ints, levels, levels, scales[:, :1], scales),
        lambda: ops.kv_store_q8(rows, rows, ints, levels, levels, None, None),
        lambda: ops.kv_store_q8(rows, rows[:4], ints, levels, levels, scales, scales),
        lambda: ops.kv_store(rows, rows, ints, levels, levels),
        lambda: ops.kv_load(ints[:5], pages, pages, rows, rows.clone(), scales, scales),
        lambda: ops.kv_load(ints[:5], levels, levels, rows, rows.clone()),
        lambda: ops.kv_load(ints[:5], pages, pages, rows, rows.clone().half()),
        lambda: ops.attention_shared(rows, levels, levels, table, ints, ints, 1, rows.clone(), rows),
        lambda: ops.attention_shared(rows, pages, pages, table, ints, ints, 1, rows.clone(), rows, prefix_lens=ints),
        lambda: ops.attention_shared(rows, pages, pages, table, ints, ints, 1, rows.clone(), rows, prefix_table=table),
        lambda: ops.attention_shared(rows, pages, pages, table, ints, ints, 1, rows.clone(), ints, status=ints.long()),
        lambda: ops.attention_shared(rows, pages, pages, table, ints, ints, 1, rows.clone(), ints, status=ints[:0]),
        lambda: ops.attention_paged(rows, levels, levels, table, ints, ints, 1, rows.clone(), rows),
        lambda: ops.quantize_q4(w, packed, ws, 48),
        lambda: ops.quantize_q4(w, packed[:, :32], ws, 64),
        lambda: ops.quantize_q4(w[:4], packed, ws, 64),
        lambda: ops.quantize_q4(w, packed, ws.float(), 64),
        lambda: ops.dequantize_q4(packed, ws, 32, w),
        lambda: ops.dequantize_q4(packed, ws, 64, w.double()),
        lambda: ops.matvec_q4(w, packed, ws, 64, torch.zeros(4, 5)),
        lambda: ops.matvec_q4(w, packed, ws, 64, torch.zeros(5, 5), bias=torch.zeros(4)),
        # all well but for the device
        lambda: ops.kv_store_q8(rows, rows, ints, levels, levels.clone(), scales, scales.clone()),
        lambda: ops.quantize_q4(w, packed, ws, 64),
        lambda: ops.matvec_q4(w, packed, ws, 64, torch.zeros(5, 5)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")


def test_host_memory_is_refused():
    """Without a device the call reports that; with one, memory the device does not own is refused."""
    import torch
    t, s = torch.zeros(4, 16, 128), torch.zeros(4, 2, 16)
    slots = torch.zeros(2, dtype=torch.int32)
    want = ARG if torch.cuda.is_available() else DEVICE
    assert L.tie_kv_store_q8(t.data_ptr(), t.data_ptr(), 128, slots.data_ptr(), 2, t.data_ptr(), t.data_ptr(), s.data_ptr(),
                             s.data_ptr(), 4, 2, 0) == want
    assert L.tie_quantize_q4(t.data_ptr(), 128, 2, 128, 64, t.data_ptr(), s.data_ptr(), 0) == want
    assert L.tie_matvec_q4(t.data_ptr(), 128, 2, t.data_ptr(), s.data_ptr(), 4, 128, 64, 0, 0, 0, 0, t.data_ptr(), 4, 0) == want


def test_definitions_agree_with_one_another():
    """The packed layout, read back as the header states it, and levels next to a border."""
    rng = np.random.default_rng(0)
    q = rng.integers(-7, 8, (3, 300))
    word = ref.pack_q4(q).view(np.uint32).reshape(3, 3, 16)
    for c in (0, 7, 8, 31, 32, 127, 128, 299):
        b, r = divmod(c, 128)
        assert ((word[:, b, 4 * (r % 32 // 8) + r // 32] >> (4 * (r % 8)) & 15).astype(int) - 8 == q[:, c]).all()
    x = np.array([[127.0, 0.5, 1.5, -2.5, np.nextafter(np.float32(0.5), np.float32(1)), 126.49999]], np.float32)
    levels, scale = ref.levels(x, 127)
    assert scale[0] == 1.0 and levels[0].tolist() == [127, 0, 2, -2, 1, 126]
