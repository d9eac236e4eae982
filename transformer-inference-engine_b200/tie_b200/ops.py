"""The operators over device memory (``include/tie_b200.h``): page plans, K/V row
stores, attention over the paged cache, beam selection and cache reordering.

Arguments are torch tensors on a CUDA device. Outputs and workspaces are the
caller's; nothing is allocated or waited for. Work runs on ``stream`` (a
``cudaStream_t`` as an int), by default torch's current stream of the tensors'
device. Shapes, types and layouts that the C entry points cannot see are
checked here (``ValueError``); their own refusals raise ``ModelError``.

The sizes of a page pool come from its tensors: ``k_pages`` and ``v_pages`` are
[n_pages, 16, n_kv_head * 64] (``kv_reorder`` also takes
[n_layer, n_pages, 16, n_kv_head * 64]), float32 or bfloat16, contiguous.
"""
from __future__ import annotations

import torch

from .lib import TIE_KV_BF16, TIE_KV_F32, ModelError, library

PAGE_ROWS = 16
HEAD_DIM = 64

_INT, _F32, _BF16 = torch.int32, torch.float32, torch.bfloat16
# torch's current stream of a device as an integer; the public call builds a
# Stream object first (2.3 us against 0.1 us)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda device: torch.cuda.current_stream(device).cuda_stream)


def _chk(rc, where):
    if rc:
        raise ModelError(rc, where)


def _wrong(name, what):
    raise ValueError(f"{name}: {what} is wanted")


def _ints(name, t, n, device):
    """The address of a contiguous int32 tensor of at least n elements on `device` (None stays None)."""
    if t is None:
        return None
    if t.dtype is not _INT or t.numel() < n or t.get_device() != device or not t.is_contiguous():
        _wrong(name, f"a contiguous int32 tensor of {n} elements on device {device}")
    return t.data_ptr()


def _floats(name, t, n, device):
    if t.dtype is not _F32 or t.numel() < n or t.get_device() != device or not t.is_contiguous():
        _wrong(name, f"a contiguous float32 tensor of {n} elements on device {device}")
    return t.data_ptr()


def _rows(name, t, width, device):
    """A float32 matrix of `width` columns whose rows are contiguous: (address, leading dimension)."""
    if t.dtype is not _F32 or t.dim() != 2 or t.get_device() != device:
        _wrong(name, f"a float32 matrix on device {device}")
    n, w = t.shape
    ld, one = t.stride()
    if w != width or (one != 1 and w > 1):
        _wrong(name, f"[rows, {width}] with contiguous rows")
    return t.data_ptr(), ld if n > 1 else max(ld, width)


def _pool(k, v):
    """(format, n_pages, n_kv_head, layers, layer stride, device) of a pool's two tensors."""
    shape, dtype, device = k.shape, k.dtype, k.get_device()
    if device < 0 or v.shape != shape or v.dtype is not dtype or v.get_device() != device or not (k.is_contiguous() and v.is_contiguous()):
        _wrong("k_pages and v_pages", "one shape, type and CUDA device, contiguous,")
    if dtype is _F32:
        fmt = TIE_KV_F32
    elif dtype is _BF16:
        fmt = TIE_KV_BF16
    else:
        _wrong("k_pages, v_pages", "float32 or bfloat16")
    if len(shape) == 3:
        layers, (n_pages, rows, w) = 1, shape
    elif len(shape) == 4:
        layers, n_pages, rows, w = shape
    else:
        rows = 0
    if rows != PAGE_ROWS or w % HEAD_DIM:
        _wrong("k_pages, v_pages", f"[n_pages, {PAGE_ROWS}, n_kv_head * {HEAD_DIM}]")
    return fmt, n_pages, w // HEAD_DIM, layers, n_pages * PAGE_ROWS * w, device


def _table(t, device):
    if t.dtype is not _INT or t.dim() != 2 or not t.is_contiguous() or t.get_device() != device or device < 0:
        _wrong("page_table", f"a contiguous int32 [n_seq, pages_per_seq] on device {device}")
    return t.shape


def _workspace(t, device):
    if not t.is_contiguous() or t.get_device() != device:
        _wrong("workspace", f"a contiguous tensor on device {device}")
    return t.data_ptr(), t.numel() * t.element_size()


def page_plan(ctx_lens, new_lens, page_table, n_pages, row_start, seq_of, pos_of, slot_of, status, free_pages=None,
              n_free=None, n_free_out=None, stream=None):
    """Assigns pages to new positions and writes row starts and slot maps (tie_page_plan)."""
    d = page_table.get_device()
    n_seq, width = _table(page_table, d)
    rows = seq_of.numel()
    _chk(library().tie_page_plan(
        _ints("ctx_lens", ctx_lens, n_seq, d), _ints("new_lens", new_lens, n_seq, d), n_seq, page_table.data_ptr(), width,
        n_pages, _ints("free_pages", free_pages, 0, d), 0 if free_pages is None else free_pages.numel(),
        _ints("n_free", n_free, 1, d), _ints("n_free_out", n_free_out, 1, d), _ints("row_start", row_start, n_seq + 1, d),
        _ints("seq_of", seq_of, rows, d), _ints("pos_of", pos_of, rows, d), _ints("slot_of", slot_of, rows, d), rows,
        _ints("status", status, 1, d), _raw_stream(d) if stream is None else stream), "tie_page_plan")


def kv_store(k, v, slots, k_pages, v_pages, stream=None):
    """Rows of k and v [rows, n_kv_head * 64] (float32, any row stride that both have) into their slots (tie_kv_store)."""
    fmt, n_pages, heads, layers, _, d = _pool(k_pages, v_pages)
    if layers != 1:
        _wrong("k_pages, v_pages", "one layer")
    rows = k.shape[0]
    kp, ld = _rows("k", k, heads * HEAD_DIM, d)
    vp, ldv = _rows("v", v, heads * HEAD_DIM, d)
    if v.shape[0] != rows or ldv != ld:
        _wrong("k and v", "one shape and row stride")
    _chk(library().tie_kv_store(kp, vp, ld, _ints("slots", slots, rows, d), rows, k_pages.data_ptr(), v_pages.data_ptr(),
                                fmt, n_pages, heads, _raw_stream(d) if stream is None else stream), "tie_kv_store")


def attention_paged_workspace():
    """Bytes of workspace of attention_paged on the current device."""
    return library().tie_attention_paged_workspace()


def attention_paged(q, k_pages, v_pages, page_table, row_start, ctx_lens, max_new, out, workspace, scale=None,
                    status=None, stream=None):
    """Causal attention of the new rows q over the pages that hold them (tie_attention_paged).
    scale: 1 / sqrt(64) by default."""
    fmt, n_pages, kv_heads, layers, _, d = _pool(k_pages, v_pages)
    if layers != 1:
        _wrong("k_pages, v_pages", "one layer")
    n_seq, width = _table(page_table, d)
    w = q.shape[-1]
    if w % HEAD_DIM or out.shape != q.shape:
        _wrong("q and out", f"one shape [rows, n_head * {HEAD_DIM}]")
    qp, ldq = _rows("q", q, w, d)
    op, ldo = _rows("out", out, w, d)
    wp, wn = _workspace(workspace, d)
    _chk(library().tie_attention_paged(
        qp, ldq, w // HEAD_DIM, k_pages.data_ptr(), v_pages.data_ptr(), fmt, n_pages, kv_heads, page_table.data_ptr(), width,
        _ints("row_start", row_start, n_seq + 1, d), _ints("ctx_lens", ctx_lens, n_seq, d), n_seq, max_new, q.shape[0],
        0.125 if scale is None else scale, op, ldo, wp, wn, _ints("status", status, 1, d),
        _raw_stream(d) if stream is None else stream), "tie_attention_paged")


def beam_select_workspace(n_req, beams, vocab):
    """Bytes of workspace of beam_select on the current device."""
    return library().tie_beam_select_workspace(n_req, beams, vocab)


def beam_select(logits, scores, beams, next_ids, parent, scores_out, workspace, done=None, done_out=None, eos_id=-1,
                stream=None):
    """One step of beam search over logits [n_req * beams, vocab] (tie_beam_select)."""
    d = logits.get_device()
    n, vocab = logits.shape
    if beams <= 0 or n % beams or d < 0:
        _wrong("logits", "n_req * beams rows on a CUDA device")
    lp, ldl = _rows("logits", logits, vocab, d)
    wp, wn = _workspace(workspace, d)
    _chk(library().tie_beam_select(
        lp, ldl, _floats("scores", scores, n, d), _ints("done", done, n, d), n // beams, beams, vocab, eos_id,
        _ints("next_ids", next_ids, n, d), _ints("parent", parent, n, d), _floats("scores_out", scores_out, n, d),
        _ints("done_out", done_out, n, d), wp, wn, _raw_stream(d) if stream is None else stream), "tie_beam_select")


def kv_reorder(k_pages, v_pages, page_table, parent, first, length, beams, stream=None):
    """Every layer's cached rows follow the beams' parents (tie_kv_reorder)."""
    fmt, n_pages, heads, layers, stride, d = _pool(k_pages, v_pages)
    n, width = _table(page_table, d)
    if beams <= 0 or n % beams:
        _wrong("page_table", "n_req * beams sequences")
    r = n // beams
    _chk(library().tie_kv_reorder(
        k_pages.data_ptr(), v_pages.data_ptr(), fmt, layers, stride, n_pages, heads, page_table.data_ptr(), width,
        _ints("parent", parent, n, d), _ints("first", first, r, d), _ints("length", length, r, d), r, beams,
        _raw_stream(d) if stream is None else stream), "tie_kv_reorder")
