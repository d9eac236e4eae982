"""The operators over device memory (``include/tie_b200.h``): page plans, K/V row
stores, attention over the paged cache, beam selection and cache reordering.

Arguments are device tensors (anything with ``data_ptr``, ``shape``, ``stride``,
``dtype`` and ``device``: torch tensors). Outputs and workspaces are the
caller's; nothing is allocated or waited for. Work runs on ``stream`` (a
``cudaStream_t`` as an int), by default torch's current stream of the tensors'
device. Shapes, types and layouts that the C entry points cannot see are
checked here (``ValueError``); their own refusals raise ``ModelError``.

The sizes of a page pool come from its tensors: ``k_pages`` and ``v_pages`` are
[n_pages, 16, n_kv_head * 64] (``kv_reorder`` also takes
[n_layer, n_pages, 16, n_kv_head * 64]), float32 or bfloat16, contiguous.
"""
from __future__ import annotations

from .lib import TIE_KV_BF16, TIE_KV_F32, _chk, library

PAGE_ROWS = 16
HEAD_DIM = 64


def _stream(t, stream):
    if stream is not None:
        return stream
    import torch
    return torch.cuda.current_stream(t.device).cuda_stream


def _need(ok, what):
    if not ok:
        raise ValueError(what)


_NAMES = {}


def _type(t):
    """The element type's name, of torch.float32 as of any object that prints alike."""
    n = _NAMES.get(t.dtype)
    if n is None:
        n = _NAMES[t.dtype] = str(t.dtype).rpartition(".")[2]
    return n


def _ints(name, t, n, device):
    """A contiguous int32 vector of at least n elements on `device`: its address (None stays None)."""
    if t is None:
        return None
    _need(_type(t) == "int32" and t.is_contiguous() and t.numel() >= n and t.device == device,
          f"{name}: {n} contiguous int32 elements on {device} are wanted")
    return t.data_ptr()


def _rows(name, t, width, device):
    """A float32 matrix of `width` columns whose rows are contiguous: (address, leading dimension)."""
    _need(_type(t) == "float32" and t.dim() == 2 and t.shape[1] == width and t.stride(1) == 1 and t.device == device,
          f"{name}: float32 [rows, {width}] with contiguous rows on {device} is wanted")
    return t.data_ptr(), t.stride(0) if t.shape[0] > 1 else max(t.stride(0), width)


def _pool(k, v):
    """(format, n_pages, n_kv_head, layers, layer stride) of a pool's two tensors."""
    _need(k.shape == v.shape and k.dtype == v.dtype and k.device == v.device and k.is_contiguous() and v.is_contiguous(),
          "k_pages and v_pages: two contiguous tensors of one shape, type and device are wanted")
    shape, kind = k.shape, _type(k)
    _need(len(shape) in (3, 4) and shape[-2] == PAGE_ROWS and shape[-1] % HEAD_DIM == 0 and kind in ("float32", "bfloat16"),
          f"k_pages, v_pages: float32 or bfloat16 [n_pages, {PAGE_ROWS}, n_kv_head * {HEAD_DIM}] is wanted")
    layers = shape[0] if len(shape) == 4 else 1
    n_pages = shape[-3]
    return (TIE_KV_BF16 if kind == "bfloat16" else TIE_KV_F32, n_pages, shape[-1] // HEAD_DIM, layers,
            n_pages * PAGE_ROWS * shape[-1])


def _table(t, device):
    _need(_type(t) == "int32" and t.dim() == 2 and t.is_contiguous() and t.device == device,
          f"page_table: contiguous int32 [n_seq, pages_per_seq] on {device} is wanted")
    return t.shape


def page_plan(ctx_lens, new_lens, page_table, n_pages, row_start, seq_of, pos_of, slot_of, status, free_pages=None,
              n_free=None, n_free_out=None, stream=None):
    """Assigns pages to new positions and writes row starts and slot maps (tie_page_plan)."""
    d = page_table.device
    n_seq, width = _table(page_table, d)
    rows = seq_of.numel()
    _chk(library().tie_page_plan(
        _ints("ctx_lens", ctx_lens, n_seq, d), _ints("new_lens", new_lens, n_seq, d), n_seq, page_table.data_ptr(), width,
        n_pages, _ints("free_pages", free_pages, 0, d), 0 if free_pages is None else free_pages.numel(),
        _ints("n_free", n_free, 1, d), _ints("n_free_out", n_free_out, 1, d), _ints("row_start", row_start, n_seq + 1, d),
        _ints("seq_of", seq_of, rows, d), _ints("pos_of", pos_of, rows, d), _ints("slot_of", slot_of, rows, d), rows,
        _ints("status", status, 1, d), _stream(page_table, stream)), "tie_page_plan")


def kv_store(k, v, slots, k_pages, v_pages, stream=None):
    """Rows of k and v [rows, n_kv_head * 64] (float32, any row stride that both have) into their slots (tie_kv_store)."""
    fmt, n_pages, heads, layers, _ = _pool(k_pages, v_pages)
    _need(layers == 1, "kv_store: the pages of one layer are wanted")
    d, rows = k_pages.device, k.shape[0]
    kp, ld = _rows("k", k, heads * HEAD_DIM, d)
    vp, ldv = _rows("v", v, heads * HEAD_DIM, d)
    _need(v.shape[0] == rows and ldv == ld, "kv_store: k and v of one shape and row stride are wanted")
    _chk(library().tie_kv_store(kp, vp, ld, _ints("slots", slots, rows, d), rows, k_pages.data_ptr(), v_pages.data_ptr(),
                                fmt, n_pages, heads, _stream(k_pages, stream)), "tie_kv_store")


def attention_paged_workspace():
    """Bytes of workspace of attention_paged on the current device."""
    return library().tie_attention_paged_workspace()


def attention_paged(q, k_pages, v_pages, page_table, row_start, ctx_lens, max_new, out, workspace, scale=None,
                    status=None, stream=None):
    """Causal attention of the new rows q over the pages that hold them (tie_attention_paged).
    scale: 1 / sqrt(64) by default."""
    fmt, n_pages, kv_heads, layers, _ = _pool(k_pages, v_pages)
    _need(layers == 1, "attention_paged: the pages of one layer are wanted")
    d = k_pages.device
    n_seq, width = _table(page_table, d)
    w = q.shape[-1]
    _need(w % HEAD_DIM == 0 and out.shape == q.shape, "attention_paged: q and out of one shape [rows, n_head * 64] are wanted")
    qp, ldq = _rows("q", q, w, d)
    op, ldo = _rows("out", out, w, d)
    _need(workspace.is_contiguous() and workspace.device == d, "attention_paged: a contiguous workspace on the device is wanted")
    _chk(library().tie_attention_paged(
        qp, ldq, w // HEAD_DIM, k_pages.data_ptr(), v_pages.data_ptr(), fmt, n_pages, kv_heads, page_table.data_ptr(), width,
        _ints("row_start", row_start, n_seq + 1, d), _ints("ctx_lens", ctx_lens, n_seq, d), n_seq, max_new, q.shape[0],
        0.125 if scale is None else scale, op, ldo, workspace.data_ptr(), workspace.numel() * workspace.element_size(),
        _ints("status", status, 1, d), _stream(q, stream)), "tie_attention_paged")


def beam_select_workspace(n_req, beams, vocab):
    """Bytes of workspace of beam_select on the current device."""
    return library().tie_beam_select_workspace(n_req, beams, vocab)


def beam_select(logits, scores, beams, next_ids, parent, scores_out, workspace, done=None, done_out=None, eos_id=-1,
                stream=None):
    """One step of beam search over logits [n_req * beams, vocab] (tie_beam_select)."""
    d = logits.device
    n, vocab = logits.shape
    _need(beams > 0 and n % beams == 0, "beam_select: n_req * beams rows of logits are wanted")
    lp, ldl = _rows("logits", logits, vocab, d)
    for name, t in (("scores", scores), ("scores_out", scores_out)):
        _need(_type(t) == "float32" and t.is_contiguous() and t.numel() >= n and t.device == d,
              f"{name}: {n} contiguous float32 elements on {d} are wanted")
    _need(workspace.is_contiguous() and workspace.device == d, "beam_select: a contiguous workspace on the device is wanted")
    _chk(library().tie_beam_select(
        lp, ldl, scores.data_ptr(), _ints("done", done, n, d), n // beams, beams, vocab, eos_id,
        _ints("next_ids", next_ids, n, d), _ints("parent", parent, n, d), scores_out.data_ptr(),
        _ints("done_out", done_out, n, d), workspace.data_ptr(), workspace.numel() * workspace.element_size(),
        _stream(logits, stream)), "tie_beam_select")


def kv_reorder(k_pages, v_pages, page_table, parent, first, length, beams, stream=None):
    """Every layer's cached rows follow the beams' parents (tie_kv_reorder)."""
    fmt, n_pages, heads, layers, stride = _pool(k_pages, v_pages)
    d = k_pages.device
    n, width = _table(page_table, d)
    _need(beams > 0 and n % beams == 0, "kv_reorder: n_req * beams sequences are wanted")
    r = n // beams
    _chk(library().tie_kv_reorder(
        k_pages.data_ptr(), v_pages.data_ptr(), fmt, layers, stride, n_pages, heads, page_table.data_ptr(), width,
        _ints("parent", parent, n, d), _ints("first", first, r, d), _ints("length", length, r, d), r, beams,
        _stream(k_pages, stream)), "tie_kv_reorder")
