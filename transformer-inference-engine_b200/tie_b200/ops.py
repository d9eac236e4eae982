"""The operators over device memory (``include/tie_b200.h``): page plans, K/V row
stores, attention over the paged cache, beam selection and cache reordering.

Arguments are torch tensors on a CUDA device. Outputs and workspaces are the
caller's; nothing is allocated or waited for. Work runs on ``stream`` (a
``cudaStream_t`` as an int), by default torch's current stream of the tensors'
device. Shapes, types and layouts that the C entry points cannot see are
checked before the call (``ValueError``, by csrc/python/ops_module.cpp); their
own refusals raise ``ModelError``.

The sizes of a page pool come from its tensors: ``k_pages`` and ``v_pages`` are
[n_pages, 16, n_kv_head * 64] (``kv_reorder`` also takes
[n_layer, n_pages, 16, n_kv_head * 64]), float32 or bfloat16, contiguous.
"""
from __future__ import annotations

import ctypes

import torch

from .lib import ModelError, library

PAGE_ROWS = 16
HEAD_DIM = 64

_module = None


def _ops():
    """tie_b200._ops over the loaded library; raises (no fallback) when it is not built."""
    global _module
    if _module is None:
        try:
            from . import _ops as m
        except ImportError as e:
            raise ImportError("tie_b200._ops is not built; run tie_b200.build") from e
        lib = library()
        m.init(torch.Tensor, torch.Tensor.__dlpack_c_exchange_api__,
               *(ctypes.cast(f, ctypes.c_void_p).value for f in (
                   lib.tie_page_plan, lib.tie_kv_store, lib.tie_attention_paged, lib.tie_beam_select, lib.tie_kv_reorder)))
        _module = m
    return _module


def page_plan(ctx_lens, new_lens, page_table, n_pages, row_start, seq_of, pos_of, slot_of, status, free_pages=None,
              n_free=None, n_free_out=None, stream=None):
    """Assigns pages to new positions and writes row starts and slot maps (tie_page_plan)."""
    rc = (_module or _ops()).page_plan(ctx_lens, new_lens, page_table, n_pages, row_start, seq_of, pos_of, slot_of, status,
                                       free_pages, n_free, n_free_out, stream)
    if rc:
        raise ModelError(rc, "tie_page_plan")


def kv_store(k, v, slots, k_pages, v_pages, stream=None):
    """Rows of k and v [rows, n_kv_head * 64] (float32, any row stride that both have) into their slots (tie_kv_store)."""
    rc = (_module or _ops()).kv_store(k, v, slots, k_pages, v_pages, stream)
    if rc:
        raise ModelError(rc, "tie_kv_store")


def attention_paged_workspace():
    """Bytes of workspace of attention_paged on the current device."""
    return library().tie_attention_paged_workspace()


def attention_paged(q, k_pages, v_pages, page_table, row_start, ctx_lens, max_new, out, workspace, scale=None,
                    status=None, stream=None):
    """Causal attention of the new rows q over the pages that hold them (tie_attention_paged).
    scale: 1 / sqrt(64) by default. status: an int32 tensor that receives an error code when a bounded wait in
    the kernel has expired, which nothing else tells."""
    rc = (_module or _ops()).attention_paged(q, k_pages, v_pages, page_table, row_start, ctx_lens, max_new, out, workspace,
                                             0.125 if scale is None else scale, status, stream)
    if rc:
        raise ModelError(rc, "tie_attention_paged")


def beam_select_workspace(n_req, beams, vocab):
    """Bytes of workspace of beam_select on the current device."""
    return library().tie_beam_select_workspace(n_req, beams, vocab)


def beam_select(logits, scores, beams, next_ids, parent, scores_out, workspace, done=None, done_out=None, eos_id=-1,
                stream=None):
    """One step of beam search over logits [n_req * beams, vocab] (tie_beam_select)."""
    rc = (_module or _ops()).beam_select(logits, scores, beams, next_ids, parent, scores_out, workspace, done, done_out,
                                         eos_id, stream)
    if rc:
        raise ModelError(rc, "tie_beam_select")


def kv_reorder(k_pages, v_pages, page_table, parent, first, length, beams, stream=None):
    """Every layer's cached rows follow the beams' parents (tie_kv_reorder)."""
    rc = (_module or _ops()).kv_reorder(k_pages, v_pages, page_table, parent, first, length, beams, stream)
    if rc:
        raise ModelError(rc, "tie_kv_reorder")
