"""What the operators over device memory accept and refuse at the edges of their arguments (no GPU needed)."""
import pytest

import tie_b200
from test_ops_cpu import ARG, ATTN, DEVICE, OK, PLAN, STORE, _call

L = tie_b200.library()


def _no_gpu():
    import torch
    return not torch.cuda.is_available()


def test_arrays_without_rows_need_no_address():
    assert _call(L.tie_kv_store, STORE, rows=0, k=None, v=None, slots=None) == OK
    assert _call(L.tie_attention_paged, ATTN, rows=0, q=None, out=None) == OK
    assert _call(L.tie_kv_store, STORE, rows=0, k=None, v=None, slots=None, k_pages=None) == ARG
    assert _call(L.tie_attention_paged, ATTN, rows=0, q=None, out=None, ws=None) == ARG
    assert _call(L.tie_kv_store, STORE, rows=1, slots=None) == ARG
    assert _call(L.tie_attention_paged, ATTN, rows=1, out=None) == ARG


@pytest.mark.parametrize("changed,refused", [
    (dict(free=None, max_free=0), False), (dict(max_free=0), False), (dict(free=None, n_free=None, n_free_out=None), False),
    (dict(free=None, max_free=1), True), (dict(free=None, max_free=0, n_free_out=None), True),
    (dict(free=None, max_free=0, n_free=None), True), (dict(max_free=0, n_free=None), True)])
def test_an_empty_free_list_needs_no_address(changed, refused):
    """A call that passes the checks of its arguments goes on to look for the device."""
    if _no_gpu():
        assert _call(L.tie_page_plan, PLAN, **changed) == (ARG if refused else DEVICE)
    elif refused:
        assert _call(L.tie_page_plan, PLAN, **changed) == ARG
