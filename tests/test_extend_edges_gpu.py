"""Appending to and searching over the paged pool where a call does not follow the simplest one before it."""
import numpy as np
import pytest

import oracle
import tie_b200
from tie_b200 import synth

pytestmark = pytest.mark.gpu
ARG = tie_b200.MODEL_STATUS.index("MODEL_ERR_ARG")


@pytest.fixture()
def fresh(tiny_paths):
    w, inv, cfg = tiny_paths
    with tie_b200.Model(w, inv, cfg) as m:
        yield m, oracle.Oracle(w, cfg)


def test_an_extension_adds_nothing_to_the_attention_statistics(fresh):
    m, _ = fresh
    ids = synth.prompt_ids(m.vocab, 2, 24, seed=3)
    m.batch_reserve(2, 32)
    m.collect_attn_stats(True)
    m.extend_batch(ids[:, :4])                       # the first call: no statistics of any kind yet
    assert m.attn_rowsum_range()[2] == 0
    m.prefill_batch(ids[:, :9])
    before = m.attn_rowsum_range()
    assert before[2] > 0
    m.extend_batch(ids[:, 9:20])
    assert m.attn_rowsum_range() == before
    m.decode_step_batch(ids[:, 20])                  # and the next call's are counted once
    assert m.attn_rowsum_range()[2] == before[2] + before[2] // 9
