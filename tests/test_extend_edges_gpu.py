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


def test_an_extension_of_sequences_that_hold_less_is_refused(fresh):
    """Released, never filled, or overwritten by a call that failed: there is nothing to attend to."""
    m, ref = fresh
    ids = synth.prompt_ids(m.vocab, 3, 30, seed=4)
    m.batch_reserve_pages(3, 48, 5)
    m.prefill_batch(ids[:2, :12])
    assert m.extend_batch(ids[:, 12:14], check=False)[0] == ARG          # the third was never filled
    _, lg = m.extend_batch(ids[:2, 12:14], want_logits=True)
    m.batch_release(1)
    assert m.extend_batch(ids[:2, 14:15], check=False)[0] == ARG
    _, more = m.extend_batch(ids[:1, 14:16], want_logits=True)           # the first still holds its positions
    want = ref.prefill(ids[0, :16])
    assert np.abs(np.concatenate([lg[0], more[0]]) - want[12:16]).max() <= 1e-3
    m.prefill_batch(ids[:2, :16])                                        # filled again
    m.extend_batch(ids[:2, 16:17])
    m.prefill_batch(ids[:2, :12])
    assert m.generate_beam(ids[:1, :12], 3, 25, check=False)[0] == tie_b200.MODEL_STATUS.index("MODEL_ERR_CAPACITY")
    assert m.extend_batch(ids[:2, 12:13], check=False)[0] == ARG         # the search had begun to overwrite them
    m.prefill_batch(ids[:2, :8])
    nxt, lg = m.extend_batch(ids[:2, 8:20], want_logits=True)
    assert np.abs(lg - np.stack([ref.prefill(p[:20])[8:] for p in ids[:2]])).max() <= 1e-3


@pytest.mark.parametrize("beams,n_new,with_eos", [(3, 14, False), (5, 9, True), (4, 1, False), (1, 6, False), (2, 2, False), (6, 20, False)])
def test_the_pool_holds_the_continuations_that_a_search_returns(fresh, beams, n_new, with_eos):
    """Decoding or extending after a search goes on from each returned continuation, in their order (the engine's
    contract with the oracle's logits, max-abs 1e-3)."""
    m, ref = fresh
    R, T = 3, 7
    prompts = synth.prompt_ids(m.vocab, R, T, seed=beams)
    m.batch_reserve(R * beams, T + n_new + 3)
    eos = -1
    if with_eos:
        eos = int(m.generate_beam(prompts, beams, n_new)[0][0, 0, n_new // 2])
    ids, _ = m.generate_beam(prompts, beams, n_new, eos)
    whole = np.concatenate([np.repeat(prompts, beams, 0), ids.reshape(R * beams, n_new)], 1).astype(np.int32)
    _, lg = m.decode_step_batch(whole[:, -1], want_logits=True)
    more = synth.prompt_ids(m.vocab, R * beams, 3, seed=1)
    _, lg2 = m.extend_batch(more, want_logits=True)
    for s in range(R * beams):
        want = ref.prefill(np.concatenate([whole[s], more[s]]).astype(np.int32))[T + n_new - 1:]
        assert np.abs(lg[s] - want[0]).max() <= 1e-3 and np.abs(lg2[s] - want[1:]).max() <= 1e-3, s


@pytest.mark.parametrize("kind", [tie_b200.TIE_STEP_PERSISTENT, tie_b200.TIE_STEP_STREAM])
def test_beam_search_and_extension_with_every_step_kernel(fresh, kind):
    m, ref = fresh
    prompts = synth.prompt_ids(m.vocab, 2, 9, seed=12)
    m.batch_reserve(4, 40)
    want = m.generate_beam(prompts, 2, 16)
    m.set_step_kernel(kind)
    ids, scores = m.generate_beam(prompts, 2, 16)
    assert np.abs(scores - want[1]).max() <= 2e-3 * 16
    assert np.array_equal(ids, want[0]) or np.abs(np.diff(want[1], axis=1)).min() < 2e-3 * 16
    whole = np.concatenate([np.repeat(prompts, 2, 0), ids.reshape(4, 16)], 1).astype(np.int32)
    _, lg = m.decode_step_batch(whole[:, -1], want_logits=True)
    nxt, lg2 = m.extend_batch(whole[:, :5], want_logits=True)
    for s in range(4):
        full = ref.prefill(np.concatenate([whole[s], whole[s, :5]]).astype(np.int32))[24:]
        assert np.abs(lg[s] - full[0]).max() <= 1e-3 and np.abs(lg2[s] - full[1:]).max() <= 1e-3


@pytest.mark.parametrize("fmt", [tie_b200.TIE_WEIGHTS_BF16, tie_b200.TIE_WEIGHTS_INT8])
def test_an_extension_agrees_with_a_prefill_in_every_weight_format(fresh, fmt):
    m, _ = fresh
    ids = synth.prompt_ids(m.vocab, 3, 30, seed=6)
    m.set_weight_format(fmt)
    m.batch_reserve(3, 40)
    _, want = m.prefill_batch(ids, want_logits=True)
    _, a = m.prefill_batch(ids[:, :11], want_logits=True)
    _, b = m.extend_batch(ids[:, 11:29], want_logits=True)
    _, c = m.extend_batch(ids[:, 29:], want_logits=True)
    assert np.abs(np.concatenate([a, b, c], 1) - want).max() <= 1e-3
    out, scores = m.generate_beam(ids[:, :12], 1, 9)
    assert np.array_equal(out[:, 0], m.generate_greedy(ids[:, :12], 9))
