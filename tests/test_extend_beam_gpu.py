"""Tokens appended to the paged pool (model_extend_batch) and beam search (model_generate_beam):
the model paths over the page plan, the row store, paged attention, beam selection and cache
reordering, against the CPU oracle and against the paths that were there."""
import numpy as np
import pytest

import oracle
import tie_b200
from tie_b200 import synth

pytestmark = pytest.mark.gpu
ARG, CAPACITY, RANGE = (tie_b200.MODEL_STATUS.index(s) for s in ("MODEL_ERR_ARG", "MODEL_ERR_CAPACITY", "MODEL_ERR_RANGE"))


@pytest.fixture(scope="module")
def tiny(tiny_paths):
    w, inv, cfg = tiny_paths
    with tie_b200.Model(w, inv, cfg) as m:
        yield m, oracle.Oracle(w, cfg)


@pytest.mark.parametrize("pieces", [(5, 1), (1, 1, 1), (7, 9), (16, 16, 3), (1, 40), (30, 8, 9, 1), (64,)])
@pytest.mark.parametrize("n_seq", [1, 3])
def test_a_prompt_in_pieces_has_the_prompts_logits(tiny, tiny_paths, pieces, n_seq):
    """The first piece by prefill (or, with one piece, by extending an empty pool), the others appended: the
    engine's contract with the oracle's logits (max-abs 1e-3)."""
    m, ref = tiny
    T = sum(pieces)
    ids = synth.prompt_ids(m.vocab, n_seq, T, seed=T)
    want = np.stack([ref.prefill(p) for p in ids])
    at, got = 0, []
    if len(pieces) == 1:
        with tie_b200.Model(*tiny_paths) as fresh:
            fresh.batch_reserve(n_seq, T)
            nxt, lg = fresh.extend_batch(ids, want_logits=True)
        got.append(lg)
    else:
        m.batch_reserve(n_seq, T)
        _, lg = m.prefill_batch(ids[:, :pieces[0]], want_logits=True)
        got.append(lg)
        at = pieces[0]
        for n in pieces[1:]:
            nxt, lg = m.extend_batch(ids[:, at:at + n], want_logits=True)
            got.append(lg)
            at += n
    got = np.concatenate(got, axis=1)
    assert np.abs(got - want).max() <= 1e-3
    assert np.array_equal(nxt, got[:, -1].argmax(1))


def test_generation_goes_on_after_an_extension(tiny):
    """Prefill, extend, decode: the tokens of one greedy generation over the whole prompt."""
    m, ref = tiny
    ids = synth.prompt_ids(m.vocab, 2, 23, seed=9)
    m.batch_reserve(2, 40)
    m.prefill_batch(ids[:, :6])
    nxt, _ = m.extend_batch(ids[:, 6:])
    out = [nxt]
    for _ in range(9):
        nxt, _ = m.decode_step_batch(out[-1])
        out.append(nxt)
    want = np.stack([ref.greedy(p, 10)[0] for p in ids])
    assert np.array_equal(np.stack(out, 1), want)


def test_an_extension_takes_pages_as_it_needs_them(tiny):
    m, _ = tiny
    ids = synth.prompt_ids(m.vocab, 2, 40, seed=2)
    m.batch_reserve_pages(2, 64, 5)
    m.prefill_batch(ids[:, :16])
    assert m.batch_free_pages() == 3
    m.extend_batch(ids[:, 16:32])
    assert m.batch_free_pages() == 1
    rc, _, _ = m.extend_batch(ids[:, 32:33], check=False)           # a page for each, one is left
    assert rc == CAPACITY
    m.batch_reserve(2, 64)


def test_extension_refusals(tiny):
    m, _ = tiny
    ids = synth.prompt_ids(m.vocab, 2, 8, seed=2)
    m.batch_reserve_pages(2, 16, 2)
    m.prefill_batch(ids)
    L = tie_b200.library()
    assert m.extend_batch(synth.prompt_ids(m.vocab, 3, 2, seed=1), check=False)[0] == ARG        # more sequences than reserved
    assert m.extend_batch(synth.prompt_ids(m.vocab, 2, 9, seed=1), check=False)[0] == CAPACITY
    bad = ids[:, :2].copy()
    bad[1, 1] = m.vocab
    assert m.extend_batch(bad, check=False)[0] == RANGE
    assert L.model_extend_batch(None, None, 1, 1, None, 0, None) == ARG
    nxt, _ = m.extend_batch(ids[:, :8])                                                          # and the pool is as it was
    assert nxt.shape == (2,)


def _beam_search(ref, prompt, beams, n_new, eos):
    """The search by the oracle's logits, all in float64: (tokens, scores), best first, and the smallest gap between
    a kept candidate and the next best one that was not (below it the choice is the arithmetic's)."""
    live, gap = [((), 0.0, False)], np.inf
    for _ in range(n_new):
        cand = []
        for b, (toks, score, done) in enumerate(live):
            if done:
                cand.append((score, b, eos))
                continue
            x = ref.prefill(np.concatenate([prompt, np.array(toks, np.int32)]).astype(np.int32))[-1].astype(np.float64)
            x = x - x.max()
            x = score + x - np.log(np.exp(x).sum())
            cand += [(x[t], b, int(t)) for t in np.argsort(-x, kind="stable")[:beams + 1]]
        cand.sort(key=lambda c: (-c[0], c[1], c[2]))
        if len(cand) > beams:
            gap = min(gap, cand[beams - 1][0] - cand[beams][0])
        live = [(live[b][0] + (t,), s, live[b][2] or t == eos) for s, b, t in cand[:beams]]
    order = sorted(range(len(live)), key=lambda i: -live[i][1])
    return [live[i][0] for i in order], [live[i][1] for i in order], gap


@pytest.mark.parametrize("beams,n_new,with_eos", [(1, 6, False), (3, 20, False), (4, 9, True), (2, 1, False), (8, 5, True)])
def test_beam_search_is_the_oracles(tiny, beams, n_new, with_eos):
    m, ref = tiny
    prompts = synth.prompt_ids(m.vocab, 2, 7, seed=beams)
    m.batch_reserve(2 * beams, 7 + n_new)
    # a token that the search does produce, so that a beam finishes early
    eos = int(_beam_search(ref, prompts[0], beams, n_new, -1)[0][0][n_new // 2]) if with_eos else -1
    ids, scores = m.generate_beam(prompts, beams, n_new, eos)
    for r in range(2):
        want, sc, gap = _beam_search(ref, prompts[r], beams, n_new, eos)
        assert gap > 2e-5, "the prompt's search hangs on the last digits: take another seed"
        # the logits agree within 1e-3 by contract, a log probability within twice that, n_new of them added
        assert np.abs(scores[r] - np.array(sc)).max() <= 2e-3 * n_new
        assert sorted(map(tuple, ids[r].tolist())) == sorted(want)
        assert (np.diff(scores[r]) <= 0).all()
        if with_eos:
            for row in ids[r]:
                hit = np.flatnonzero(row == eos)
                assert not len(hit) or (row[hit[0]:] == eos).all()


def test_one_beam_is_greedy_generation(tiny):
    m, _ = tiny
    prompts = synth.prompt_ids(m.vocab, 3, 11, seed=77)
    m.batch_reserve(3, 40)
    ids, _ = m.generate_beam(prompts, 1, 20)
    assert np.array_equal(ids[:, 0], m.generate_greedy(prompts, 20))


def test_beam_search_on_the_batched_paths(mini_paths):
    """More than eight sequences take the tensor-core decode; the best beam is at least as probable as greedy's."""
    w, inv, cfg = mini_paths
    with tie_b200.Model(w, inv, cfg) as m:
        prompts = synth.prompt_ids(m.vocab, 5, 30, seed=5)
        m.batch_reserve(20, 80)
        ids, scores = m.generate_beam(prompts, 4, 40)
        wide, wide_scores = m.generate_beam(prompts[2:3], 4, 40)    # four sequences: the streaming decode
        assert np.abs(scores[2] - wide_scores[0]).max() <= 2e-3 * 40
        greedy, greedy_scores = m.generate_beam(prompts, 1, 40)
        assert (scores[:, 0] >= greedy_scores[:, 0] - 1e-3).all()
        assert m.kernel_launches() > 0


def test_beam_refusals(tiny):
    m, _ = tiny
    p = synth.prompt_ids(m.vocab, 2, 7, seed=1)
    m.batch_reserve_pages(4, 16, 4)
    assert m.generate_beam(p, 3, 4, check=False)[0] == ARG           # six sequences, four reserved
    assert m.generate_beam(p, 2, 11, check=False)[0] == CAPACITY
    assert m.generate_beam(p[:1], 17, 2, check=False)[0] == CAPACITY
    assert m.generate_beam(p, 2, 2, eos_id=m.vocab, check=False)[0] == RANGE
    assert m.generate_beam(np.full((1, 3), -1), 2, 2, check=False)[0] == RANGE
    assert tie_b200.library().model_generate_beam(None, None, 1, 1, 1, 1, -1, None, None) == ARG
