"""Beam search from the paged 8-bit KV cache (qnt_beam_search).

One beam is greedy decoding.  Several are held to the f16 caches' log-probabilities: the cache's rounding moves a step's by less than
a tenth of what another context with the same last token does (its share of the values is under 1%, so a factor of ten is left),
while a beam that read another's positions would move them by about that distance itself."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def log_probs(m, ids, valid):
    """log p of every token after each of the prefixes ids[: i + 1], from the f16 caches, in f64."""
    out = []
    for p, t in enumerate(ids):
        x = m.forward(int(t), p)[:valid].astype(np.float64)
        x -= x.max()
        out.append(x - np.log(np.exp(x).sum()))
    return out


@pytest.mark.parametrize("name, n, page", [("tiny_q8", 37, 16), ("tiny_q4sl", 70, 64), ("tiny_q8", 530, 32)])
def test_one_beam_is_greedy(qb, models, name, n, page):
    ctx = 512 if n < 500 else 512 + 64
    m = qb.Model(models("tiny_long" if n > 500 else name), ctx_len=ctx)
    try:
        prompt = np.random.default_rng(n).integers(0, m.hp.n_tokens, n)
        m.batch_init_paged(4, ctx, 4 * (ctx // page), page)
        want = [m.prefill_batch(0, prompt)]
        for _ in range(11):
            want.append(int(m.decode_batch([0], [want[-1]])[0]))
        m.batch_reset(0)
        (ids, score), = m.beam_search(prompt, 1, 12)
        assert ids.tolist() == want and score < 0
        # the best of one step's beams are the most likely tokens
        first = m.beam_search(prompt, 4, 1)
        assert first[0][0].tolist() == want[:1] and [s for _, s in first] == sorted((s for _, s in first), reverse=True)
        assert len({int(i[0]) for i, _ in first}) == 4
    finally:
        m.close()


@pytest.mark.parametrize("name, n, beams, steps, page", [("tiny_q8", 21, 4, 20, 16), ("tiny_q4sl", 64, 8, 9, 32), ("tiny_q8", 5, 3, 30, 64)])
def test_scores_are_the_answers_log_probabilities(qb, models, name, n, beams, steps, page):
    m = qb.Model(models(name), ctx_len=512)
    try:
        rng = np.random.default_rng(n)
        valid = m.hp.n_tokens
        prompt = rng.integers(0, valid, n)
        m.batch_init_paged(beams, 256, beams * 16 + 4, page)
        got = m.beam_search(prompt, beams, steps)
        scores = [s for _, s in got]
        assert scores == sorted(scores, reverse=True) and len({tuple(i.tolist()) for i, _ in got}) == beams
        for ids, score in got:
            assert len(ids) == steps
            whole = np.concatenate([prompt, ids[:-1]])
            right = log_probs(m, whole, valid)[n - 1:]
            other = whole.copy()
            other[: n - 1] = rng.integers(0, valid, n - 1)
            wrong = log_probs(m, other, valid)[n - 1:]
            want = sum(lp[t] for lp, t in zip(right, ids))
            apart = sum(np.abs(a - b).max() for a, b in zip(right, wrong))
            assert abs(score - want) <= 0.1 * apart, (score, want, apart)
        assert m.beam_search(prompt, beams, steps)[0][0].tolist() == got[0][0].tolist()  # sequences and pages were given back
        m.prefill_batch(beams - 1, prompt)
    finally:
        m.close()


def test_beams_end(qb, models):
    """The token that the best beam takes second ends it: it stays with its score, the others go on; with one beam the search stops."""
    m = qb.Model(models("tiny_q8"), ctx_len=512)
    try:
        prompt = np.random.default_rng(8).integers(0, m.hp.n_tokens, 30)
        m.batch_init_paged(4, 128, 40, 16)
        free = m.beam_search(prompt, 1, 8)[0][0]
        end = int(free[2])
        stop = free.tolist().index(end) + 1
        (ids, _), = m.beam_search(prompt, 1, 8, end_id=end)
        assert ids.tolist() == free.tolist()[:stop]
        for ids, score in m.beam_search(prompt, 4, 8, end_id=end):
            assert end not in ids.tolist()[:-1] and (len(ids) == 8 or ids[-1] == end) and np.isfinite(score)
    finally:
        m.close()


def test_what_is_refused(qb, models):
    m = qb.Model(models("tiny_q8"), ctx_len=512)
    try:
        prompt = np.arange(20)
        m.batch_init(4, 128)
        with pytest.raises(qb.QntError, match="paged"):
            m.beam_search(prompt, 2, 4)
        m.batch_init_paged(4, 64, 6, 16)
        for args in ((prompt, 0, 4), (prompt, 5, 4), (prompt, 65, 4), (prompt, 2, 0), (prompt[:0], 2, 4)):
            with pytest.raises(qb.QntError, match="1 .. 64 beams"):
                m.beam_search(*args)
        with pytest.raises(qb.QntError, match="exceed"):
            m.beam_search(prompt, 2, 46)
        with pytest.raises(qb.QntError, match="embedding"):
            m.beam_search([m.hp.vocab_size], 2, 4)
        with pytest.raises(qb.QntError, match="no free pages"):
            m.beam_search(prompt, 4, 40)
        first = m.beam_search(prompt, 2, 8)  # the refused calls left nothing behind
        m.prefill_batch(1, prompt)
        with pytest.raises(qb.QntError, match="must be empty"):
            m.beam_search(prompt, 2, 4)
        m.batch_reset(1)
        assert m.beam_search(prompt, 2, 8)[0][0].tolist() == first[0][0].tolist()
    finally:
        m.close()
