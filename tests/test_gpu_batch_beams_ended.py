"""Beams that end within a search from the paged cache while others go on (qnt_beam_search): each answer, ended ones included, has the
log-probabilities of its own tokens.  The bound is that of test_gpu_batch_beams.py."""
import numpy as np
import pytest

from test_gpu_batch_beams import log_probs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name, n, beams, steps, at", [("tiny_q8", 30, 4, 8, 2), ("tiny_q8", 21, 4, 12, 1), ("tiny_q4sl", 64, 8, 9, 3)])
def test_ended_beams_keep_their_score(qb, models, name, n, beams, steps, at):
    m = qb.Model(models(name), ctx_len=512)
    try:
        rng = np.random.default_rng(n)
        valid = m.hp.n_tokens
        prompt = rng.integers(0, valid, n)
        m.batch_init_paged(beams, 256, beams * 16 + 4, 16)
        free = m.beam_search(prompt, beams, steps)
        end = int(free[0][0][at])  # where the best free answer takes this, it now ends
        got = m.beam_search(prompt, beams, steps, end_id=end)
        ended = [ids for ids, _ in got if ids[-1] == end]
        assert any(len(ids) < steps for ids in ended)
        scores = [s for _, s in got]
        assert scores == sorted(scores, reverse=True) and len({tuple(i.tolist()) for i, _ in got}) == beams
        for ids, score in got:
            assert end not in ids.tolist()[:-1] and (len(ids) == steps or ids[-1] == end)
            whole = np.concatenate([prompt, ids[:-1]])
            other = whole.copy()
            other[: n - 1] = rng.integers(0, valid, n - 1)
            right, wrong = log_probs(m, whole, valid)[n - 1:], log_probs(m, other, valid)[n - 1:]
            want = sum(lp[t] for lp, t in zip(right, ids))
            assert abs(score - want) <= 0.1 * sum(np.abs(a - b).max() for a, b in zip(right, wrong)), (score, want)
    finally:
        m.close()
