"""CPU checks of Model.beam_search's numbers: what does not fit 32 bits is not taken for its lower half."""
import numpy as np
import pytest


class NoModel:
    h = None  # (refused by the library, were it called)


@pytest.mark.parametrize("prompt, beams, n_gen, end_id", [
    ([1, 2], 2, 4, 2 ** 32 + 5), ([1, 2], 2, 4, -(2 ** 32) + 5), ([1, 2], 2, 2 ** 32 + 4, -1), ([1, 2], 2 ** 32 + 2, 4, -1),
    (np.array([1, 2 ** 32 + 2]), 2, 4, -1), ([1, -(2 ** 32) + 2], 2, 4, -1)])
def test_numbers_past_32_bits(qb, prompt, beams, n_gen, end_id):
    with pytest.raises(ValueError, match="past 32 bits"):
        qb.Model.beam_search(NoModel(), prompt, beams, n_gen, end_id)


def test_others_reach_the_library(qb):
    for prompt in ([1, 2], [], np.array([3]), np.array([2 ** 31 - 1])):
        with pytest.raises(qb.QntError, match="null model"):
            qb.Model.beam_search(NoModel(), prompt, 2, 4)
