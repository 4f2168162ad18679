"""kv4_score.score refuses texts that it cannot score, before it runs any of them."""
import types

import numpy as np
import pytest

from midge_b200 import kv4_score


class NoModel:
    f = dict(vocab=100)

    def step(self, tokens):
        raise AssertionError("no step for a refused text")


@pytest.mark.parametrize("ids", [[], [5], [1, 2, 100], [1, 2, -1], [100, 1], np.array([3, 4, 2 ** 31 - 1])])
def test_refused(ids):
    with pytest.raises(ValueError):
        kv4_score.score(NoModel(), ids)


def test_the_last_token_is_scored_and_not_stepped(monkeypatch):
    seen = []
    model = types.SimpleNamespace(f=dict(vocab=100), step=lambda tokens: seen.append(tokens[0]) or np.zeros((len(tokens[0]), 100)))
    monkeypatch.setattr(kv4_score, "logprobs", lambda rows, ids, top: (np.asarray(ids, float),) * 4)
    lp, *_ = kv4_score.score(model, [7, 8, 99], step=1)
    assert seen == [[7], [8]] and list(lp) == [8, 99]
