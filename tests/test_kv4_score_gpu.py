"""midge_b200.kv4_score: a whole model over the 4-bit paged cache, with the
operators called together as a host would call them.

The steps' size must not matter: the projections and the attention of 16
tokens and of one differ in fp32 rounding only (2e-6 of a logit's terms per
matvec, a few layers: within 1e-3), except where that moves a key or value
across a midpoint of its 4 bits, a change of one number of a head by a step;
at rates near 1e-6 per number that is a handful in a whole run, so the median
is held to the rounding and the largest to 0.05.  Against the f16 cache only
the sign of life is checked: 4 bits keep a number to a quarter at worst and 7%
in the mean, which for these random models moves log probabilities by far
less than their own spread."""
import numpy as np
import pytest

from midge_b200 import abi, kv4_score
from midge_b200 import container as ct

pytestmark = pytest.mark.gpu


def _model(tmp_path, kind):
    if kind == "sinks":
        spec, edt = ct.config_spec("c1_tiny")
    else:
        spec = ct.qwen3_spec(hidden=256, n_layers=2, n_heads=4, n_kv_heads=2, head_dim=128, vocab=1024, experts=8,
                             top_k=2, ffn=256)
        edt = "q8r"
    return ct.write_synthetic_model(str(tmp_path / kind), spec, edt, seed=3), spec


@pytest.mark.parametrize("kind", ["sinks", "norms"])
def test_score_of_a_model(torch_cuda, tmp_path, kind):
    path, spec = _model(tmp_path, kind)
    rng = np.random.default_rng(5)
    ids = rng.integers(0, spec["vocab"], 150)
    m = kv4_score.Kv4Model(path, 150, seqs=2, page=32)
    lp, ent, ai, al = kv4_score.score(m, ids, seq=0, top=3)
    one, ent1, _, _ = kv4_score.score(m, ids, seq=1, top=3, step=1)  # token by token, the other sequence's pages
    assert lp.shape == (149,) and ai.shape == (149, 3)
    assert np.median(np.abs(lp - one)) < 1e-3 and np.abs(lp - one).max() < 0.05
    assert np.median(np.abs(ent - ent1)) < 1e-3
    assert (np.diff(al, axis=1) <= 0).all() and (al[:, 0] >= lp).all()
    e = abi.Model.from_dir(path, ctx=160)
    rows = e.forward_batch(0, ids[:-1].astype(np.int32), logits_mode=2).astype(np.float64)
    e.close()
    z = rows - rows.max(1, keepdims=True)
    f16 = z[np.arange(149), ids[1:]] - np.log(np.exp(z).sum(1))
    assert np.isfinite(lp).all() and np.corrcoef(lp, f16)[0, 1] > 0.9
    assert abs(lp.mean() - f16.mean()) < 0.25 * f16.std()


def test_several_sequences_in_a_step(torch_cuda, tmp_path):
    """Sequences of different lengths advance together as they do alone."""
    path, spec = _model(tmp_path, "sinks")
    rng = np.random.default_rng(6)
    texts = [rng.integers(0, spec["vocab"], n) for n in (40, 9, 23)]
    alone = kv4_score.Kv4Model(path, 64, seqs=3, page=32)
    want = [kv4_score.score(alone, t, seq=i, top=0, step=5)[0] for i, t in enumerate(texts)]
    m = kv4_score.Kv4Model(path, 64, seqs=3, page=32)
    got = [[] for _ in texts]
    at = [0, 0, 0]
    while any(at[i] < len(t) - 1 for i, t in enumerate(texts)):
        part = {i: list(t[at[i]:min(at[i] + 5, len(t) - 1)]) for i, t in enumerate(texts) if at[i] < len(t) - 1}
        rows = m.step(part)
        ids = np.concatenate([texts[i][at[i] + 1:at[i] + 1 + len(part[i])] for i in sorted(part)])
        lp = kv4_score.logprobs(rows, ids, 0)[0]
        k = 0
        for i in sorted(part):
            got[i].extend(lp[k:k + len(part[i])])
            k += len(part[i])
            at[i] += len(part[i])
    for g, w in zip(got, want):
        d = np.abs(np.array(g) - w)
        assert np.median(d) < 1e-3 and d.max() < 0.05


def test_step_refusals(torch_cuda, tmp_path):
    path, spec = _model(tmp_path, "sinks")
    m = kv4_score.Kv4Model(path, 8, page=32)
    for bad in ({0: []}, {0: [1] * 17}, {0: [spec["vocab"]]}, {0: [-1]}, {0: [1] * 9}):
        with pytest.raises(ValueError):
            m.step(bad)
