"""mg_logprobs of rows whose entries lie further apart than fp32 sums can be
carried over: a thread meets entries around 0, then 39 above them (its sums
stay against the first), then finite ones tens of orders of magnitude larger.
Tolerances as in test_logprobs_gpu (z within 2^-17, the entropy within 2^-16
(1 + H)), and 2^-22 of a log probability."""
import numpy as np
import pytest

from tests import kv4_ref as ref
from tests.test_logprobs_gpu import run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,far", [("f32", 1e30), ("f32", 3e38), ("f32", 1e22), ("bf16", 1e30), ("bf16", 1e24)])
@pytest.mark.parametrize("V,rows", [(27000, 600), (90000, 2), (201088, 1)])
def test_far_larger_entries_last(torch_cuda, kind, far, V, rows):
    rng = np.random.default_rng(V)
    x = rng.standard_normal((rows, V)).astype(np.float32)
    x[:, V // 3:] += 39
    x[:, V - V // 3:] = rng.choice([0.5, 1.0], (rows, V // 3)) * far
    x[:, V - 5] = far
    ids = np.stack([np.array([V - 5, 3])] * rows)
    (lp, ent, _, _), x = run(torch_cuda, x, ids, 0, kind)
    for r in range(0, rows, 37):
        wlp, went, _, _ = ref.logprobs(x[r], ids[r], 0)
        assert abs(ent[r] - went) <= 2.0 ** -16 * (1 + went)
        assert (np.abs(lp[r] - wlp) <= 2.0 ** -17 + 2.0 ** -22 * np.abs(wlp)).all()
    assert np.isfinite(ent).all() and np.isfinite(lp).all()
