"""mg_kv4_attn where the range of f16 and fp32 is at stake: weights far below
the largest one, but many, and enormous scores.

Tolerance, from the arithmetic, over strong positions of value 0 and weak ones
of one sign: the result is the weak ones' share, so that everything is
relative to it: scores off by ds = 2^-19 max scale sum |q k| (e^(2 ds) of a
weight), 2^-18 for fp32 sums, the exponential and 22-bit weights, 2^-10 where
weights are rounded to f16, and the type's rounding; a weight may also lose
2^-32 of the largest one, each of the weak ones."""
import numpy as np
import pytest

from tests import kv4_ref as ref
from tests.test_kv4_gpu import TYPES, Dev, run_attn

pytestmark = pytest.mark.gpu


def strong_and_weak(D, n, page, every):
    """One sequence of n positions and one key/value head: position 0, or every 32nd, has the key (6, 0, 0, ...) and the value
    0, all others the key 0 and the value 3."""
    n_pages = -(-n // page)
    h = ref.Cache(1, D, page, np.arange(n_pages)[None], n_pages)
    strong = np.zeros(D)
    strong[0] = 6.0

    def first(x, v):
        h.store(0, 0, 0, x, True)
        h.store(0, 0, 0, np.full(D, v), False)

    for p in range(1, 32):
        h.store(0, p, 0, np.zeros(D), True)
        h.store(0, p, 0, np.full(D, 3.0), False)
    first(strong if every else np.zeros(D), 0.0 if every else 3.0)
    h.pool[:] = h.pool[0, 0, 0]
    first(strong, 0.0)
    return h


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("nq,heads", [(1, 4), (3, 5), (20, 4)])
@pytest.mark.parametrize("gap", [0.0, 8.0, 12.3, 17.5, 20.0])
@pytest.mark.parametrize("every", [False, True])
def test_many_small_weights(torch_cuda, kind, D, nq, heads, gap, every):
    """First tokens whose scores are `gap` above 32767 others, each of e^-20 of their weight: one for all, or one for each 31."""
    n = 32768
    dev = Dev(torch_cuda, strong_and_weak(D, n, 256, every))
    q = np.zeros((nq, heads, D))
    q[:, :, 0] = gap / 6
    qs = np.array([0, nq])
    for max_kv in (n, 1):  # cut into pieces, and whole
        got, qq = run_attn(torch_cuda, dev, kind, q.reshape(nq, -1), qs, [n], heads, 1.0, max_kv=max_kv)
        score = 6 * qq[0, 0]  # of the strong ones, the others' is 0
        seen = np.arange(n - nq + 1, n + 1)
        strong = -(-seen // 32) if every else np.ones(nq)
        share = ((seen - strong) / strong * np.exp(-score))[:, None]
        want = 3 * share / (1 + share)
        rel = np.expm1(2.0 ** -18 * score) + 2.0 ** -18 + (0 if kind == "f32" else 2.0 ** -10) + TYPES[kind][2]
        tol = rel * want + 3 * (seen / strong)[:, None] * 2.0 ** -32 + (2.0 ** -24 if kind == "f16" else 0)
        assert (np.abs(got - want) <= tol).all(), (want[0, 0], got[0, 0])


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("nq", [1, 30])
@pytest.mark.parametrize("size", [1e5, 3e7])
def test_enormous_scores(torch_cuda, kind, nq, size):
    """Scores of 6e5 and 2e8, whose differences fp32 holds to a few units: the largest takes everything, in whichever block of
    positions it lies, and nothing overflows."""
    n = 700
    h = strong_and_weak(64, n, 32, False)
    k = np.zeros(64)
    for p, f in ((0, 1.0), (300, 3.0), (301, 2.0), (450, 6.0), (699, 4.0)):
        k[0] = f
        h.store(0, p, 0, k, True)
        h.store(0, p, 0, np.full(64, f), False)
    dev = Dev(torch_cuda, h)
    q = np.zeros((nq, 4, 64))
    q[:, :, 0] = size if kind != "f16" else 6e4
    scale = 1.0 if kind != "f16" else size / 6e4
    got, _ = run_attn(torch_cuda, dev, kind, q.reshape(nq, -1), np.array([0, nq]), [n], 4, scale)
    want = np.where(np.arange(n - nq, n) >= 450, 6.0, 0.0)
    assert (np.abs(got - want[:, None]) <= 2.0 ** -7).all()
    got, _ = run_attn(torch_cuda, dev, kind, q.reshape(nq, -1), np.array([0, nq]), [n], 4, -scale)
    assert np.isfinite(got).all()
