"""mg_kv4_attn of 16-bit types over caches so long that a running sum of one
sign loses what it truncates: many query rows, whole and cut units, more
units than the GPU holds at a time (they take turns at the places where long
sums rest).

Tolerances: over equal weak values the result is their share, relative to
which weights are rounded to f16 (2^-12 at worst, all alike), scores are off by
ds = 2^-19 of the largest, sums by 2^-13 (1024 truncated additions at 2^-23
each), and the result by the type's rounding; a weight may lose 2^-32 of the
largest.  Random caches as in
test_kv4_gpu."""
import numpy as np
import pytest

from tests import kv4_ref as ref
from tests.test_kv4_gpu import TYPES, Dev, check_attn, run_attn
from tests.test_kv4_mixed_gpu import random_pages
from tests.test_kv4_range_gpu import strong_and_weak

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("seqs,cut", [(1, False), (1, True), (10, True), (170, False)])
def test_half_a_million_equal_values(torch_cuda, kind, D, seqs, cut):
    """All sequences read the same pages.  The first position's score is 1.7 above the others'."""
    n, nq, heads = 524288, 30, 4
    host = strong_and_weak(D, n, 4096, False)
    host.table = np.repeat(host.table, seqs, 0)
    dev = Dev(torch_cuda, host)
    q = np.zeros((seqs * nq, heads, D))
    q[:, :, 0] = 1.7 / 6
    got, qq = run_attn(torch_cuda, dev, kind, q.reshape(len(q), -1), nq * np.arange(seqs + 1), [n] * seqs, heads, 1.0,
                       max_kv=n if cut else 1, repeat=2)
    score = 6 * qq[0, 0]
    share = (np.arange(n - nq, n) * np.exp(-score))[:, None]
    want = np.tile(3 * share / (1 + share), (seqs, 1))
    rel = 2.0 ** -12 + np.expm1(2.0 ** -18 * score) + 2.0 ** -13 + TYPES[kind][2] / 2
    assert (np.abs(got - want) <= rel * want + 3 * n * 2.0 ** -32 / (1 + share[0, 0])).all(), (want[0, 0], got[0, 0])


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rising", [False, True])
def test_random_long_caches(torch_cuda, kind, D, rising):
    """40000 positions in one go; scores of no order, and scores whose largest comes later and later."""
    rng = np.random.default_rng(D + rising)
    lengths, nq, heads = [40000, 18000], [21, 33], 4
    h = random_pages(rng, lengths, 1, D, 256)
    q = rng.standard_normal((54, heads * D)) * 0.3
    if rising:  # scales of the keys from 2^-7 to 2^2 along the pages, keys and queries of dimension 0 of one sign
        for s, length in enumerate(lengths):
            for i in range(-(-length // 256)):
                h.pool[h.table[s, i], 0, :, 32 * D:33 * D] = (8 + 9 * 256 * i // length) << 2
        q = np.abs(q)
        h.pool[..., :16 * D] &= 0x77
    dev = Dev(torch_cuda, h)
    qs = np.concatenate([[0], np.cumsum(nq)])
    for max_kv in (1, 40000):
        got, qq = run_attn(torch_cuda, dev, kind, q, qs, lengths, heads, D ** -0.5, max_kv=max_kv, repeat=2)
        check_attn(got, qq, dev, kind, qs, lengths, heads, D ** -0.5)
