"""mg_kv4_attn of 16-bit types, few query rows, over caches so long and of so
many sequences that one warp sums tens of thousands of positions.  All
sequences read the same pages.  Tolerances as in test_kv4_long_sums_gpu."""
import numpy as np
import pytest

from tests.test_kv4_gpu import TYPES, Dev, check_attn, run_attn
from tests.test_kv4_mixed_gpu import random_pages
from tests.test_kv4_range_gpu import strong_and_weak

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("nq,heads", [(1, 4), (3, 5)])
@pytest.mark.parametrize("seqs", [1, 300, 1800])
def test_half_a_million_equal_values(torch_cuda, kind, D, nq, heads, seqs):
    """Cut finely, cut in pieces that are long themselves, and whole; with the hint of the length and with one far too small."""
    n = 524288
    host = strong_and_weak(D, n, 4096, False)
    host.table = np.repeat(host.table, seqs, 0)
    dev = Dev(torch_cuda, host)
    q = np.zeros((seqs * nq, heads, D))
    q[:, :, 0] = 1.7 / 6
    for max_kv in (n, 1):
        got, qq = run_attn(torch_cuda, dev, kind, q.reshape(len(q), -1), nq * np.arange(seqs + 1), [n] * seqs, heads, 1.0,
                           max_kv=max_kv, repeat=2)
        score = 6 * qq[0, 0]
        share = (np.arange(n - nq, n) * np.exp(-score))[:, None]
        want = np.tile(3 * share / (1 + share), (seqs, 1))
        rel = 2.0 ** -12 + np.expm1(2.0 ** -18 * score) + 2.0 ** -13 + TYPES[kind][2] / 2
        assert (np.abs(got - want) <= rel * want + 3 * n * 2.0 ** -32 / (1 + share[0, 0])).all(), (want[0, 0], got[0, 0])


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rising", [False, True])
def test_random_long_caches(torch_cuda, kind, D, rising):
    """140000 positions of each of 1800 sequences, two kinds of queries; sinks, and largest scores that come later and later."""
    rng = np.random.default_rng(D + rising)
    n, heads, seqs = 140000, 4, 1800
    h = random_pages(rng, [n], 1, D, 256)
    q = rng.standard_normal((2, heads * D)) * 0.3
    if rising:  # as in test_kv4_long_sums_gpu
        for i in range(-(-n // 256)):
            h.pool[h.table[0, i], 0, :, 32 * D:33 * D] = (8 + 9 * 256 * i // n) << 2
        q = np.abs(q)
        h.pool[..., :16 * D] &= 0x77
    table = h.table
    h.table = np.repeat(table, seqs, 0)
    dev = Dev(torch_cuda, h)
    sinks = rng.standard_normal(heads)
    got, qq = run_attn(torch_cuda, dev, kind, np.tile(q, (seqs // 2, 1)), np.arange(seqs + 1), [n] * seqs, heads, D ** -0.5, 0,
                       sinks, repeat=2)
    assert (got.reshape(-1, 2, heads * D) == got[:2]).all()
    h.table = np.repeat(table, 2, 0)
    check_attn(got[:2], qq[:2], dev, kind, [0, 1, 2], [n, n], heads, D ** -0.5, 0, sinks)
