"""mg_kv4_attn calls that mix kinds of sequences: single tokens behind long
caches next to prompt chunks, over several key/value heads; more sequences
than the many-row kernel orders by their work.  Tolerances as in
test_kv4_gpu; every call twice, for the same bits."""
import numpy as np
import pytest

from tests import kv4_ref as ref
from tests.test_kv4_gpu import Dev, check_attn, filled, run_attn, tables

pytestmark = pytest.mark.gpu


def random_pages(rng, lengths, n_kv, D, page):
    """A cache of random codes and scales around 1, the bytes straight into the pages."""
    t, n_pages = tables(rng, lengths, page)
    h = ref.Cache(n_kv, D, page, t, n_pages, 0xFF)
    h.pool[..., :32 * D] = rng.integers(0, 256, h.pool[..., :32 * D].shape, dtype=np.uint8)
    h.pool[..., 32 * D:] = rng.integers(48, 62, h.pool[..., 32 * D:].shape, dtype=np.uint8)
    return h


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D,window", [(64, 0), (64, 300), (128, 0)])
def test_single_tokens_and_chunks(torch_cuda, kind, D, window):
    rng = np.random.default_rng(D + window)
    lengths, nq = [3000, 5000, 700, 1, 0, 2500, 33], [1, 1, 70, 1, 1, 20, 0]
    dev = Dev(torch_cuda, random_pages(rng, lengths, 3, D, 64))
    qs = np.concatenate([[0], np.cumsum(nq)])
    q = rng.standard_normal((qs[-1], 12 * D)) * 0.3
    sinks = rng.standard_normal(12)
    got, q = run_attn(torch_cuda, dev, kind, q, qs, lengths, 12, D ** -0.5, window, sinks, repeat=2)
    check_attn(got, q, dev, kind, qs, lengths, 12, D ** -0.5, window, sinks)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("n", [511, 512, 513, 700])
def test_many_sequences_of_all_kinds(torch_cuda, kind, n):
    rng = np.random.default_rng(n)
    nq = rng.choice([0, 1, 1, 1, 2], n)
    nq[rng.integers(0, n, 5)] = [40, 17, 60, 33, 21]
    lengths = [int(x) for x in np.maximum(rng.integers(0, 90, n), nq)]
    dev = Dev(torch_cuda, filled(rng, lengths, 1, 64, 32))
    qs = np.concatenate([[0], np.cumsum(nq)])
    q = rng.standard_normal((qs[-1], 4 * 64))
    got, q = run_attn(torch_cuda, dev, kind, q, qs, lengths, 4, 0.125, repeat=2)
    check_attn(got, q, dev, kind, qs, lengths, 4, 0.125)
