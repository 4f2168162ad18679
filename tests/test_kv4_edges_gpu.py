"""Corners of the 4-bit cache operators and of token scoring that ordinary
calls do not meet: pools and rows whose offsets pass 32 bits, a max_q below a
sequence's queries, windows up to the largest int, negative and zero scales.
Tolerances as in test_kv4_gpu and test_logprobs_gpu, whose helpers these are."""
import numpy as np
import pytest

from midge_b200 import abi
from tests import kv4_ref as ref
from tests.test_kv4_gpu import TYPES, Dev, check_attn, filled, run_append, run_attn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nq", [1, 3, 40])
@pytest.mark.parametrize("kind", list(TYPES))
def test_pool_beyond_32_bits(torch_cuda, kind, nq):
    """Pages in the last bytes of a pool of 5 GB, by append, read and attention."""
    torch = torch_cuda
    rng = np.random.default_rng(nq)
    h = filled(rng, [100, 130], 2, 128, 64)
    dev = Dev(torch, h)
    one = h.pool[0].size
    n_pages = 5 * 2 ** 30 // one
    pool = torch.empty(n_pages, one, dtype=torch.uint8, device="cuda")
    small = h.pool.shape[0]
    pool[n_pages - small:] = dev.pool.reshape(small, one)
    inside = (h.table >= 0) & (h.table < small)
    dev.table = torch.from_numpy(np.where(inside, h.table + (n_pages - small), h.table).astype(np.int32)).cuda()
    dev.c.n_pages, dev.c.pages, dev.c.table = n_pages, pool.data_ptr(), dev.table.data_ptr()
    n = 2 * nq
    seq, pos = np.repeat([0, 1], nq), np.concatenate([np.arange(100 - nq, 100), np.arange(130 - nq, 130)])
    k, v, q = (rng.standard_normal((n, w)) for w in (256, 256, 1024))
    _, (_, kk, vv) = run_append(torch, dev, kind, q, k, v, seq, pos, 8)
    for i in range(n):
        for hd in range(2):
            h.store(seq[i], pos[i], hd, kk[i].reshape(2, 128)[hd], True)
            h.store(seq[i], pos[i], hd, vv[i].reshape(2, 128)[hd], False)
    assert np.array_equal(pool[n_pages - small:].cpu().numpy(), h.pool.reshape(small, one))
    sd, pd = (torch.from_numpy(x.astype(np.int32)).cuda() for x in (seq, pos))
    back = torch.empty(n, 256, device="cuda")
    abi.check(abi.lib.mg_kv4_read(dev.ref(), 0, n, sd.data_ptr(), pd.data_ptr(), back.data_ptr(), 256, None, 0, None))
    want = np.stack([np.concatenate([h.load(seq[i], pos[i] + 1, hd, True)[pos[i]] for hd in range(2)]) for i in range(n)])
    assert np.array_equal(back.cpu().numpy(), want)
    qs = np.array([0, nq, n])
    got, qq = run_attn(torch, dev, kind, q, qs, [100, 130], 8, 0.09)
    check_attn(got, qq, dev, kind, qs, [100, 130], 8, 0.09)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("nq,max_q", [([5, 2], 2), ([3, 1], 1), ([30, 9], 20), ([200, 70], 70)])
def test_rows_beyond_max_q_are_left(torch_cuda, kind, nq, max_q):
    rng = np.random.default_rng(max_q)
    lengths = [210, 77]
    dev = Dev(torch_cuda, filled(rng, lengths, 2, 64, 32))
    qs = np.concatenate([[0], np.cumsum(nq)])
    got, q = run_attn(torch_cuda, dev, kind, rng.standard_normal((qs[-1], 512)), qs, lengths, 8, 0.125, max_q=max_q)
    want, bs, bv = ref.attention(dev.host, q, qs, lengths, 8, 0.125, 0, None)
    left = np.concatenate([np.arange(n) >= max_q for n in nq])
    assert left.any() and (got[left] == 7.0).all()
    fixed = got.copy()
    fixed[left] = want.reshape(got.shape)[left]
    check_attn(fixed, q, dev, kind, qs, lengths, 8, 0.125)


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 40, 2 ** 30])
@pytest.mark.parametrize("nq", [[1, 9, 0], [2, 40, 1], [120, 100, 300]])
def test_windows_beyond_the_cache(torch_cuda, window, nq):
    """As no window, for sequences with more queries than positions too."""
    rng = np.random.default_rng(nq[0])
    lengths = [90, 5, 333]
    dev = Dev(torch_cuda, filled(rng, lengths, 2, 64, 32))
    qs = np.concatenate([[0], np.cumsum(nq)])
    got, q = run_attn(torch_cuda, dev, "f32", rng.standard_normal((qs[-1], 512)), qs, lengths, 8, 0.125, window)
    check_attn(got, q, dev, "f32", qs, lengths, 8, 0.125)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("nq", [[1, 1], [60, 40]])
def test_negative_and_zero_scale(torch_cuda, kind, nq):
    """A negative scale is the same as negated queries; zero weighs alike all that a query sees."""
    rng = np.random.default_rng(8)
    lengths = [140, 61]
    dev = Dev(torch_cuda, filled(rng, lengths, 2, 64, 32))
    qs = np.concatenate([[0], np.cumsum(nq)])
    q0 = rng.standard_normal((qs[-1], 512))
    got, q = run_attn(torch_cuda, dev, kind, q0, qs, lengths, 8, -0.2)
    check_attn(got, -q, dev, kind, qs, lengths, 8, 0.2)
    got, q = run_attn(torch_cuda, dev, kind, q0, qs, lengths, 8, 0.0)
    check_attn(got, q, dev, kind, qs, lengths, 8, 0.0)


def test_logits_rows_beyond_32_bits(torch_cuda):
    """Two rows 2^32 + 8 elements apart."""
    torch = torch_cuda
    V, ld = 5003, 2 ** 32 + 8
    x = torch.empty(ld + V, dtype=torch.float16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    rows = torch.randn(2, V, device="cuda", generator=g).half() * 3
    x[:V], x[ld:] = rows[0], rows[1]
    ids = torch.tensor([[4], [5002]], dtype=torch.int32, device="cuda")
    lp, ent = torch.empty(2, 1, device="cuda"), torch.empty(2, device="cuda")
    ai, al = torch.empty(2, 4, dtype=torch.int32, device="cuda"), torch.empty(2, 4, device="cuda")
    work = torch.zeros(abi.check_size(abi.lib.mg_logprobs_work(V, 2, 4)), dtype=torch.uint8, device="cuda")
    abi.check(abi.lib.mg_logprobs(1, x.data_ptr(), ld, V, 2, ids.data_ptr(), 1, 4, lp.data_ptr(), ent.data_ptr(),
                                  ai.data_ptr(), al.data_ptr(), work.data_ptr(), work.numel(), None))
    want = torch.log_softmax(rows.double(), -1)
    torch.cuda.synchronize()
    # fp32 sums of V terms: 2^-17 of a log probability of some 10 and of the entropy covers them
    assert torch.allclose(lp[:, 0].double(), want[[0, 1], [4, 5002]], rtol=0, atol=1e-4)
    assert torch.allclose(ent.double(), -(want.exp() * want).sum(-1), rtol=0, atol=1e-4)
    top = want.topk(4)
    assert torch.allclose(al.double(), top.values, rtol=0, atol=1e-4)
    assert torch.equal(want.gather(1, ai.long()), top.values)
