"""mg_logprobs against 64 bits (tests/kv4_ref.py).

Tolerances: a difference x - m is one fp32 rounding (2^-24 of it); the terms
of the sum are off by 2^-22 (1 + |d|) each, those that matter have |d| < 20,
and sums of positive terms keep that: z within 2^-17.  The entropy adds the
same for its weighted sum, times 1 + H.  Alternatives are exact: the device
compares the logits themselves."""
import numpy as np
import pytest

from midge_b200 import abi
from tests import kv4_ref as ref

pytestmark = pytest.mark.gpu
ACT = {"f32": 0, "f16": 1, "bf16": 2}
TOL = 2.0 ** -17


def run(torch, x, ids, top, kind, pad=0, stream=None):
    dt = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[kind]
    n, V = x.shape
    xd = torch.from_numpy(np.pad(x.astype(np.float32), ((0, 0), (0, pad)), constant_values=1e4)).cuda().to(dt)
    idd = torch.from_numpy(np.ascontiguousarray(ids, np.int32)).cuda()
    n_ids = ids.shape[1]
    lp = torch.full((n, n_ids), 7.0, device="cuda")
    ent = torch.full((n,), 7.0, device="cuda")
    ai, al = torch.full((n, top), 7, dtype=torch.int32, device="cuda"), torch.full((n, top), 7.0, device="cuda")
    need = abi.check_size(abi.lib.mg_logprobs_work(V, n, top))
    work = torch.zeros(max(16, need), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    last = None
    for _ in range(2):
        abi.check(abi.lib.mg_logprobs(ACT[kind], xd.data_ptr(), V + pad, V, n, idd.data_ptr() if n_ids else None, n_ids,
                                      top, lp.data_ptr() if n_ids else None, ent.data_ptr(),
                                      ai.data_ptr() if top else None, al.data_ptr() if top else None, work.data_ptr(),
                                      work.numel(), stream))
        torch.cuda.synchronize()
        got = [t.cpu().numpy() for t in (lp, ent, ai, al)]
        if last is not None:
            assert all(np.array_equal(a, b, equal_nan=True) for a, b in zip(got, last))  # the same bits every time
        last = got
    return last, xd.float().cpu().numpy()[:, :V]


def check(got, x, ids, top):
    lp, ent, ai, al = got
    for r in range(len(x)):
        wlp, went, order, wal = ref.logprobs(x[r], ids[r], top)
        wlp, wal = wlp.astype(np.float32).astype(np.float64), wal.astype(np.float32).astype(np.float64)  # what f32 holds
        fin = np.isfinite(wlp)
        assert np.array_equal(fin, np.isfinite(lp[r])) and np.array_equal(wlp[~fin], lp[r][~fin])
        assert (np.abs(lp[r][fin] - wlp[fin]) <= TOL + 2.0 ** -22 * np.abs(wlp[fin])).all()
        assert abs(ent[r] - went) <= 2 * TOL * (1 + went)
        n = len(order)
        assert np.array_equal(ai[r][:n], order) and (ai[r][n:] == -1).all() and (al[r][n:] == -np.inf).all()
        fin = np.isfinite(wal)
        assert np.array_equal(wal[~fin], al[r][:n][~fin])
        assert (np.abs(al[r][:n][fin] - wal[fin]) <= TOL + 2.0 ** -22 * np.abs(wal[fin])).all()


@pytest.mark.parametrize("kind", list(ACT))
@pytest.mark.parametrize("V", [1, 2, 31, 33, 1000, 4097, 50001, 201088])
@pytest.mark.parametrize("rows,top,n_ids,pad", [(1, 5, 1, 0), (3, 32, 4, 1), (7, 1, 0, 8), (200, 20, 1, 0), (2, 0, 2, 3)])
def test_logprobs(torch_cuda, kind, V, rows, top, n_ids, pad):
    if rows * V > 8_000_000:
        rows = 8_000_000 // V
    rng = np.random.default_rng(V + rows)
    x = rng.standard_normal((rows, V)) * 2
    x[np.arange(rows)[:, None], rng.integers(0, V, (rows, 4))] += rng.uniform(0, 14, (rows, 4))
    ids = rng.integers(0, V, (rows, n_ids))
    if n_ids > 1:
        ids[:, 1] = [-1, V, 2 ** 31 - 1, 0][rows % 4]
    got, x = run(torch_cuda, x, ids, top, kind, pad)
    check(got, x, ids, top)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("V", [513, 70003])
@pytest.mark.parametrize("rows", [1, 300])
def test_orders_and_ties(torch_cuda, kind, V, rows):
    """Rows that rise, fall, are all alike, repeat a few values, have their
    largest in one place after another."""
    rng = np.random.default_rng(V)
    kinds = [np.linspace(-20, 20, V), np.linspace(20, -20, V), np.zeros(V), np.full(V, -3e38), rng.integers(0, 3, V),
             np.where(np.arange(V) % 97 == 0, 5.0, 0.0), np.where(np.arange(V) > V - 40, np.arange(V) - V, -50.0)]
    if rows > 1:
        x = np.stack([kinds[r % len(kinds)] for r in range(8)])
        x = np.concatenate([x, rng.standard_normal((rows - 8, V))]) if V < 1000 else x
    else:
        x = np.stack(kinds[:1])
    for top in (1, 32):
        for row in ([x] if rows > 1 else [k[None] for k in kinds]):
            ids = rng.integers(0, V, (len(row), 1))
            got, xx = run(torch_cuda, row, ids, top, kind)
            check(got, xx, ids, top)


@pytest.mark.parametrize("V,rows", [(300, 6), (201088, 1), (60000, 6)])
def test_masked_rows(torch_cuda, V, rows):
    """Banned tokens (-infinity), rows of nothing else, NaN among the logits,
    fewer possible tokens than alternatives."""
    rng = np.random.default_rng(V)
    for which in range(5):
        x = rng.standard_normal((rows, V)).astype(np.float32)
        x[:, V // 3:V // 2] = -np.inf
        if which == 1:
            x[0] = -np.inf
        if which == 2:
            x[0] = -np.inf
            x[0, [7, V - 1]] = [1.0, 1.0]
        if which == 3:
            x[0, ::3] = np.nan
            x[0, 0] = np.nan
        if which == 4:
            x[0] = -3.4e38
            x[0, 11] = 3.4e38
        ids = np.stack([np.array([1, V // 3, V - 1])] * rows)
        got, xx = run(torch_cuda, x, ids, 8, "f32")
        check(got, xx, ids, 8)


@pytest.mark.parametrize("kind", list(ACT))
@pytest.mark.parametrize("V,rows", [(5000, 200), (201088, 2)])
def test_few_tokens_allowed(torch_cuda, kind, V, rows):
    """Constrained decoding: 0 to 40 possible tokens, everything else banned."""
    rng = np.random.default_rng(V)
    x = np.full((rows, V), -np.inf, np.float32)
    for r in range(rows):
        k = r % 41 if rows > 2 else 7 + r * 30
        x[r, rng.choice(V, k, replace=False)] = rng.integers(-8, 8, k)
    ids = rng.integers(0, V, (rows, 1))
    got, xx = run(torch_cuda, x, ids, 32, kind)
    check(got, xx, ids, 32)


def test_plus_infinity_is_nan(torch_cuda):
    x = np.zeros((2, 40), np.float32)
    x[0, 3] = np.inf
    (lp, ent, ai, al), _ = run(torch_cuda, x, np.array([[0], [0]]), 2, "f32")
    assert np.isnan(lp[0, 0]) and np.isnan(ent[0]) and ai[0, 0] == 3
    assert abs(lp[1, 0] + np.log(40)) < 1e-5 and abs(ent[1] - np.log(40)) < 1e-5


def test_on_a_stream(torch_cuda):
    rng = np.random.default_rng(1)
    st = torch_cuda.cuda.Stream()
    x = rng.standard_normal((5, 3000))
    ids = rng.integers(0, 3000, (5, 1))
    got, x = run(torch_cuda, x, ids, 3, "f32", stream=st.cuda_stream)
    check(got, x, ids, 3)
