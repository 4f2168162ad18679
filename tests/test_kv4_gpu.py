"""The 4-bit paged cache on the device: mg_kv4_append, mg_kv4_read and
mg_kv4_attn through the C ABI against the 64-bit restatement in kv4_ref.

Tolerances, from the arithmetic:
  * stored bytes: exact (keys are computed in 64 bits, values only compared);
  * queries out: the norm and the rotation are fp32 (relative 2^-20 of the
    head's largest magnitude covers the sum of 128 squares and six roundings),
    then one rounding to the type (2^-11 f16, 2^-8 bf16 units);
  * attention: a query is kept to 2^-21 of its row's largest magnitude or
    better, so a score is off by at most ds = 2^-19 max_t scale sum |q k| and a
    weight by e^(2 ds); fp32 sums, the exponential and 22-bit weights add
    2^-18; all of it times max |v|.  f16 and bf16 round the weights to f16
    (2^-10 max |v|) and the result to the type.
"""
import ctypes as C

import numpy as np
import pytest

from midge_b200 import abi
from tests import kv4_ref as ref

pytestmark = pytest.mark.gpu
TYPES = {"f32": (0, np.float32, 0.0), "f16": (1, np.float16, 2.0 ** -11), "bf16": (2, None, 2.0 ** -8)}


def to_dev(torch, x, kind):
    t = torch.from_numpy(np.ascontiguousarray(x, np.float32)).cuda()
    return t.to({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[kind])


class Dev:
    """A cache on the device with the host copy it started from."""

    def __init__(self, torch, host, stray=False):
        self.torch, self.host = torch, host
        self.pool = torch.from_numpy(host.pool.copy()).cuda()
        self.table = torch.from_numpy(host.table).cuda()
        self.c = abi.MgKv4(n_kv_heads=host.n_kv, head_dim=host.D, page_size=host.page, n_seqs=host.table.shape[0],
                           n_pages=host.pool.shape[0], pages=self.pool.data_ptr(), table=self.table.data_ptr(),
                           ld_table=host.table.shape[1])

    def ref(self):
        return C.byref(self.c)


def tables(rng, lengths, page, spare=1, width=None):
    """Page tables in random order; unused entries point outside the pool."""
    need = [-(-n // page) for n in lengths]
    order = rng.permutation(sum(need) + spare)
    t = np.full((len(lengths), width or max(1, max(need))), -7, np.int32)
    t[:, 1::2] = 1 << 30
    at = 0
    for i, n in enumerate(need):
        t[i, :n] = order[at:at + n]
        at += n
    return t, sum(need) + spare


def filled(rng, lengths, n_kv, D, page, fill=0xFF):
    """A cache with the given numbers of positions; every byte that no
    position owns is `fill` (0xFF: codes -6 and NaN scales)."""
    t, n_pages = tables(rng, lengths, page)
    h = ref.Cache(n_kv, D, page, t, n_pages, fill)
    for s, n in enumerate(lengths):
        for head in range(n_kv):
            k, v = rng.standard_normal((n, D)), rng.standard_normal((n, D))
            k[:, 5] *= 5
            for p in range(n):
                h.store(s, p, head, k[p], True)
                h.store(s, p, head, v[p], False)
    return h


# ------------------------------------------------------------------ append
def run_append(torch, dev, kind, q, k, v, seq, pos, heads, qn=None, kn=None, co=None, si=None, pad=0, stream=None):
    """Rows with `pad` extra elements each; returns q_out rows."""
    act = TYPES[kind][0]
    n, kvd = k.shape
    D = dev.host.D

    def rows(x):
        return to_dev(torch, np.pad(x, ((0, 0), (0, pad))), kind)

    qd, kd, vd = rows(q), rows(k), rows(v)
    qo = torch.full((n, heads * D + pad), 7.0, device="cuda", dtype=qd.dtype)
    f = [None if a is None else torch.from_numpy(np.ascontiguousarray(a, np.float32)).cuda() for a in (qn, kn, co, si)]
    ip = [None if a is None else torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda() for a in (seq, pos)]
    P = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    torch.cuda.synchronize()
    abi.check(abi.lib.mg_kv4_append(dev.ref(), act, n, heads, P(qd), heads * D + pad, P(kd), kvd + pad, P(vd),
                                    kvd + pad, P(f[0]), P(f[1]), 1e-6, P(f[2]), P(f[3]),
                                    0 if co is None else co.shape[0], P(ip[0]), P(ip[1]), P(qo), heads * D + pad,
                                    stream))
    torch.cuda.synchronize()
    return qo.float().cpu().numpy(), [t.float().cpu().numpy().astype(np.float64) for t in (qd, kd, vd)]


def turned(x, w, pos, co, si, D, eps=1e-6):
    """Norm and rotation of rows [n, heads * D] in 64 bits."""
    y = x.reshape(len(x), -1, D).astype(np.float64)
    if w is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * w.astype(np.float64)
    if co is not None:
        c, s = co[pos].astype(np.float64)[:, None], si[pos].astype(np.float64)[:, None]
        a, b = y[..., :D // 2], y[..., D // 2:]
        y = np.concatenate([a * c - b * s, b * c + a * s], -1)
    return y


def rope(n, D):
    a = np.arange(n)[:, None] * 10000.0 ** (-np.arange(D // 2) / (D // 2))
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("D,heads,n_kv", [(64, 8, 2), (128, 5, 1), (64, 3, 3), (128, 8, 4)])
@pytest.mark.parametrize("norm,turn,pad", [(True, True, 0), (False, True, 8), (True, False, 1), (False, False, 3)])
def test_append_stores_exact_bytes(torch_cuda, kind, D, heads, n_kv, norm, turn, pad):
    rng = np.random.default_rng(D + heads + 10 * norm + turn)
    page, count = 64, [1, 37, 70]
    first = [63, 0, 30]
    lengths = [a + b for a, b in zip(first, count)]
    t, n_pages = tables(rng, lengths, page)
    h = ref.Cache(n_kv, D, page, t, n_pages, 0xA5)
    dev = Dev(torch_cuda, h)
    seq = np.repeat(np.arange(3), count)
    pos = np.concatenate([f + np.arange(c) for f, c in zip(first, count)])
    order = rng.permutation(len(pos))  # tokens in any order
    seq, pos = seq[order], pos[order]
    n = len(pos)
    q, k, v = (rng.standard_normal((n, w * D)) * np.exp(rng.uniform(-4, 4, (n, 1))) for w in (heads, n_kv, n_kv))
    v[0] = 0.0
    qn, kn = (1 + 0.2 * rng.standard_normal((2, D))).astype(np.float32) if norm else (None, None)
    co, si = rope(max(lengths), D) if turn else (None, None)
    got, (q, k, v) = run_append(torch_cuda, dev, kind, q, k, v, seq, pos, heads, qn, kn, co, si, pad)
    q, k, v = q[:, :heads * D], k[:, :n_kv * D], v[:, :n_kv * D]
    kk, vv = turned(k, kn, pos, co, si, D), v.reshape(n, n_kv, D)
    for i in range(n):
        for hd in range(n_kv):
            h.store(seq[i], pos[i], hd, kk[i, hd], True)
            h.store(seq[i], pos[i], hd, vv[i, hd], False)
    assert np.array_equal(dev.pool.cpu().numpy(), h.pool)  # also: nothing else was touched
    want = turned(q, qn, pos, co, si, D)
    big = np.abs(want).max(-1, keepdims=True)
    tol = 2.0 ** -20 * big + TYPES[kind][2] * np.abs(want) + (2.0 ** -25 if kind == "f16" else 0)
    assert (np.abs(got[:, :heads * D].reshape(n, heads, D) - want) <= tol).all()
    assert (got[:, heads * D:] == 7.0).all()


def test_append_skips_padding_and_strays(torch_cuda):
    rng = np.random.default_rng(5)
    t, n_pages = tables(rng, [100, 100], 32, width=4)
    t[:] = np.arange(8).reshape(2, 4)
    h = ref.Cache(2, 64, 32, t, 8, 0x3C)
    dev = Dev(torch_cuda, h)
    seq = np.array([0, 0, 1, 2, -1, 0, 1])
    pos = np.array([5, -1, 128, 3, 3, 60, 1 << 30])  # 128 = beyond the table, 60 = beyond the rotation
    n = len(pos)
    q, k, v = rng.standard_normal((3, n, 128))
    co, si = rope(50, 64)
    got, (q, k, v) = run_append(torch_cuda, dev, "f32", q, k, v, seq, pos, 2, co=co, si=si)
    kk = turned(k, None, np.minimum(np.maximum(pos, 0), 49), co, si, 64)
    for hd in range(2):
        h.store(0, 5, hd, kk[0, hd], True)
        h.store(0, 5, hd, v[0].reshape(2, 64)[hd], False)
    assert np.array_equal(dev.pool.cpu().numpy(), h.pool)
    assert (got[1:] == 7.0).all() and not (got[0] == 7.0).any()


def test_append_extreme_numbers(torch_cuda):
    """Infinities saturate, NaN is 0, subnormals and ties round as described."""
    rng = np.random.default_rng(6)
    h = ref.Cache(1, 64, 32, [[0]], 1)
    dev = Dev(torch_cuda, h)
    v = rng.standard_normal((6, 64)) * 1e-6
    v[0, :40] = [np.inf, -np.inf, np.nan, 1e30, -1e-30, 0.0, -0.0, 3.0] * 5
    v[1] = 1e38
    v[2] = 6 * np.where(np.arange(64) % 2, 1, -1) / 8.0 ** rng.integers(0, 3, 64)
    v[3, :9] = [6, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, -5]
    v[4] = 2.0 ** -16 * rng.uniform(-1, 1, 64)
    k = np.flip(v, 1).copy()
    k[0] = np.nan_to_num(k[0], nan=1.0, posinf=1.0, neginf=-1.0)
    run_append(torch_cuda, dev, "f32", np.zeros((6, 64)), k, v, None, np.arange(6), 1)
    v32, k32 = v.astype(np.float32).astype(np.float64), k.astype(np.float32).astype(np.float64)
    for i in range(6):
        h.store(0, i, 0, k32[i], True)
        h.store(0, i, 0, v32[i], False)
    assert np.array_equal(dev.pool.cpu().numpy(), h.pool)
    assert np.isfinite(h.load(0, 6, 0, False)).all()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("D,n_kv,page", [(64, 3, 32), (128, 2, 96)])
def test_read_is_exact(torch_cuda, kind, D, n_kv, page):
    torch = torch_cuda
    rng = np.random.default_rng(D)
    h = filled(rng, [33, 100], n_kv, D, page)
    dev = Dev(torch, h)
    seq = np.array([0, 1, 1, 1, 0, 1, 0, 5], np.int32)
    pos = np.array([32, 99, 0, 64, 0, 31, -1, 0], np.int32)
    sd, pd = torch.from_numpy(seq).cuda(), torch.from_numpy(pos).cuda()
    dt = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[kind]
    k, v = torch.full((8, n_kv * D + 5), 9.0, dtype=dt, device="cuda"), torch.full((8, n_kv * D), 9.0, dtype=dt, device="cuda")
    torch.cuda.synchronize()
    abi.check(abi.lib.mg_kv4_read(dev.ref(), TYPES[kind][0], 8, sd.data_ptr(), pd.data_ptr(), k.data_ptr(),
                                  n_kv * D + 5, v.data_ptr(), n_kv * D, None))
    abi.check(abi.lib.mg_kv4_read(dev.ref(), TYPES[kind][0], 8, sd.data_ptr(), pd.data_ptr(), None, 0, v.data_ptr(),
                                  n_kv * D, None))
    torch.cuda.synchronize()
    k, v = k.double().cpu().numpy(), v.double().cpu().numpy()
    for i in range(8):
        for hd in range(n_kv):
            for got, keys in ((k, True), (v, False)):
                want = np.zeros(D) if pos[i] < 0 or seq[i] > 1 else h.load(seq[i], pos[i] + 1, hd, keys)[-1]
                assert np.array_equal(got[i, hd * D:(hd + 1) * D], want)
    assert (k[:, n_kv * D:] == 9.0).all()


# --------------------------------------------------------------- attention
def run_attn(torch, dev, kind, q, q_start, kv_len, heads, scale, window=0, sinks=None, pad=0, max_q=None, max_kv=None,
             repeat=1, work=None, stream=None):
    act = TYPES[kind][0]
    D = dev.host.D
    qd = to_dev(torch, np.pad(q, ((0, 0), (0, pad))), kind)
    out = torch.full((q.shape[0], heads * D + pad), 7.0, device="cuda", dtype=qd.dtype)
    qs, kl = (torch.from_numpy(np.asarray(x, np.int32)).cuda() for x in (q_start, kv_len))
    sk = None if sinks is None else torch.from_numpy(np.asarray(sinks, np.float32)).cuda()
    mq = max_q or max(1, int(np.diff(q_start).max()))
    mk = int(max(kv_len)) if max_kv is None else max_kv
    need = abi.check_size(abi.lib.mg_kv4_attn_work(dev.ref(), heads, mq, mk))
    if work is None:
        work = torch.zeros(max(16, need), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    res = []
    for _ in range(repeat):
        abi.check(abi.lib.mg_kv4_attn(dev.ref(), act, heads, qd.data_ptr(), heads * D + pad, qs.data_ptr(),
                                      kl.data_ptr(), mq, mk, scale, window, None if sk is None else sk.data_ptr(),
                                      out.data_ptr(), heads * D + pad, work.data_ptr(), work.numel(), stream))
        torch.cuda.synchronize()
        res.append(out.float().cpu().numpy())
    for r in res[1:]:
        assert np.array_equal(r, res[0])  # the same bits every time
    assert (res[0][:, heads * D:] == 7.0).all()
    return res[0][:, :heads * D], qd.float().cpu().numpy().astype(np.float64)[:, :heads * D]


def check_attn(got, q, dev, kind, q_start, kv_len, heads, scale, window=0, sinks=None):
    want, bs, bv = ref.attention(dev.host, q, q_start, kv_len, heads, scale, window, sinks)
    ds = 2.0 ** -19 * bs
    tol = (np.expm1(2 * ds) + 2.0 ** -18) * bv
    if kind != "f32":
        tol = tol + 2.0 ** -10 * bv
    tol = tol[..., None] + TYPES[kind][2] * np.abs(want) + (2.0 ** -24 if kind == "f16" else 0)
    err = np.abs(got.reshape(want.shape) - want)
    assert (err <= tol).all(), float((err - tol).max())


CASES = [
    # lengths, queries, page: single tokens; lengths around tiles and pages; empty caches; idle sequences
    ([1, 2, 31, 32, 33, 64, 65, 95], [1] * 8, 32),
    ([0, 5, 0, 200], [1, 1, 0, 1], 64),
    ([257], [1], 256),
    ([5, 40, 300], [5, 2, 3], 64),             # a few tokens, one sequence with nothing before them
    ([3, 130], [9, 12], 96),                   # more queries than positions: the first see nothing
    ([150, 64, 129], [70, 64, 1], 32),         # chunks
    ([400], [400], 128),
]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("D,heads,n_kv", [(64, 16, 2), (128, 8, 2), (64, 3, 3), (128, 5, 1), (64, 48, 2)])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention(torch_cuda, kind, D, heads, n_kv, case):
    lengths, nq, page = CASES[case]
    rng = np.random.default_rng(100 * case + D + heads)
    dev = Dev(torch_cuda, filled(rng, lengths, n_kv, D, page))
    qs = np.concatenate([[0], np.cumsum(nq)])
    q = rng.standard_normal((qs[-1], heads * D)) * 1.5
    sinks = rng.standard_normal(heads) if case % 2 else None
    got, q = run_attn(torch_cuda, dev, kind, q, qs, lengths, heads, D ** -0.5, 0, sinks, pad=case, repeat=2)
    check_attn(got, q, dev, kind, qs, lengths, heads, D ** -0.5, 0, sinks)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("window", [1, 7, 32, 100, 5000])
@pytest.mark.parametrize("nq", [[1, 1, 1], [4, 1, 6], [60, 33, 80]])
def test_attention_window(torch_cuda, kind, window, nq):
    rng = np.random.default_rng(window + nq[0])
    lengths = [90, 33, 333]
    dev = Dev(torch_cuda, filled(rng, lengths, 2, 64, 32))
    qs = np.concatenate([[0], np.cumsum(nq)])
    q = rng.standard_normal((qs[-1], 8 * 64))
    sinks = rng.standard_normal(8)
    got, q = run_attn(torch_cuda, dev, kind, q, qs, lengths, 8, 0.125, window, sinks)
    check_attn(got, q, dev, kind, qs, lengths, 8, 0.125, window, sinks)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n", [1, 40])
def test_attention_peaked_and_large(torch_cuda, kind, n):
    """Scores in the hundreds (one position takes everything), queries of very
    different sizes, sinks of -infinity and far above every score."""
    rng = np.random.default_rng(n)
    dev = Dev(torch_cuda, filled(rng, [200, 77], 2, 64, 64))
    qs = np.array([0, n, 2 * n])
    q = rng.standard_normal((2 * n, 8, 64))
    q *= np.array([1e-6, 1e-2, 1, 30, 60, 1, 1, 100])[None, :, None]
    sinks = np.array([-np.inf, 0, -np.inf, 5, 500, 80, -200, -np.inf])
    got, q = run_attn(torch_cuda, dev, kind, q.reshape(2 * n, -1), qs, [200, 77], 8, 0.3, 0, sinks)
    check_attn(got, q, dev, kind, qs, [200, 77], 8, 0.3, 0, sinks)
    assert np.isfinite(got).all()


def test_attention_nothing_seen(torch_cuda):
    """Empty sequences give zeros, with sinks and without, for any kind of call."""
    rng = np.random.default_rng(3)
    h = filled(rng, [0, 0], 2, 64, 32)
    dev = Dev(torch_cuda, h)
    for nq in (1, 3, 50):
        for sinks in (None, np.zeros(8)):
            qs = np.array([0, nq, 2 * nq])
            got, _ = run_attn(torch_cuda, dev, "f32", rng.standard_normal((2 * nq, 512)), qs, [0, 0], 8, 1.0, 0, sinks)
            assert (got == 0).all()


@pytest.mark.parametrize("lengths,nq", [([5000], [1]), ([4999, 12], [3, 3]), ([3000], [40]), ([2100, 1], [200, 1])])
@pytest.mark.parametrize("kind,D", [("f32", 64), ("f32", 128), ("bf16", 128)])
def test_attention_long(torch_cuda, kind, D, lengths, nq):
    """Long enough that several blocks share a sequence; the hint max_kv from
    far too small to far too large gives the same within the tolerance."""
    rng = np.random.default_rng(sum(lengths))
    t, n_pages = tables(rng, lengths, 128)
    h = ref.Cache(1, D, 128, t, n_pages, 0xFF)
    # random codes and scales, the bytes straight into the pages
    codes = rng.integers(0, 256, h.pool[..., :32 * D].shape, dtype=np.uint8)
    h.pool[..., :32 * D] = codes
    h.pool[..., 32 * D:] = rng.integers(48, 62, h.pool[..., 32 * D:].shape, dtype=np.uint8)
    dev = Dev(torch_cuda, h)
    qs = np.concatenate([[0], np.cumsum(nq)])
    q = rng.standard_normal((qs[-1], 4 * D))
    for mk in (0, None, 200000):
        got, qq = run_attn(torch_cuda, dev, kind, q, qs, lengths, 4, D ** -0.5, 0, rng.standard_normal(4) * 0 + 1,
                           max_kv=mk, repeat=3)
        check_attn(got, qq, dev, kind, qs, lengths, 4, D ** -0.5, 0, np.ones(4))


def test_workspace_reused_between_sizes_and_streams(torch_cuda):
    """One workspace for calls of several sizes in turn, on a stream of its own."""
    torch = torch_cuda
    rng = np.random.default_rng(8)
    dev = Dev(torch, filled(rng, [700, 20], 1, 64, 64))
    need = max(abi.check_size(abi.lib.mg_kv4_attn_work(dev.ref(), 4, n, 700)) for n in (1, 5, 50))
    work = torch.zeros(need, dtype=torch.uint8, device="cuda")
    st = torch.cuda.Stream()
    for nq in ([1, 1], [5, 2], [1, 0], [50, 20], [1, 1]):
        qs = np.concatenate([[0], np.cumsum(nq)])
        q = rng.standard_normal((qs[-1], 4 * 64))
        got, q = run_attn(torch, dev, "f32", q, qs, [700, 20], 4, 0.125, work=work, stream=st.cuda_stream, repeat=2)
        check_attn(got, q, dev, "f32", qs, [700, 20], 4, 0.125)


def test_append_then_attend_in_a_graph(torch_cuda):
    """A decode step captured once and replayed: the positions move on the device."""
    torch = torch_cuda
    rng = np.random.default_rng(11)
    h = filled(rng, [60, 31], 2, 64, 32, fill=0xFF)
    t, n_pages = tables(rng, [96, 96], 32)
    h2 = ref.Cache(2, 64, 32, t, n_pages, 0xFF)
    for s, n in enumerate([60, 31]):
        for hd in range(2):
            for keys in (True, False):
                x = h.load(s, n, hd, keys)
                for p in range(n):
                    h2.store(s, p, hd, x[p], keys)
    dev = Dev(torch, h2)
    q, k, v = (torch.randn(2, w, device="cuda") for w in (512, 128, 128))
    qo, out = torch.empty_like(q), torch.empty_like(q)
    pos, kl = torch.tensor([59, 30], dtype=torch.int32, device="cuda"), torch.tensor([60, 31], dtype=torch.int32, device="cuda")
    seq = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    qs = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    work = torch.zeros(abi.check_size(abi.lib.mg_kv4_attn_work(dev.ref(), 8, 1, 96)), dtype=torch.uint8, device="cuda")
    co, si = (torch.from_numpy(x).cuda() for x in rope(96, 64))
    P = lambda t: t.data_ptr()  # noqa: E731

    def step(st):
        abi.check(abi.lib.mg_kv4_append(dev.ref(), 0, 2, 8, P(q), 512, P(k), 128, P(v), 128, None, None, 0.0, P(co),
                                        P(si), 96, P(seq), P(pos), P(qo), 512, st))
        abi.check(abi.lib.mg_kv4_attn(dev.ref(), 0, 8, P(qo), 512, P(qs), P(kl), 1, 96, 0.125, 0, None, P(out), 512,
                                      P(work), work.numel(), st))

    def check():
        torch.cuda.synchronize()
        p = pos.cpu().numpy()
        kk = turned(k.cpu().numpy(), None, p, *(x.cpu().numpy() for x in (co, si)), 64)
        for s in range(2):
            for hd in range(2):
                h2.store(s, p[s], hd, kk[s, hd], True)
                h2.store(s, p[s], hd, v.cpu().numpy().astype(np.float64)[s].reshape(2, 64)[hd], False)
        assert np.array_equal(dev.pool.cpu().numpy(), h2.pool)
        check_attn(out.cpu().numpy(), qo.cpu().numpy().astype(np.float64), dev, "f32", [0, 1, 2], p + 1, 8, 0.125)

    step(None)  # sets kernel attributes before the capture
    check()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(torch.cuda.current_stream().cuda_stream)
    for i in range(3):
        for x in (q, k, v):
            x.normal_()
        pos += 1
        kl += 1
        g.replay()
        check()
