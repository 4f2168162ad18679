"""mg_kv4_append's query norms where the sum of squares passes fp32's range
either way.  Tolerance as in test_kv4_gpu: 2^-20 of the head's largest
magnitude and the type's rounding."""
import numpy as np
import pytest

from midge_b200 import abi
from tests import kv4_ref as ref
from tests.test_kv4_gpu import TYPES, Dev, to_dev

pytestmark = pytest.mark.gpu


def norm_rows(torch, x, w, eps, kind, D):
    """mg_kv4_append's queries [n, heads D] with a norm and nothing else."""
    n, heads = x.shape[0], x.shape[1] // D
    dev = Dev(torch, ref.Cache(1, D, 32, [[0]], 1))
    q, k = to_dev(torch, x, kind), to_dev(torch, np.ones((n, D)), kind)
    out, wd = torch.full_like(q, 7.0), torch.from_numpy(w).cuda()
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    abi.check(abi.lib.mg_kv4_append(dev.ref(), TYPES[kind][0], n, heads, q.data_ptr(), heads * D, k.data_ptr(), D,
                                    k.data_ptr(), D, wd.data_ptr(), None, eps, None, None, 0, None, pos.data_ptr(),
                                    out.data_ptr(), heads * D, None))
    torch.cuda.synchronize()
    return out.double().cpu().numpy().reshape(n, heads, D), q.double().cpu().numpy().reshape(n, heads, D)


def check_norm(got, x, w, eps, kind):
    want = x / np.sqrt((x * x).mean(-1, keepdims=True) + float(np.float32(eps))) * w.astype(np.float64)
    big = np.abs(want).max(-1, keepdims=True)
    tol = 2.0 ** -20 * big + TYPES[kind][2] * np.abs(want) + (2.0 ** -25 if kind == "f16" else 0)
    assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("D,heads", [(64, 8), (128, 5)])
def test_query_norm_of_huge_numbers(torch_cuda, kind, D, heads):
    """Heads of 1e18 to 1e38 among ordinary ones: 1e19 squared is beyond fp32, the result is not."""
    rng = np.random.default_rng(D)
    x = rng.uniform(-1, 1, (6, heads, D))
    x *= 10.0 ** np.array([18, 19, 20, 30, 38, 0])[:, None, None]
    x[2, 1::2] /= 1e20  # ordinary heads next to huge ones
    x[3, 0, 1:] = 0.0
    w = (1 + 0.2 * rng.standard_normal(D)).astype(np.float32)
    got, x = norm_rows(torch_cuda, x.reshape(6, -1), w, 1e-6, kind, D)
    check_norm(got, x, w, 1e-6, kind)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("D,heads", [(64, 8), (128, 5)])
@pytest.mark.parametrize("eps", [0.0, 1e-35])
def test_query_norm_of_tiny_numbers(torch_cuda, kind, D, heads, eps):
    """With an eps of (nearly) nothing the norm of 1e-15 to 1e-36 counts: their squares are below fp32."""
    rng = np.random.default_rng(D)
    x = rng.uniform(-1, 1, (6, heads, D))
    x *= 10.0 ** np.array([-15, -18, -20, -25, -36, 0])[:, None, None]
    x[2, 1::2] *= 1e20
    w = (1 + 0.2 * rng.standard_normal(D)).astype(np.float32)
    got, x = norm_rows(torch_cuda, x.reshape(6, -1), w, eps, kind, D)
    check_norm(got, x, w, eps, kind)


@pytest.mark.parametrize("kind", list(TYPES))
def test_query_norm_of_infinities(torch_cuda, kind):
    """A finite number over an infinite norm is 0; the infinity itself, and heads with a NaN, are NaN; others are untouched."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((2, 4, 64))
    x[0, 1, 7], x[0, 2, 40], x[1, 0, 63] = np.inf, np.nan, -np.inf
    w = np.ones(64, np.float32)
    got, x = norm_rows(torch_cuda, x.reshape(2, -1), w, 1e-6, kind, 64)
    for t, h, d in ((0, 1, 7), (1, 0, 63)):
        assert np.isnan(got[t, h, d]) and (np.delete(got[t, h], d) == 0).all()
    assert np.isnan(got[0, 2]).all()
    whole = np.ones((2, 4), bool)
    whole[0, 1:3] = whole[1, 0] = False
    check_norm(got[whole], x[whole], w, 1e-6, kind)
