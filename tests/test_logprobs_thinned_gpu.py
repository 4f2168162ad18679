"""mg_logprobs where more entries reach the bound than are ranked at once (97
to 1024 candidates: short rows, rows of few distinct values), whole rows and
rows cut over blocks, many rows at a time and many times over: the candidates
are thinned by the whole block, so every warp has to come to the same count.
Alternatives are exact (value, then index), so there is no tolerance for
them; log probabilities as in test_logprobs_gpu."""
import numpy as np
import pytest

from midge_b200 import abi

pytestmark = pytest.mark.gpu
TOL = 2.0 ** -17


def repeated(torch, x, top, times):
    """x: device f32 rows.  The alternatives of every one of `times` calls against the first, which is returned."""
    n, V = x.shape
    ent = torch.empty(n, device="cuda")
    ai, al = torch.empty(n, top, dtype=torch.int32, device="cuda"), torch.empty(n, top, device="cuda")
    work = torch.zeros(abi.check_size(abi.lib.mg_logprobs_work(V, n, top)), dtype=torch.uint8, device="cuda")
    first, off = None, torch.zeros((), dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    for _ in range(times):
        ai.fill_(-9)
        torch.cuda.synchronize()
        abi.check(abi.lib.mg_logprobs(0, x.data_ptr(), V, V, n, None, 0, top, None, ent.data_ptr(), ai.data_ptr(),
                                      al.data_ptr(), work.data_ptr(), work.numel(), None))
        torch.cuda.synchronize()
        if first is None:
            first = (ai.clone(), al.clone())
        off += (ai != first[0]).sum() + (al != first[1]).sum()
    assert int(off) == 0
    return first


def check(torch, x, top, times):
    ai, al = repeated(torch, x, top, times)
    xs = x.cpu().numpy()
    want = np.argsort(-xs, axis=1, kind="stable")[:, :top]
    assert np.array_equal(ai.cpu().numpy(), want)
    d = torch.log_softmax(x.double(), -1).gather(1, ai.long())
    assert ((al.double() - d).abs() <= TOL + 2.0 ** -22 * d.abs()).all()


@pytest.mark.parametrize("V", [200, 333, 517, 1000])
@pytest.mark.parametrize("top", [20, 32])
def test_short_rows_many_times(torch_cuda, V, top):
    g = torch_cuda.Generator(device="cuda").manual_seed(V)
    check(torch_cuda, torch_cuda.randn(3000, V, device="cuda", generator=g) * 3, top, 100)


@pytest.mark.parametrize("V,rows,above", [(4097, 900, 300), (50001, 600, 900), (70003, 3, 150), (201088, 1, 900), (201088, 8, 400)])
def test_ties_above_the_rest_many_times(torch_cuda, V, rows, above):
    """`above` equal entries in random places above a floor: all of them candidates, the lowest indexes the answer."""
    g = torch_cuda.Generator(device="cuda").manual_seed(above)
    x = torch_cuda.randn(rows, V, device="cuda", generator=g).clamp_(-3, 3)
    at = torch_cuda.stack([torch_cuda.randperm(V, device="cuda", generator=g)[:above] for _ in range(rows)])
    x.scatter_(1, at, 5.0)
    for top in (1, 20, 32):
        check(torch_cuda, x, top, 40)
