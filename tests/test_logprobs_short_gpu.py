"""mg_logprobs of short 16-bit rows: all lengths around those whose vectors fill
fewer groups of threads than there are alternatives, exactly as in
test_logprobs_gpu, and at the pace of the lengths next to them (a row whose
candidates do not fit takes a pass for each alternative, some seven times as
long)."""
import numpy as np
import pytest

from midge_b200 import abi
from tests.test_logprobs_gpu import check, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("V", [1017, 1024, 1025, 1150, 1217, 1500, 1969, 1998, 2040, 2047, 2048, 2049, 2063])
@pytest.mark.parametrize("pad", [0, 3])
def test_alternatives(torch_cuda, kind, V, pad):
    rng = np.random.default_rng(V)
    x = rng.standard_normal((6, V)) * 2
    ids = rng.integers(0, V, (6, 1))
    for top in (20, 32):
        got, xx = run(torch_cuda, x, ids, top, kind, pad)
        check(got, xx, ids, top)


@pytest.mark.parametrize("V,longer,top", [(1500, 2100, 32), (1200, 1300, 20)])
def test_pace(torch_cuda, V, longer, top):
    torch = torch_cuda

    def us(V):
        x = torch.randn(2048, V, device="cuda").bfloat16()
        ent, al = torch.empty(2048, device="cuda"), torch.empty(2048, top, device="cuda")
        ai = torch.empty(2048, top, dtype=torch.int32, device="cuda")
        work = torch.zeros(abi.check_size(abi.lib.mg_logprobs_work(V, 2048, top)), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        best = float("inf")
        for _ in range(5):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in "ab")
            a.record()
            for _ in range(20):
                abi.check(abi.lib.mg_logprobs(2, x.data_ptr(), V, V, 2048, None, 0, top, None, ent.data_ptr(), ai.data_ptr(),
                                              al.data_ptr(), work.data_ptr(), work.numel(),
                                              torch.cuda.current_stream().cuda_stream))
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b) * 50)
        return best

    assert us(V) < 3 * us(longer)
