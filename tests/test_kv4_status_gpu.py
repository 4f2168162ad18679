"""mg_kv4_attn_status: what a timed-out wait inside mg_kv4_attn leaves behind
reaches the caller, and nobody else.  The failure is made on the host, by
writing a code over the workspace; no kernel is made to wait."""
import ctypes as C

import numpy as np
import pytest

from midge_b200 import abi, kv4_score
from tests.test_kv4_gpu import Dev, check_attn, filled, run_attn
from tests.test_kv4_score_gpu import _model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nq", [1, 40])
def test_a_marked_workspace_is_told_and_made_ready(torch_cuda, nq):
    torch = torch_cuda
    rng = np.random.default_rng(nq)
    dev = Dev(torch, filled(rng, [700, 20], 1, 64, 64))
    work = torch.zeros(abi.check_size(abi.lib.mg_kv4_attn_work(dev.ref(), 4, nq, 700)), dtype=torch.uint8, device="cuda")
    st = torch.cuda.Stream()
    qs = np.array([0, nq, 2 * nq])

    def attend():
        q0 = rng.standard_normal((2 * nq, 256))
        got, q = run_attn(torch, dev, "f32", q0, qs, [700, 20], 4, 0.125, work=work, stream=st.cuda_stream)
        check_attn(got, q, dev, "f32", qs, [700, 20], 4, 0.125)

    attend()
    status = lambda: abi.lib.mg_kv4_attn_status(work.data_ptr(), work.numel(), st.cuda_stream)  # noqa: E731
    assert status() == abi.MG_OK
    work.view(torch.int32).fill_(41)
    torch.cuda.synchronize()
    assert status() == abi.MG_ERR_TIMEOUT
    assert b"code 41" in abi.lib.mg_last_error()
    assert int(work.count_nonzero()) == 0 and status() == abi.MG_OK
    attend()
    assert status() == abi.MG_OK


def test_a_model_is_not_told_of_it(torch_cuda, tmp_path):
    """The engine's own check goes by its own word; scoring over the 4-bit cache raises."""
    torch = torch_cuda
    path, spec = _model(tmp_path, "sinks")
    m = kv4_score.Kv4Model(path, 40, page=32)
    m.step({0: [1, 2, 3]})
    m.work.view(torch.int32).fill_(42)
    torch.cuda.synchronize()
    e = abi.Model.from_dir(path, ctx=40)
    e.forward_batch(0, np.array([1, 2, 3], np.int32), logits_mode=2)
    e.close()
    with pytest.raises(abi.MidgeError) as x:
        abi.check(abi.lib.mg_kv4_attn_status(m.work.data_ptr(), m.work.numel(), None))
    assert x.value.code == abi.MG_ERR_TIMEOUT
    assert np.isfinite(m.step({0: [4]}).cpu().numpy()).all()


def test_wait_selftest_leaves_the_workspace_alone(torch_cuda):
    dev = Dev(torch_cuda, filled(np.random.default_rng(0), [50], 1, 64, 64))
    work = torch_cuda.zeros(abi.check_size(abi.lib.mg_kv4_attn_work(dev.ref(), 4, 1, 50)), dtype=torch_cuda.uint8, device="cuda")
    d = C.c_int(0)
    assert abi.lib.mg_wait_selftest(10, C.byref(d)) == abi.MG_ERR_TIMEOUT
    torch_cuda.cuda.synchronize()
    assert abi.lib.mg_kv4_attn_status(work.data_ptr(), work.numel(), None) == abi.MG_OK
