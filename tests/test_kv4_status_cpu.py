"""Refusals of mg_kv4_attn_status, before any device call."""
import ctypes as C

import pytest

from midge_b200 import abi
from tests.test_kv4_cpu import P, cache


@pytest.mark.parametrize("work,size", [(None, 1 << 40), (P, 0), (P, -1), (P, 64), (P + 8, 1 << 40)])
def test_refusals(work, size):
    assert abi.lib.mg_kv4_attn_status(work, size, None) == abi.MG_ERR_ARG
    assert b"kv4_attn_status" in abi.lib.mg_last_error()


def test_every_workspace_has_a_status():
    """The least of a workspace has room for it: one sequence, one head, one query."""
    c = cache(n_kv_heads=1, n_seqs=1)
    need = abi.check_size(abi.lib.mg_kv4_attn_work(C.byref(c), 1, 1, 1))
    assert abi.lib.mg_kv4_attn_status(P, need - 20 - 1, None) == abi.MG_ERR_ARG
