"""Rows that are not aligned to their type are refused on the host: a load of them would fault on the device."""
import ctypes as C

import pytest

from midge_b200 import abi
from tests.test_kv4_cpu import P, append, attn, cache, refused

TYPES = [(0, 1), (0, 2), (1, 1), (2, 3)]  # type, bytes off


@pytest.mark.parametrize("act,off", TYPES)
def test_refused(act, off):
    c = C.byref(cache())
    for row in ("q", "k", "v", "qo"):
        refused(append(c, act=act, **{row: P + off}), b"aligned")
    for row in ("q", "out"):
        refused(attn(c, act=act, **{row: P + off}), b"aligned")
    refused(abi.lib.mg_kv4_read(c, act, 1, None, P, P + off, 512, P, 512, None), b"aligned")
    refused(abi.lib.mg_kv4_read(c, act, 1, None, P, P, 512, P + off, 512, None), b"aligned")
    refused(abi.lib.mg_logprobs(act, P + off, 100, 100, 1, P, 1, 0, P, P, None, None, P, 1 << 40, None), b"aligned")


def test_an_element_further_is_taken():
    """Nothing to do, so that nothing is launched."""
    for act, off in ((0, 4), (1, 2), (2, 2)):
        assert append(C.byref(cache()), act=act, n=0, q=P + off, k=P + off, v=P + off, qo=P + off) == abi.MG_OK
        assert abi.lib.mg_logprobs(act, P + off, 100, 100, 0, None, 0, 0, None, P, None, None, P, 1 << 40, None) == abi.MG_OK
