"""An output whose rows would lie over one another is refused on the host, as such queries are."""

import ctypes

import pytest

from calibquant_b200 import _lib
from test_chunk_abi import chunk_args, lib, p16      # noqa: F401 (fixtures)


@pytest.mark.parametrize("strides", [(0, 1024, 128), (4096, 0, 128), (4096, 1024, 0), (4096, -1024, 128)], ids=str)
def test_rows_over_one_another(lib, p16, strides):      # noqa: F811
    a = chunk_args(p16, batch=2, out_strides=strides)
    assert lib.cq_chunk_attn_workspace_bytes(ctypes.byref(a)) == 0
    assert lib.cq_chunk_attn(ctypes.byref(a), p16, 1 << 30, None) == _lib.CQ_ERR_BAD_ARG


def test_strides_that_nothing_uses(lib, p16):      # noqa: F811
    a = chunk_args(p16, batch=1, q_len=1, out_strides=(0, 0, 128), q_strides=(0, 0, 128))
    assert lib.cq_chunk_attn_workspace_bytes(ctypes.byref(a)) > 0
