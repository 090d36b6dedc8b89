"""CPU checks of the layouts that the paged entry points refuse: rows that share memory with other rows."""
import ctypes
import os

import pytest
import torch

import paged_ctypes as PC
from test_paged_capi import CU, ECUDA, EINVAL, LIB


@pytest.fixture(scope="module")
def lib():
    return PC.load(LIB)


def rc(lib, call, **kw):
    d = PC.desc(**kw)
    return getattr(lib, "fcci_paged_" + call)(ctypes.byref(d), None)


@pytest.mark.parametrize("call", ["append", "decode", "prefill"])
@pytest.mark.parametrize("field", ["k_stride_t", "v_stride_t"])
@pytest.mark.parametrize("e4m3,stride", [(False, 64), (False, 96), (False, 120), (True, 112), (True, 64)])
def test_rows_of_a_page_that_overlap(lib, call, field, e4m3, stride):
    """A row has head_dim elements, whatever their size: a smaller step between rows is refused."""
    kw = dict(cu_seqlens_q=CU, total_q=5, max_seqlen_q=3) if call == "prefill" else {}
    assert rc(lib, call, e4m3=e4m3, **{field: stride}, **kw) == EINVAL
    assert b"overlap" in lib.fcci_last_error_string()
    if not torch.cuda.is_available():  # the packed row passes, as far as the device
        assert rc(lib, call, e4m3=e4m3, **{field: 128}, **kw) == ECUDA
