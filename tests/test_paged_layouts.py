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


@pytest.mark.parametrize("call,field,kw", [
    ("append", "k_stride_h", dict(k_stride_h=0)),                          # a pool that is broadcast over its heads
    ("decode", "v_stride_h", dict(v_stride_h=0)),
    ("append", "k_stride_p", dict(k_stride_p=0)),                          # ... over its pages
    ("append", "k_stride_h", dict(k_stride_t=128, k_stride_h=128)),        # head 1 of row 0 is head 0 of row 1
    ("decode", "v_stride_p", dict(v_stride_p=64 * 128)),                   # page 1 of head 0 is page 0 of head 1
    ("append", "k_scales_stride_h", dict(k_scales_stride_h=0)),
    ("decode", "v_scales_stride_p", dict(v_scales_stride_p=1)),
    ("decode", "out_stride_t", dict(out_stride_t=0)),
    ("decode", "out_stride_h", dict(out_stride_h=64)),
    ("decode", "out_stride_t", dict(out_stride_t=128)),
    ("prefill", "out_stride_t", dict(out_stride_t=0, cu_seqlens_q=CU, total_q=5, max_seqlen_q=3)),
    ("prefill", "k_stride_p", dict(k_stride_p=128, cu_seqlens_q=CU, total_q=5, max_seqlen_q=3)),
])
def test_outputs_that_share_memory(lib, call, field, kw):
    """What a call writes may not lie twice in the same place."""
    assert rc(lib, call, **kw) == EINVAL, field
    assert b"overlap" in lib.fcci_last_error_string()


def test_layouts_that_share_nothing(lib):
    """Any order of pages, heads and rows, gaps between them, dimensions of extent 1 with any stride, and, where nothing is
    written, pools that are broadcast."""
    if torch.cuda.is_available():
        pytest.skip("on a GPU these would run on made-up addresses")
    D, page, Hkv, pages = 128, 64, 2, 8
    for t, h, p in ((D, page * D, Hkv * page * D), (Hkv * D, D, Hkv * page * D), (D, pages * page * D, page * D),
                    (pages * Hkv * D, pages * D, D), (D + 16, page * (D + 16), 3 * page * (D + 16))):
        for e4m3 in (True, False):
            assert rc(lib, "append", e4m3=e4m3, k_stride_t=t, k_stride_h=h, k_stride_p=p) == ECUDA
            assert rc(lib, "decode", e4m3=e4m3, v_stride_t=t, v_stride_h=h, v_stride_p=p) == ECUDA
    assert rc(lib, "append", Hq=1, Hkv=1, k_stride_h=0, k_scales_stride_h=0) == ECUDA
    assert rc(lib, "append", num_pages=1, k_stride_p=0, k_scales_stride_p=0) == ECUDA
    assert rc(lib, "append", k_scales_stride_p=1, k_scales_stride_h=8) == ECUDA
    assert rc(lib, "decode", B=1, total_q=1, out_stride_t=0) == ECUDA
    assert rc(lib, "decode", k_new=None, v_new=None, k_stride_h=0, v_stride_p=0, k_scales_stride_h=0) == ECUDA
    assert rc(lib, "append", k_new_stride_t=0, v_new_stride_h=0, q_stride_t=0) == ECUDA
