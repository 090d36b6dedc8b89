"""CPU checks of the paged cache's boundary: descriptor layout, refusals of the C ABI and of the Python entry points,
page bookkeeping's arithmetic."""
import ctypes
import os
import subprocess

import pytest
import torch

import paged_ctypes as PC
from oracle import paged_oracle as P

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "fully_custom_cuda_inference_lamma2_b200", "libfcci_decode.so")
OK, EINVAL, EUNSUPPORTED, EWORKSPACE, ECUDA = 0, 1, 2, 3, 4


@pytest.fixture(scope="module")
def lib():
    return PC.load(LIB)


def test_descriptor_layout_matches_header(tmp_path):
    src = tmp_path / "layout.cpp"
    names = [n for n, _ in PC.PagedDesc._fields_]
    src.write_text('#include <cstdio>\n#include <cstddef>\n#include "fcci_paged.h"\nint main() {\n'
                   'std::printf("%zu\\n", sizeof(fcci_paged_desc));\n'
                   + "".join(f'std::printf("%zu\\n", offsetof(fcci_paged_desc, {n}));\n' for n in names) + "return 0; }\n")
    exe = tmp_path / "layout"
    cuda_inc = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "include")
    subprocess.run(["g++", "-I", os.path.join(ROOT, "include"), "-I", cuda_inc, str(src), "-o", str(exe)], check=True)
    out = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert out[0] == ctypes.sizeof(PC.PagedDesc)
    assert out[1:] == [getattr(PC.PagedDesc, n).offset for n in names]


CU = 0xD0000
BAD = [
    ("abi_version", 2, EINVAL), ("B", 0, EINVAL), ("Hq", 7, EINVAL), ("Hkv", 0, EINVAL), ("D", 96, EUNSUPPORTED),
    ("page_size", 48, EUNSUPPORTED), ("page_size", 256, EUNSUPPORTED), ("page_size", 0, EUNSUPPORTED),
    ("cache_type", 2, EINVAL), ("k_pages", None, EINVAL), ("v_pages", None, EINVAL), ("page_table", None, EINVAL),
    ("seq_lens", None, EINVAL), ("k_scales", None, EINVAL), ("v_scales", None, EINVAL), ("num_pages", 0, EINVAL),
    ("max_pages", 0, EINVAL), ("max_pages", 1 << 30, EINVAL), ("page_table_stride", -4, EINVAL), ("k_new", None, EINVAL),
    ("total_q", -1, EINVAL), ("total_q", 3, EINVAL), ("max_seqlen_q", -1, EINVAL), ("rotary_dim", 8, EUNSUPPORTED),
    ("rotary_dim", 144, EUNSUPPORTED), ("rotary_dim", -16, EUNSUPPORTED), ("rope_theta", 0.0, EINVAL),
    ("rope_theta", float("nan"), EINVAL), ("rope_theta", 1e-7, EINVAL), ("rope_theta", float("inf"), EINVAL), ("k_pages", 0x40008, EINVAL),
    ("v_new", 0x30002, EINVAL), ("q", 0x10004, EINVAL), ("k_stride_p", 8, EINVAL), ("v_stride_t", 64, EINVAL),
    ("k_stride_t", 0, EINVAL), ("k_stride_h", -128, EINVAL), ("q_stride_h", 132, EINVAL), ("k_scales_stride_p", -1, EINVAL),
    ("workspace", None, None), ("workspace_bytes", 1000, None),
]


@pytest.mark.parametrize("call", ["append", "decode"])
@pytest.mark.parametrize("field,value,status", BAD)
def test_refusals(lib, call, field, value, status):
    d = PC.desc(**{field: value})
    rc = getattr(lib, "fcci_paged_" + call)(ctypes.byref(d), None)
    if status is None:  # the workspace's size depends on the device
        assert rc in (EWORKSPACE, ECUDA)
    else:
        assert rc == status and lib.fcci_last_status() == status and lib.fcci_last_error_string()


def test_more_refusals(lib):
    def rc(call, **kw):
        d = PC.desc(**kw)
        return getattr(lib, "fcci_paged_" + call)(ctypes.byref(d), None)

    for call in ("append", "decode", "prefill"):
        assert getattr(lib, "fcci_paged_" + call)(None, None) == EINVAL
    assert rc("decode", scale=0.0) == EINVAL and rc("decode", scale=float("nan")) == EINVAL
    assert rc("decode", scale=float("inf")) == EINVAL
    assert rc("decode", q=None) == EINVAL and rc("decode", out=None) == EINVAL
    assert rc("decode", cu_seqlens_q=CU) == EINVAL, "decode takes one token a sequence"
    assert rc("decode", k_new=None, v_new=None, advance=1) == EINVAL
    assert rc("decode", Hq=34, Hkv=2) == EUNSUPPORTED and rc("decode", D=256, Hq=18, page=64) == EUNSUPPORTED
    assert rc("decode", D=256, page=128) == EUNSUPPORTED
    assert rc("decode", e4m3=False, k_scales=0x60000) == EINVAL
    assert rc("decode", flags=2) == EINVAL and rc("append", flags=1) == EINVAL
    assert rc("prefill", cu_seqlens_q=CU, flags=1) == EINVAL
    assert rc("append", q_rot_out=None) == EINVAL and rc("append", q=None) == EINVAL
    assert rc("append", k_new=None, v_new=None) == EINVAL
    assert rc("prefill") == EINVAL, "prefill needs cu_seqlens_q"
    assert rc("prefill", cu_seqlens_q=CU, D=64) == EUNSUPPORTED
    assert rc("prefill", cu_seqlens_q=CU, k_new=None, v_new=None) == EINVAL
    assert rc("append", B=65536, total_q=65536) == EUNSUPPORTED
    # what passes all checks gets as far as the device, of which there is none here
    if not torch.cuda.is_available():
        for e4m3 in (True, False):
            assert rc("append", e4m3=e4m3, k_stride_t=128) == ECUDA
            assert rc("decode", e4m3=e4m3) == ECUDA
            assert rc("prefill", e4m3=e4m3, cu_seqlens_q=CU, total_q=5, max_seqlen_q=3) == ECUDA
        assert rc("append", q=None, q_rot_out=None) == ECUDA


def test_workspace_bytes_of_invalid_shapes(lib):
    for bad in ((0, 8, 2, 128, 1, 1, 0), (1, 8, 3, 128, 1, 1, 0), (1, 8, 2, 100, 1, 1, 0), (1, 8, 2, 128, -1, 1, 0),
                (1, 8, 2, 128, 1, -1, 0), (1, 8, 2, 128, 1, 1, -1)):
        assert lib.fcci_paged_workspace_bytes(*bad, 0) == 0
    assert lib.fcci_paged_workspace_init(None, 1 << 20, None) == EWORKSPACE
    assert lib.fcci_paged_workspace_init(0xC0000, 64, None) == EWORKSPACE
    flags = ctypes.c_uint32()
    assert lib.fcci_paged_read_error(None, ctypes.byref(flags), 0, None) == EINVAL


def test_python_entry_points_refuse_host_tensors():
    import fully_custom_cuda_inference_lamma2_b200 as pkg

    av = pkg.attn_varlen
    k = torch.zeros(1, 2, 128, dtype=torch.float16)
    pool = torch.zeros(3, 2, 16, 128, dtype=torch.float16)
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="must be CUDA"):
        av.paged_append(k, k, pool, pool, table, lens)
    with pytest.raises(RuntimeError, match="must be CUDA"):
        av.paged_decode(k, pool, pool, k, table, lens)
    with pytest.raises(RuntimeError, match="must be CUDA"):
        av.paged_prefill(k, k, k, pool, pool, k, table, lens, table, 1)
    for bad in (dict(dtype=torch.bfloat16), dict(page_size=24), dict(page_size=128, head_dim=256), dict(num_pages=0)):
        kw = dict(num_pages=4, page_size=16, head_dim=128)
        kw.update(bad)
        head_dim = kw.pop("head_dim")
        with pytest.raises(ValueError):
            pkg.PagedKVCache(1, 1, 1, head_dim, device="cpu", **kw)


def test_oracle_scale_and_grid():
    """The oracle's own arithmetic: against torch's e4m3 cast, and the scale's border at 448 * 2^e."""
    x = torch.randn(4096, dtype=torch.float64) * 30
    x[:10] = torch.tensor([0.0, 448.0, -448.0, 2.0 ** -9, 2.0 ** -10, 1.5 * 2 ** -9, 17.0, 18.0, 19.0, 2.0 ** -6])
    assert torch.equal(P.e4m3_grid(x), x.to(torch.float32).to(torch.float8_e4m3fn).double())
    for e in (-15, -3, 0, 8):
        top = 448.0 * 2.0 ** e
        assert P.scale_exponent(top) == e
        assert P.scale_exponent(top * (1 + 2 ** -20)) == min(8, e + 1)
    assert P.scale_exponent(0.0) == -15 and P.scale_exponent(1e9) == 8
