"""ctypes mirror of fcci_paged_desc (include/fcci_paged.h)."""
import ctypes as C

I32, I64, P = C.c_int32, C.c_int64, C.c_void_p


class PagedDesc(C.Structure):
    _fields_ = [
        ("abi_version", I32), ("B", I32), ("Hq", I32), ("Hkv", I32), ("D", I32), ("total_q", I32), ("max_seqlen_q", I32),
        ("cu_seqlens_q", P), ("q", P), ("q_stride_t", I64), ("q_stride_h", I64), ("k_new", P), ("k_new_stride_t", I64),
        ("k_new_stride_h", I64), ("v_new", P), ("v_new_stride_t", I64), ("v_new_stride_h", I64), ("cache_type", I32),
        ("page_size", I32), ("num_pages", I32), ("max_pages", I32), ("k_pages", P), ("k_stride_p", I64),
        ("k_stride_h", I64), ("k_stride_t", I64), ("v_pages", P), ("v_stride_p", I64), ("v_stride_h", I64),
        ("v_stride_t", I64), ("k_scales", P), ("k_scales_stride_p", I64), ("k_scales_stride_h", I64), ("v_scales", P),
        ("v_scales_stride_p", I64), ("v_scales_stride_h", I64), ("page_table", P), ("page_table_stride", I64),
        ("seq_lens", P), ("out", P), ("out_stride_t", I64), ("out_stride_h", I64), ("q_rot_out", P), ("scale", C.c_float),
        ("rope_theta", C.c_float), ("rotary_dim", I32), ("advance", I32), ("max_kv_tokens", I32), ("workspace", P),
        ("workspace_bytes", C.c_size_t), ("flags", C.c_uint32),
    ]


def load(path):
    lib = C.CDLL(path)
    for f in ("fcci_paged_append", "fcci_paged_decode", "fcci_paged_prefill"):
        getattr(lib, f).restype = C.c_int
        getattr(lib, f).argtypes = [P, P]
    lib.fcci_paged_workspace_bytes.restype = C.c_size_t
    lib.fcci_paged_workspace_bytes.argtypes = [I32] * 7 + [C.c_int]
    lib.fcci_paged_workspace_init.argtypes = [P, C.c_size_t, P]
    lib.fcci_paged_workspace_init.restype = C.c_int
    lib.fcci_paged_read_error.argtypes = [P, P, C.c_int, P]
    lib.fcci_paged_read_error.restype = C.c_int
    lib.fcci_last_error_string.restype = C.c_char_p
    lib.fcci_last_status.restype = C.c_int
    return lib


def desc(B=2, Hq=8, Hkv=2, D=128, page=64, e4m3=True, **kw):
    """A descriptor that passes every argument check (its pointers are aligned numbers, never read on the host)."""
    d = PagedDesc(abi_version=1, B=B, Hq=Hq, Hkv=Hkv, D=D, total_q=B, max_seqlen_q=1, q=0x10000, q_stride_t=Hq * D,
                  q_stride_h=D, k_new=0x20000, k_new_stride_t=Hkv * D, k_new_stride_h=D, v_new=0x30000,
                  v_new_stride_t=Hkv * D, v_new_stride_h=D, cache_type=1 if e4m3 else 0, page_size=page, num_pages=8,
                  max_pages=4, k_pages=0x40000, k_stride_p=Hkv * page * D, k_stride_h=page * D, k_stride_t=D,
                  v_pages=0x50000, v_stride_p=Hkv * page * D, v_stride_h=page * D, v_stride_t=D,
                  k_scales=0x60000 if e4m3 else None, k_scales_stride_p=Hkv, k_scales_stride_h=1,
                  v_scales=0x70000 if e4m3 else None, v_scales_stride_p=Hkv, v_scales_stride_h=1, page_table=0x80000,
                  page_table_stride=4, seq_lens=0x90000, out=0xA0000, out_stride_t=Hq * D, out_stride_h=D,
                  q_rot_out=0xB0000, scale=0.1, rope_theta=10000.0, rotary_dim=D, advance=0, max_kv_tokens=-1,
                  workspace=0xC0000, workspace_bytes=1 << 40)
    for k, v in kw.items():
        setattr(d, k, v)
    return d
