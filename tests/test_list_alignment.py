"""Lists of 32-bit numbers that do not start on one are refused (no GPU: answered before a device is looked for).
A kernel would fault on them."""
import ctypes as C

import pytest
from test_cache_8bit_checks import append_args, decode_args
from test_pages_overlap import READ, WRITTEN, arguments


@pytest.fixture(scope="module")
def lib():
    from tritonops_b200 import _lib, build
    build.build_library()
    return _lib.lib()


@pytest.mark.parametrize("off", [1, 2])
@pytest.mark.parametrize("kind", ["grow", "fork", "compact"])
def test_books(lib, kind, off):
    for field in READ[kind] + WRITTEN[kind]:
        a = arguments(kind, 100)
        setattr(a, field, getattr(a, field) + off)
        assert getattr(lib, f"b200attn_pages_{kind}")(C.byref(a), None) == -5, field


@pytest.mark.parametrize("off", [1, 2])
def test_cache_in_8_bits(lib, off):
    for field in ("page_table", "seqlens", "cu_new"):
        a = append_args()
        setattr(a, field, 0x20000 + off)
        assert lib.b200attn_kv_append_8bit(C.byref(a), None) == -5, field
    for field in ("page_table", "seqlens", "status_word"):
        a = decode_args()
        setattr(a, field, 0x20000 + off)
        assert lib.b200attn_paged_decode_8bit_fwd(C.byref(a), None) == -5, field
