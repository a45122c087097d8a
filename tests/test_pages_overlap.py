"""The page operators' C entry points refuse books of which a result overlaps something else of the call
(no GPU: every case is answered before a device is looked for)."""
import ctypes as C
import itertools

import pytest
import torch

READ = {"grow": ["page_table", "seqlens", "page_refs", "new_tokens"], "fork": ["page_table", "seqlens", "page_refs", "parents"],
        "compact": ["page_table", "page_refs"]}
WRITTEN = {"grow": ["page_table_out", "page_refs_out", "missing_out"],
           "fork": ["page_table_out", "seqlens_out", "page_refs_out", "missing_out"],
           "compact": ["page_table_out", "page_refs_out", "live_out"]}
SLOTS, WIDTH = 4, 8


@pytest.fixture(scope="module")
def lib():
    from tritonops_b200 import _lib, build
    build.build_library()
    return _lib.lib()


def arguments(kind, pages):
    from tritonops_b200 import _lib
    a = {"grow": _lib.PagesGrowArgs, "fork": _lib.PagesForkArgs, "compact": _lib.PagesCompactArgs}[kind]()
    for i, f in enumerate(READ[kind] + WRITTEN[kind] + ["workspace"]):
        setattr(a, f, 0x10000000 * (i + 1))
    a.workspace_bytes = 1 << 26
    a.slots, a.max_pages_per_seq, a.num_pages = SLOTS, WIDTH, pages
    if kind != "compact":
        a.page_size = 16
    return a


def extent(lib, kind, field, pages):
    if field == "workspace":
        return getattr(lib, f"b200attn_pages_{kind}_workspace_bytes")(C.byref(arguments(kind, pages)))
    return 4 * {"page_table": SLOTS * WIDTH, "page_refs": pages, "missing": 1, "live": 1}.get(field.removesuffix("_out"), SLOTS)


@pytest.mark.parametrize("pages", [100, 1 << 18])
@pytest.mark.parametrize("kind", ["grow", "fork", "compact"])
def test_results_lie_apart(lib, kind, pages):
    call = getattr(lib, f"b200attn_pages_{kind}")
    written = WRITTEN[kind] + (["workspace"] if pages > 100 else [])
    pairs = [(r, w) for r in READ[kind] for w in written] + list(itertools.combinations(written, 2))
    for first, second in pairs:
        a = arguments(kind, pages)
        end = getattr(a, first) + extent(lib, kind, first, pages)
        setattr(a, second, end - 4 if second != "workspace" else (end - 1) & ~15)
        assert call(C.byref(a), None) == -7, (first, second)
        start = getattr(a, first) - extent(lib, kind, second, pages)
        setattr(a, second, start + 4 if second != "workspace" else (start + 16) & ~15)
        assert call(C.byref(a), None) == -7, (second, first)


@pytest.mark.parametrize("kind", ["grow", "fork", "compact"])
def test_lists_read_may_be_one(lib, kind):
    """The same list for two inputs, and results right behind one another, are fine (answered by the look for a
    device, or by what comes after it)."""
    a = arguments(kind, 100)
    a.page_refs_out = a.page_table_out + 4 * SLOTS * WIDTH
    if kind == "grow":
        a.new_tokens = a.seqlens
    if not torch.cuda.is_available():
        assert getattr(lib, f"b200attn_pages_{kind}")(C.byref(a), None) == -10
