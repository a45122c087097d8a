"""What the C entry points of the 8-bit cache and of its pages refuse (no GPU: every case is answered
before a device is looked for), their argument structs, and the oracle's own steps by hand."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from oracle import paged_cache_oracle as orc

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    from tritonops_b200 import _lib, build
    build.build_library()
    return _lib.lib()


def test_struct_sizes_match_header(tmp_path):
    from tritonops_b200 import _lib
    names = {"paged_decode_8bit_args": _lib.PagedDecode8bitArgs, "kv_append_8bit_args": _lib.KvAppend8bitArgs,
             "page_pool": _lib.PagePool, "pages_grow_args": _lib.PagesGrowArgs, "pages_fork_args": _lib.PagesForkArgs,
             "pages_compact_args": _lib.PagesCompactArgs}
    fields = [(n, f[0]) for n, s in names.items() for f in s._fields_]
    src = tmp_path / "p.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "b200attn.h"\nint main(){\n'
                   + "".join(f'printf("%zu\\n", sizeof(b200attn_{n}));\n' for n in names)
                   + "".join(f'printf("%zu\\n", offsetof(b200attn_{n}, {f}));\n' for n, f in fields) + "return 0;}\n")
    exe = tmp_path / "p"
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    got = list(map(int, subprocess.check_output([str(exe)]).split()))
    assert got == [C.sizeof(s) for s in names.values()] + [getattr(names[n], f).offset for n, f in fields]


def decode_args():
    from tritonops_b200._lib import PagedDecode8bitArgs
    a = PagedDecode8bitArgs()
    for f in ("q", "k_pages", "v_pages", "k_scales", "v_scales", "o", "page_table", "seqlens", "workspace"):
        setattr(a, f, 0x10000)
    a.workspace_bytes = 1 << 40
    a.dtype, a.cache_dtype, a.batch, a.queries = 1, 3, 2, 1
    a.heads_q, a.heads_kv, a.head_dim = 8, 2, 128
    a.page_size, a.block_tokens, a.num_pages, a.max_pages_per_seq, a.max_seqlen = 64, 16, 10, 400, 25600
    return a


@pytest.mark.parametrize("field,value,code", [
    ("q", 0, -1), ("k_scales", 0, -1), ("page_table", 0, -1), ("dtype", 2, -2), ("cache_dtype", 1, -2),
    ("head_dim", 48, -3), ("heads_q", 7, -4), ("q", 0x10008, -5), ("v_pages", 0x10008, -5), ("v_scales", 0x10002, -5),
    ("q_stride_h", 12, -6), ("k_stride_t", 8, -6), ("v_stride_page", 24, -6), ("batch", 0, -7), ("queries", 0, -7),
    ("num_pages", 0, -7), ("max_pages_per_seq", 0, -7), ("max_seqlen", -1, -7), ("chunk_tokens", 64, -7),
    ("workspace", 0, -8), ("workspace_bytes", 0, -8), ("block_tokens", 8, -9), ("block_tokens", 48, -9),
    ("page_size", 72, -9), ("page_size", 0, -9), ("batch", 65536, -11)])
def test_decode_refusals(lib, field, value, code):
    a = decode_args()
    setattr(a, field, value)
    assert lib.b200attn_paged_decode_8bit_fwd(C.byref(a), None) == code


def append_args():
    from tritonops_b200._lib import KvAppend8bitArgs
    a = KvAppend8bitArgs()
    for f in ("new_k", "new_v", "k_pages", "v_pages", "k_scales", "v_scales", "page_table", "seqlens"):
        setattr(a, f, 0x10000)
    a.dtype, a.cache_dtype, a.batch, a.heads, a.head_dim, a.tokens = 0, 4, 2, 2, 64, 2
    a.page_size, a.block_tokens, a.num_pages, a.max_pages_per_seq = 64, 32, 10, 4
    return a


@pytest.mark.parametrize("field,value,code", [
    ("new_k", 0, -1), ("k_scales", 0, -1), ("seqlens", 0, -1), ("dtype", 2, -2), ("cache_dtype", 0, -2),
    ("head_dim", 80, -3), ("new_v", 0x10008, -5), ("k_scales", 0x10001, -5), ("nk_stride_t", 4, -6), ("k_stride_h", 8, -6),
    ("batch", 0, -7), ("tokens", 3, -7), ("tokens", -1, -7), ("heads", 0, -7), ("block_tokens", 256, -9),
    ("page_size", 48, -9), ("heads", 20000, -11)])
def test_append_refusals(lib, field, value, code):
    a = append_args()
    setattr(a, field, value)
    assert lib.b200attn_kv_append_8bit(C.byref(a), None) == code


def pages_args(kind):
    from tritonops_b200 import _lib
    cls = {"grow": _lib.PagesGrowArgs, "fork": _lib.PagesForkArgs, "compact": _lib.PagesCompactArgs}[kind]
    a = cls()
    at = 0x100000
    for f, t in cls._fields_:
        if t is C.c_void_p:
            setattr(a, f, at)
            at += 0x100000
    a.workspace_bytes = 1 << 20
    a.slots, a.max_pages_per_seq, a.num_pages = 4, 8, 100
    if kind != "compact":
        a.page_size = 16
    if kind != "grow":
        a.pools, a.n_pools = (_lib.PagePool * 1)(_lib.PagePool(0x9000000, 64, 64)), 1
    return a


@pytest.mark.parametrize("kind", ["grow", "fork", "compact"])
def test_pages_refusals(lib, kind):
    from tritonops_b200 import _lib
    call = getattr(lib, f"b200attn_pages_{kind}")

    def status(**change):
        a = pages_args(kind)
        for f, v in change.items():
            setattr(a, f, v)
        return call(C.byref(a), None)

    assert call(None, None) == -1
    for f in ("page_table", "page_refs", "page_table_out", "page_refs_out"):
        assert status(**{f: 0}) == -1
        assert status(**{f: getattr(pages_args(kind), f) + 2}) == -5
    for f in ("slots", "max_pages_per_seq", "num_pages"):
        assert status(**{f: 0}) == -7
    assert status(slots=1 << 20, max_pages_per_seq=1 << 20) == -11
    a = pages_args(kind)
    assert status(page_table_out=a.page_table) == -7                 # in place
    assert status(page_refs_out=a.page_refs + 4 * 99) == -7          # overlapping
    assert status(page_table_out=a.page_refs_out) == -7
    # (a workspace is needed where the bookkeeping does not fit into shared memory)
    small, large = getattr(lib, f"b200attn_pages_{kind}_workspace_bytes"), dict(num_pages=1 << 18)
    assert small(C.byref(a)) == 0
    assert status(workspace=0, **large) == -8 and status(workspace_bytes=64, **large) == -8
    assert status(workspace=a.workspace + 8, workspace_bytes=1 << 24, **large) == -5
    if kind != "compact":
        assert status(page_size=0) == -7
    if kind != "grow":
        one = lambda *p: (_lib.PagePool * 1)(_lib.PagePool(*p))  # noqa: E731
        assert status(n_pools=-1) == -7
        assert status(pools=None) == -1
        assert status(pools=one(0, 64, 64)) == -1
        assert status(pools=one(0x9000000, 0, 64)) == -7
        assert status(pools=one(0x9000000, 64, 32)) == -7
        assert status(pools=one(0x9000002, 64, 64)) == -5
        assert status(pools=one(0x9000000, 62, 64)) == -5
        assert status(pools=one(0x9000000, 1 << 31, 1 << 31)) == -11
    if kind == "fork":
        assert status(seqlens_out=a.seqlens) == -7 and status(seqlens_out=a.parents) == -7
        assert status(slots=40000) == -11
        assert status(page_size=1 << 30) == -11


def test_ops_take_cuda_tensors_only(lib):
    from tritonops_b200 import ops
    i = torch.zeros(2, 2, dtype=torch.int32)
    pool, scale = torch.zeros(2, 16, 1, 32, dtype=torch.int8), torch.zeros(2, 1, 1)
    x = torch.zeros(2, 1, 32, dtype=torch.float16)
    for call in (lambda: ops.paged_decode_8bit(x, pool, pool, scale, scale, i, i[0]),
                 lambda: ops.append_kv_8bit(pool, pool, scale, scale, x, x, i, i[0]),
                 lambda: ops.grow_pages(i, i[0], i[0], i[0], page_size=16),
                 lambda: ops.fork_pages([pool], i, i[0], i[0], i[0], page_size=16),
                 lambda: ops.compact_pages([pool], i, i[0])):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()


def test_oracle_scales_by_hand():
    e4m3, i8 = torch.float8_e4m3fn, torch.int8
    assert orc.scale_for(448.0, e4m3) == 1 and orc.scale_for(448.5, e4m3) == 2 and orc.scale_for(224.0, e4m3) == 0.5
    assert orc.scale_for(127.0, i8) == 1 and orc.scale_for(127.5, i8) == 2 and orc.scale_for(0.0, i8) == 0
    assert orc.scale_for(1e-45, i8) == 2.0 ** -126 and orc.scale_for(float("inf"), i8) != orc.scale_for(float("inf"), i8)


def test_oracle_fork_by_hand():
    """Three slots; slot 0 goes on, slot 1 forks from it, slot 2 ends."""
    i32 = torch.int32
    table = torch.tensor([[4, 2], [1, -1], [0, 3]], dtype=i32)
    lens = torch.tensor([20, 5, 32], dtype=i32)
    refs = torch.tensor([1, 1, 1, 1, 1, 0], dtype=i32)
    pool = torch.arange(6.0)[:, None]
    t, n, r, missing, pools = orc.fork([pool], table, lens, refs, torch.tensor([0, 0, -1], dtype=i32), 16)
    assert t.tolist() == [[4, 2], [4, 0], [-1, -1]] and n.tolist() == [20, 20, 0]
    assert r.tolist() == [1, 0, 1, 0, 2, 0] and int(missing) == 0 and pools[0].flatten().tolist() == [2, 1, 2, 3, 4, 5]


def test_oracle_compact_and_grow_by_hand():
    i32 = torch.int32
    t, r, n, pools = orc.compact([torch.arange(6.0)[:, None]], torch.tensor([[5, 1], [3, 9]], dtype=i32),
                                 torch.tensor([0, 2, 0, 1, 0, 1], dtype=i32))
    assert t.tolist() == [[2, 1], [0, -1]] and r.tolist() == [1, 2, 1, 0, 0, 0] and int(n) == 3
    assert pools[0].flatten().tolist() == [3, 1, 5, 3, 4, 5]
    t, r, missing = orc.grow(torch.tensor([[1, -1], [-1, -1]], dtype=i32), torch.tensor([16, 0], dtype=i32),
                             torch.tensor([0, 1, 0], dtype=i32), torch.tensor([17, 20], dtype=i32), 16)
    assert t.tolist() == [[1, 0], [2, -1]] and r.tolist() == [1, 1, 1] and int(missing) == 2


@pytest.mark.parametrize("field", ["k_stride_page", "v_stride_page", "k_stride_t", "v_stride_t", "k_stride_h", "v_stride_h",
                                   "ks_stride_page", "vs_stride_page", "ks_stride_blk", "vs_stride_blk", "ks_stride_h",
                                   "vs_stride_h"])
def test_what_is_written_lies_apart(lib, field):
    """An expanded pool or scale (a stride of 0) is refused where rows are appended, an expanded pool
    where it is read as well."""
    a, d = append_args(), decode_args()
    for x, D in ((a, 64), (d, 128)):
        for pool in "kv":
            for f, v in (("page", 64 * 2 * D), ("t", 2 * D), ("h", D)):
                setattr(x, f"{pool}_stride_{f}", v)
            for f, v in (("page", 4), ("blk", 2), ("h", 1)):
                setattr(x, f"{pool}s_stride_{f}", v)
    d.q_stride_b = d.q_stride_t = d.o_stride_b = d.o_stride_t = 8 * 128
    d.q_stride_h = d.o_stride_h = 128
    setattr(a, field, 0)
    assert lib.b200attn_kv_append_8bit(C.byref(a), None) == -6
    if field[1] == "_":
        setattr(d, field, 0)
        assert lib.b200attn_paged_decode_8bit_fwd(C.byref(d), None) == -6
