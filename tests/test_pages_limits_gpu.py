"""Page operators at the sizes where a kernel's shared memory passes what is granted without asking
(48 KB, the kernel's own variables included), and from several host threads at once."""
import os
import subprocess
import sys
import threading

import pytest
import torch

from oracle import paged_cache_oracle as orc

pytestmark = pytest.mark.gpu
i32 = torch.int32
HERE = os.path.dirname(os.path.abspath(__file__))

# Ascending, so that no call profits from a larger one before it.
# 4 * (pages + 8 * slots) bytes of a fork in one launch, 4 * slots of one with its books in a cluster
FORKS = [(64, 11743), (64, 11744), (64, 11745), (64, 11776), (128, 11264), (256, 10240), (512, 8192), (1024, 4096), (64, 11777)]
CLUSTER_FORKS = [12256, 12257, 12288, 12289]
# 4 * (pages + 2 * (pages / 2 + 1)) bytes of a compaction in one launch
COMPACTIONS = [6126, 6127, 6128, 6140, 6143, 6144]
# 4 * (3 * slots + pages) bytes of a hand-out by one CTA
HAND_OUTS = [(1, 100, 12249), (1, 100, 12250), (1, 100, 12280), (64, 8, 12096), (1, 100, 12285), (1, 100, 12286)]


def book(slots, width, pages):
    """Every other page held, row after row; pages of 16 tokens, the last of a row half full."""
    table = torch.full((slots, width), -1, dtype=i32)
    refs = torch.zeros(pages, dtype=i32)
    n = min(width, max(pages // (3 * slots), 1))
    at = (2 * torch.arange(slots * n, dtype=i32) + 1) % (pages - 1 + pages % 2)     # (odd, distinct while they fit)
    at = at[:min(slots * n, pages // 3)]
    rows = torch.full((slots * n,), -1, dtype=i32)
    rows[:len(at)] = at
    table[:, :n] = rows.view(slots, n)
    refs[at.long()] = 1
    return table, ((table >= 0).sum(1) * 16 - 8).clamp(min=0).int(), refs


def same(got, want, what):
    for x, y in zip(got, want):
        assert torch.equal(x.cpu(), y), what


def fork(slots, pages, width):
    from tritonops_b200 import ops
    table, lens, refs = book(slots, width, pages)
    pool = torch.arange(pages * 4, dtype=i32).view(pages, 4)
    dev = pool.cuda()
    par = torch.arange(slots, dtype=i32) // 4 * 4
    got = ops.fork_pages([dev], table.cuda(), lens.cuda(), refs.cuda(), par.cuda(), page_size=16)
    want = orc.fork([pool], table, lens, refs, par, 16)
    same((*got, dev), (*want[:4], want[4][0]), ("fork", slots, pages))


def compact(pages):
    from tritonops_b200 import ops
    table, _, refs = book(16, 40, pages)
    pool = torch.arange(pages * 4, dtype=i32).view(pages, 4)
    dev = pool.cuda()
    got = ops.compact_pages([dev], table.cuda(), refs.cuda())
    want = orc.compact([pool], table, refs)
    same((*got, dev), (*want[:3], want[3][0]), ("compact", pages))


def grow(slots, width, pages):
    from tritonops_b200 import ops
    table, lens, refs = book(slots, width, pages)
    new = torch.full((slots,), 40, dtype=i32)
    got = ops.grow_pages(table.cuda(), lens.cuda(), refs.cuda(), new.cuda(), page_size=16)
    same(got, orc.grow(table, lens, refs, new, 16), ("grow", slots, pages))


def every_size():
    failed = []
    for call, sizes in ((lambda s: fork(*s, 4), FORKS), (compact, COMPACTIONS), (lambda s: grow(*s), HAND_OUTS),
                        (lambda s: fork(s, s, 1), CLUSTER_FORKS)):
        for s in sizes:
            try:
                call(s)
            except (RuntimeError, ValueError) as e:
                failed.append((s, str(e)))
    assert not failed, failed


def test_sizes_at_the_granted_shared_memory():
    """In a process of its own: no kernel's limit has been raised before."""
    code = f"import sys; sys.path[:0] = [{os.path.dirname(HERE)!r}, {HERE!r}]; import test_pages_limits_gpu as t; t.every_size()"
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-4000:]


def in_threads(*calls):
    """Each of `calls` over and over on four threads with a stream each; what they raised."""
    calls = calls * 4
    raised, ready = [], threading.Barrier(len(calls), timeout=60)
    torch.cuda.synchronize()

    def loop(call):
        with torch.cuda.stream(torch.cuda.Stream()):
            ready.wait()
            try:
                for _ in range(10000):
                    call()
            except (RuntimeError, ValueError) as e:
                raised.append(str(e))

    threads = [threading.Thread(target=loop, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    return raised


def test_small_and_large_books_from_several_threads():
    """No call lowers the limit that another thread's launch relies on."""
    from tritonops_b200 import ops

    def forks(slots, pages):
        table, lens, refs = (t.cuda() for t in book(slots, 4, pages))
        par = torch.arange(slots, dtype=i32, device="cuda") // 4 * 4
        return lambda: ops.fork_pages([], table, lens, refs, par, page_size=16)

    def compactions(pages):
        table, _, refs = (t.cuda() for t in book(16, 40, pages))
        return lambda: ops.compact_pages([], table, refs)

    bad = []
    bad += in_threads(forks(64, 12400), forks(64, 28000))
    bad += in_threads(compactions(6400), compactions(14000))
    bad += in_threads(forks(12400, 12400), forks(32768, 32768))
    assert not bad
