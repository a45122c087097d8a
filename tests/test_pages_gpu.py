"""Hand-out, forking, freeing and compaction of cache pages against the plain Python of
oracle/paged_cache_oracle.py: whole numbers and moved bytes, so everything is compared for equality."""
import random

import pytest
import torch

from oracle import paged_cache_oracle as orc

pytestmark = pytest.mark.gpu
i32 = torch.int32


def book(seed, slots, width, pages, page_size, fill=0.7, bad=False):
    """A table whose rows hold distinct pages, its counts and lengths; `bad`: entries that name no page."""
    r = random.Random(seed)
    free = list(range(pages))
    r.shuffle(free)
    table, lens, refs = [], [], [0] * pages
    for _ in range(slots):
        n = min(r.randint(0, int(width * page_size * fill)), len(free) * page_size)
        row = [free.pop() for _ in range(-(-n // page_size))]
        for e in row:
            refs[e] += 1
        row += [-1] * (width - len(row))
        if bad and r.random() < 0.5:
            at = r.randrange(width)
            if row[at] >= 0:
                refs[row[at]] -= 1
            row[at] = r.choice([-5, pages, 2 ** 31 - 1])
        table.append(row)
        lens.append(n)
    return torch.tensor(table, dtype=i32), torch.tensor(lens, dtype=i32), torch.tensor(refs, dtype=i32)


def same(got, want):
    assert len(got) == len(want)
    for x, y in zip(got, want):
        assert torch.equal(x.cpu(), y), (x.cpu(), y)


SHAPES = [(1, 1, 1, 16), (3, 5, 8, 16), (8, 7, 40, 32), (33, 17, 300, 64), (256, 40, 6000, 16), (1500, 9, 9000, 48)]


@pytest.mark.parametrize("bad", [False, True])
@pytest.mark.parametrize("slots,width,pages,size", SHAPES)
def test_grow(slots, width, pages, size, bad):
    from tritonops_b200 import ops
    table, lens, refs = book(1, slots, width, pages, size, bad=bad)
    r = random.Random(2)
    for most in (0, 1, size + 1, 5 * size, width * size * 2):
        new = torch.tensor([r.randint(-1, most) for _ in range(slots)], dtype=i32)
        got = ops.grow_pages(table.cuda(), lens.cuda(), refs.cuda(), new.cuda(), page_size=size)
        same(got, orc.grow(table, lens, refs, new, size))
        # the same again asks for nothing more
        t2, r2, _ = ops.grow_pages(got[0], lens.cuda(), got[1], new.cuda(), page_size=size)
        assert torch.equal(t2, got[0]) and torch.equal(r2, got[1])


def test_grow_lengths_beyond_32_bits_and_negative_ones():
    from tritonops_b200 import ops
    table = torch.full((3, 4), -1, dtype=i32)
    lens = torch.tensor([2 ** 31 - 1, -7, 0], dtype=i32)
    new = torch.tensor([2 ** 31 - 1, 20, -3], dtype=i32)
    refs = torch.zeros(20, dtype=i32)
    got = ops.grow_pages(table.cuda(), lens.cuda(), refs.cuda(), new.cuda(), page_size=16)
    want = orc.grow(table, lens, refs, new, 16)
    same(got, want)


def pools_for(pages, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(pages, 16, 2, 32, generator=g).to(torch.bfloat16),
            torch.randint(-127, 128, (pages, 16, 2, 32), generator=g, dtype=torch.int8),
            torch.randn(pages, 1, 2, generator=g),                       # 8 bytes a page
            torch.randn(pages, 3, generator=g),                          # 12 bytes
            torch.randn(pages, 40, 111, generator=g)]                    # 17760: more than one unit, 16-byte pieces


@pytest.mark.parametrize("bad", [False, True])
@pytest.mark.parametrize("slots,width,pages,size", SHAPES)
def test_fork(slots, width, pages, size, bad):
    from tritonops_b200 import ops
    table, lens, refs = book(3, slots, width, pages, size, fill=0.5, bad=bad)
    pools = pools_for(pages, 1)
    r = random.Random(4)
    cases = [list(range(slots)), [-1] * slots, [0] * slots, [slots - 1] * slots, list(range(slots))[::-1],
             [r.randrange(-2, slots + 2) for _ in range(slots)], [b - b % 4 for b in range(slots)]]
    for parents in cases:
        par = torch.tensor(parents, dtype=i32)
        dev = [p.cuda() for p in pools]
        got = ops.fork_pages(dev, table.cuda(), lens.cuda(), refs.cuda(), par.cuda(), page_size=size)
        want = orc.fork(pools, table, lens, refs, par, size)
        same(got, want[:4])
        same(dev, want[4])


def test_fork_chain_shares_and_frees():
    """Forked twice, then all but one slot freed: the counts return to one row's."""
    from tritonops_b200 import ops
    table, lens, refs = book(5, 6, 8, 200, 16)
    lens = torch.clamp(lens, min=0)
    pools = [torch.randn(200, 16, 2, 32)]
    dev = [p.cuda() for p in pools]
    state = (table.cuda(), lens.cuda(), refs.cuda())
    ref = (pools, table, lens, refs)
    for parents in ([0, 0, 0, 3, 3, 5], [1, 1, 4, 4, 4, 4], [-1, -1, -1, 3, -1, -1]):
        par = torch.tensor(parents, dtype=i32)
        state = ops.fork_pages(dev, *state, par.cuda(), page_size=16)[:3]
        want = orc.fork(*ref, par, 16)
        ref = (want[4], *want[:3])
        same(state, want[:3])
        same(dev, want[4])
    held = int((state[0] >= 0).sum())
    assert int(state[2].sum()) == held and int(state[2].max()) == 1


def test_fork_of_lengths_past_the_row():
    from tritonops_b200 import ops
    table = torch.tensor([[0, 1], [2, -1]], dtype=i32)
    lens = torch.tensor([1000, -4], dtype=i32)
    refs = torch.tensor([1, 1, 1, 0], dtype=i32)
    par = torch.tensor([1, 0], dtype=i32)
    pool = torch.randn(4, 16)
    dev = pool.cuda()
    got = ops.fork_pages([dev], table.cuda(), lens.cuda(), refs.cuda(), par.cuda(), page_size=16)
    want = orc.fork([pool], table, lens, refs, par, 16)
    same(got, want[:4])
    assert torch.equal(dev.cpu(), want[4][0])


@pytest.mark.parametrize("count", [0, 1, 128, 129, 300])
def test_any_number_of_pools(count):
    from tritonops_b200 import ops
    table, lens, refs = book(6, 4, 5, 30, 16)
    lens[0] = max(int(lens[0]), 1)
    pools = [torch.randn(30, 16 + i % 7) for i in range(count)]
    dev = [p.cuda() for p in pools]
    par = torch.tensor([0, 0, 0, 3], dtype=i32)
    got = ops.fork_pages(dev, table.cuda(), lens.cuda(), refs.cuda(), par.cuda(), page_size=16)
    want = orc.fork(pools, table, lens, refs, par, 16)
    same(got, want[:4])
    same(dev, want[4])


@pytest.mark.parametrize("bad", [False, True])
@pytest.mark.parametrize("slots,width,pages,size", SHAPES)
def test_compact(slots, width, pages, size, bad):
    from tritonops_b200 import ops
    for seed in range(3):
        table, lens, refs = book(7 + seed, slots, width, pages, size, fill=0.3 * (seed + 0.1), bad=bad)
        if bad:     # a page nobody lists any more, and one that a row lists without a count
            refs[0], refs[pages // 2] = 2, -3
        pools = pools_for(pages, 2)
        dev = [p.cuda() for p in pools]
        got = ops.compact_pages(dev, table.cuda(), refs.cuda())
        want = orc.compact(pools, table, refs)
        same(got, want[:3])
        live = int(want[2])
        same([d[:live] for d in dev], [p[:live] for p in want[3]])
        same(dev, want[3])      # pages past the front are left as they were


def test_pools_with_room_between_pages():
    from tritonops_b200 import ops
    table, lens, refs = book(8, 6, 6, 64, 16)
    wide = torch.randn(64, 2, 16, 2, 32)
    dev = wide.cuda()
    par = torch.tensor([0, 0, 2, 2, 4, 4], dtype=i32)
    got = ops.fork_pages([dev[:, 1]], table.cuda(), lens.cuda(), refs.cuda(), par.cuda(), page_size=16)
    want = orc.fork([wide[:, 1]], table, lens, refs, par, 16)
    same(got, want[:4])
    assert torch.equal(dev[:, 1].cpu(), want[4][0]) and torch.equal(dev[:, 0].cpu(), wide[:, 0])


def test_captured_and_replayed_with_other_inputs():
    """One graph of hand-out, fork and compaction, replayed after its inputs changed; two graphs at once
    keep workspaces of their own."""
    from tritonops_b200 import ops
    sets = [book(20 + i, 12, 10, 90, 16, fill=0.4) for i in range(2)]
    new = torch.tensor([5 * i for i in range(12)], dtype=i32)
    par = torch.tensor([b - b % 3 for b in range(12)], dtype=i32)
    pool = torch.randn(90, 16, 2, 32)
    fixed = [t.cuda() for t in sets[0]] + [new.cuda(), par.cuda()]
    dev = pool.cuda()

    def step():
        t, r, _ = ops.grow_pages(fixed[0], fixed[1], fixed[2], fixed[3], page_size=16)
        t, n, r, _ = ops.fork_pages([dev], t, fixed[1], r, fixed[4], page_size=16)
        return (*ops.compact_pages([dev], t, r), n)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for which in (0, 1):
        for dst, src in zip(fixed, sets[which]):
            dst.copy_(src)
        table, lens, refs = sets[which]
        dev.copy_(pool)
        graphs[which].replay()
        torch.cuda.synchronize()
        t, r, _ = orc.grow(table, lens, refs, new, 16)
        t, n, r, _, pools = orc.fork([pool], t, lens, r, par, 16)
        t, r, live, pools = orc.compact(pools, t, r)
        same(outs[which], (t, r, live, n))
        assert torch.equal(dev.cpu(), pools[0])


def test_on_another_stream():
    from tritonops_b200 import ops
    table, lens, refs = book(9, 8, 6, 64, 16)
    pool = torch.randn(64, 16, 2, 32)
    par = torch.tensor([0, 0, 0, 0, 4, 4, 4, 4], dtype=i32)
    args = [t.cuda() for t in (pool, table, lens, refs, par)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.fork_pages([args[0]], *args[1:], page_size=16)
    s.synchronize()
    want = orc.fork([pool], table, lens, refs, par, 16)
    same(got, want[:4])
    assert torch.equal(args[0].cpu(), want[4][0])


def test_refusals():
    from tritonops_b200 import ops
    table, lens, refs = (t.cuda() for t in book(10, 4, 4, 20, 16))
    par = torch.zeros(4, dtype=i32, device="cuda")
    pool = torch.zeros(20, 16, device="cuda")
    with pytest.raises(ValueError, match="int32"):
        ops.grow_pages(table.long(), lens, refs, par, page_size=16)
    with pytest.raises(ValueError, match="each slot"):
        ops.grow_pages(table, lens[:3], refs, par, page_size=16)
    with pytest.raises(ValueError):
        ops.grow_pages(table, lens, refs, par, page_size=0)
    with pytest.raises(ValueError, match="pools"):
        ops.fork_pages([pool[:19]], table, lens, refs, par, page_size=16)
    with pytest.raises(ValueError, match="contiguous"):
        ops.fork_pages([torch.zeros(20, 4, 16, device="cuda").transpose(1, 2)], table, lens, refs, par, page_size=16)
    with pytest.raises(ValueError, match="multiples of 4"):
        ops.compact_pages([torch.zeros(20, 3, dtype=torch.int8, device="cuda")], table, refs)
    with pytest.raises(ValueError, match="apart"):
        ops.compact_pages([pool[:1].expand(20, 16)], table, refs)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.compact_pages([pool.cpu()], table, refs)


@pytest.mark.parametrize("slots,width,pages,size", [(40, 30, 40000, 16), (300, 90, 60001, 32)])
def test_books_beyond_shared_memory(slots, width, pages, size):
    """The form in which a cluster keeps the books and another kernel copies."""
    from tritonops_b200 import ops
    table, lens, refs = book(11, slots, width, pages, size, fill=0.6, bad=True)
    r = random.Random(12)
    new = torch.tensor([r.randint(0, 5 * size) for _ in range(slots)], dtype=i32)
    same(ops.grow_pages(table.cuda(), lens.cuda(), refs.cuda(), new.cuda(), page_size=size),
         orc.grow(table, lens, refs, new, size))
    pools = [torch.randn(pages, 8), torch.randint(-99, 99, (pages, 12), dtype=torch.int8)]
    for parents in ([b - b % 4 for b in range(slots)], [r.randrange(-2, slots + 2) for _ in range(slots)]):
        par = torch.tensor(parents, dtype=i32)
        dev = [p.cuda() for p in pools]
        got = ops.fork_pages(dev, table.cuda(), lens.cuda(), refs.cuda(), par.cuda(), page_size=size)
        want = orc.fork(pools, table, lens, refs, par, size)
        same(got, want[:4])
        same(dev, want[4])
    refs[0], refs[pages // 2] = 2, -3
    dev = [p.cuda() for p in pools]
    got = ops.compact_pages(dev, table.cuda(), refs.cuda())
    want = orc.compact(pools, table, refs)
    same(got, want[:3])
    same(dev, want[3])


def test_no_page_left():
    """Pages that cannot be given are counted, forks without one lose what is not in a full page."""
    from tritonops_b200 import ops
    table, lens, refs = book(13, 8, 6, 60, 16)
    refs = torch.where(refs <= 0, 1, refs)          # somebody else holds the rest
    pool = torch.randn(60, 16)
    par = torch.tensor([0, 0, 0, 3, 3, 3, 6, 6], dtype=i32)
    got = ops.fork_pages([pool.cuda()], table.cuda(), lens.cuda(), refs.cuda(), par.cuda(), page_size=16)
    want = orc.fork([pool], table, lens, refs, par, 16)
    same(got, want[:4])
    new = torch.full((8,), 20, dtype=i32)
    same(ops.grow_pages(table.cuda(), lens.cuda(), refs.cuda(), new.cuda(), page_size=16), orc.grow(table, lens, refs, new, 16))


@pytest.mark.parametrize("bad", [False, True])
@pytest.mark.parametrize("slots,width,pages,size", [(12000, 3, 20000, 16), (297, 60, 1000, 16), (2, 9000, 70001, 16)])
def test_hand_out_of_large_books(slots, width, pages, size, bad):
    """More rows than CTAs times a warp's look-ups, more CTAs than rows, rows past a CTA's share."""
    from tritonops_b200 import ops
    table, lens, refs = book(91, slots, width, pages, size, bad=bad)
    r = random.Random(92)
    for most in (0, 1, 3 * size, width * size * 2):
        new = torch.tensor([r.randint(-1, most) for _ in range(slots)], dtype=i32)
        got = ops.grow_pages(table.cuda(), lens.cuda(), refs.cuda(), new.cuda(), page_size=size)
        same(got, orc.grow(table, lens, refs, new, size))
