"""The paged cache in 8 bits: the append bit for bit, and attention over it, against the plain float64
Python of oracle/paged_cache_oracle.py.

Tolerance of the attention, from the arithmetic.  The cached numbers are exact in the products
(fp16), which are summed in fp32; what is rounded on the way is
  P, to fp16:      relative 2^-11 of each weight, or 2^-25 of the largest one where a weight is
                   below 2^-14 of it                    -> (2^-11 + 2^-24) * sum w |v|  + 2^-24 * sum |v|
  the scores:      fp32 sums of D products and the rows of Q that were scaled to fp16 (2^-25 of the
                   row's largest element):  |ds| <= scale * (D + 16) * 2^-23 * max|q| sum|k|, which moves a
                   weight by a factor e^(2 ds)          -> 2 ds * sum w |v|, twice for the quotient
  the result:      half a step of its type              -> eps / 2 * |o|
and the quotient's sum of weights is not rounded (fp32)."""
import math
import random

import pytest
import torch

from oracle import paged_cache_oracle as orc

pytestmark = pytest.mark.gpu
E4M3, I8 = torch.float8_e4m3fn, torch.int8
i32 = torch.int32


def bits(t):
    return t.contiguous().view(torch.uint8) if t.element_size() == 1 else t


def same_bits(a, b):
    a, b = bits(a.cpu()), bits(b.cpu())
    if a.dtype == torch.float32:
        return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(), b.nan_to_num())
    return torch.equal(a, b)


def cache(seed, pages, page, block, heads, D, dtype, junk=True):
    """Pools whose numbers fill their type and scales over a few octaves; `junk`: what no page table
    will name holds NaN (e4m3) or the largest numbers, its scales NaN."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(2, pages, page, heads, D, generator=g)
    x = (x * 90).clamp(-448, 448).to(E4M3) if dtype == E4M3 else (x * 28).clamp(-127, 127).to(I8)
    s = torch.exp2(torch.randint(-7, -4, (2, pages, page // block, heads), generator=g).float())
    return x[0].clone(), x[1].clone(), s[0].clone(), s[1].clone()


def spoil(pools, table, lens):
    """Everything outside the first lens[b] keys of each row: NaN numbers (the largest of int8) and,
    where a whole block is outside, NaN scales."""
    k, v, ks, vs = pools
    pages, page = k.shape[:2]
    per = ks.shape[1]
    used = torch.zeros(pages, page, dtype=torch.bool)
    for row, n in zip(table.tolist(), lens.tolist()):
        for t in range(max(n, 0)):
            if t // page < len(row) and 0 <= row[t // page] < pages:
                used[row[t // page], t % page] = True
    byte = 0x7f
    for p in (k, v):
        p.view(torch.uint8)[~used] = byte
    blocks = used.view(pages, per, page // per).any(-1)
    for s in (ks, vs):
        s[~blocks] = math.nan


def rows_of(seed, lens, page, extra=3):
    r = random.Random(seed)
    used = [-(-max(n, 0) // page) for n in lens]
    order = list(range(sum(used) + extra))
    r.shuffle(order)
    width, at, rows = max(1, max(used)) + 1, 0, []
    for u in used:
        rows.append(order[at:at + u] + [-1] * (width - u))
        at += u
    return torch.tensor(rows, dtype=i32), len(order)


def check(got, q, pools, table, lens, max_seqlen=None, scale=None):
    q4 = q if q.dim() == 4 else q[:, None]
    k, v, ks, vs = pools
    o, mass = orc.attend(q4, k, v, ks, vs, table, lens, max_seqlen, scale)
    D = q4.shape[-1]
    sc = D ** -0.5 if scale is None else abs(scale)
    group = q4.shape[2] // k.shape[2]
    # per row: the largest sum |k| over its keys, sum |v| over its keys
    bound = torch.zeros_like(o)
    cap = table.shape[1] * k.shape[1] if max_seqlen is None else min(max_seqlen, table.shape[1] * k.shape[1])
    for b in range(q4.shape[0]):
        n = min(max(int(lens[b]), 0), cap)
        _, kr = orc.sequence_rows(k, ks, table[b], n)
        _, vr = orc.sequence_rows(v, vs, table[b], n)
        if not len(kr):
            continue
        sk = kr.abs().sum(-1).amax(0).repeat_interleave(group)                    # [Hq]
        sv = vr.abs().sum(0).repeat_interleave(group, 0)                          # [Hq, D]
        ds = sc * (D + 16) * 2.0 ** -23 * q4[b].double().abs().amax(-1) * sk      # [n, Hq]
        bound[b] = (2.0 ** -11 + 2.0 ** -24 + 4 * ds[..., None]) * mass[b] + 2.0 ** -24 * sv
    bound += torch.finfo(q.dtype).eps / 2 * (o.abs() + bound) + 2.0 ** -24 * (1 if q.dtype == torch.float16 else 0)
    err = (got.cpu().double().view(o.shape) - o).abs()
    assert torch.isfinite(got).all()
    assert (err <= bound).all(), (float((err - bound).max()), float((err / bound.clamp(min=1e-30)).max()))


def attend(q, pools, table, lens, **kw):
    from tritonops_b200 import ops
    return ops.paged_decode_8bit(q.cuda(), *(p.cuda() for p in pools), table.cuda(), lens.cuda(), **kw)


LENS = [[1], [0, 5, 16, 17], [333, 64, 1, 128, 15], [1000, 2, 700]]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("cdt", [E4M3, I8])
@pytest.mark.parametrize("D,Hq,Hkv,page,block", [(128, 8, 2, 64, 64), (64, 4, 4, 16, 16), (96, 6, 1, 48, 16),
                                                 (32, 20, 1, 32, 32), (128, 32, 2, 128, 128), (128, 9, 1, 128, 16),
                                                 (64, 34, 2, 64, 32)])
def test_one_token(dtype, cdt, D, Hq, Hkv, page, block):
    for i, lens in enumerate(LENS):
        table, pages = rows_of(i, lens, page)
        n = torch.tensor(lens, dtype=i32)
        pools = cache(i, pages, page, block, Hkv, D, cdt)
        spoil(pools, table, n)
        q = torch.randn(len(lens), Hq, D, generator=torch.Generator().manual_seed(i)).to(dtype)
        check(attend(q, pools, table, n), q, pools, table, n)


@pytest.mark.parametrize("cdt", [E4M3, I8])
@pytest.mark.parametrize("n,Hq,Hkv,D,page,block", [(2, 8, 2, 128, 64, 64), (5, 8, 2, 64, 16, 16), (7, 4, 4, 96, 32, 16),
                                                   (16, 4, 1, 128, 64, 32), (33, 3, 1, 32, 16, 16), (3, 40, 2, 128, 64, 64)])
def test_newest_tokens(cdt, n, Hq, Hkv, D, page, block):
    """Also sequences shorter than the queries: the first ones see nothing and give 0."""
    lens = torch.tensor([n + 200, n, 1, 0, n // 2 + 1, 517], dtype=i32)
    table, pages = rows_of(1, lens.tolist(), page)
    pools = cache(2, pages, page, block, Hkv, D, cdt)
    spoil(pools, table, lens)
    q = torch.randn(6, n, Hq, D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    got = attend(q, pools, table, lens)
    check(got, q, pools, table, lens)
    assert (got[3] == 0).all() and (got[2, :n - 1] == 0).all()
    # one token is the same call with n = 1
    a = attend(q[:, -1:], pools, table, lens)
    b = attend(q[:, -1], pools, table, lens)
    assert torch.equal(a[:, 0], b)


@pytest.mark.parametrize("chunk", [128, 256, 1024])
@pytest.mark.parametrize("cdt", [E4M3, I8])
def test_splits(chunk, cdt):
    lens = torch.tensor([4000, 129, 128, 1, 0, 2500], dtype=i32)
    table, pages = rows_of(5, lens.tolist(), 64)
    pools = cache(6, pages, 64, 16, 2, 128, cdt)
    spoil(pools, table, lens)
    q = torch.randn(6, 8, 128, generator=torch.Generator().manual_seed(7)).half()
    check(attend(q, pools, table, lens, chunk=chunk), q, pools, table, lens)
    check(attend(q, pools, table, lens, chunk=chunk, max_seqlen=2000), q, pools, table, lens, max_seqlen=2000)


def test_more_items_than_fit_the_chip():
    lens = torch.tensor([random.Random(8).randint(0, 900) for _ in range(90)], dtype=i32)
    table, pages = rows_of(9, lens.tolist(), 16)
    pools = cache(10, pages, 16, 16, 8, 64, E4M3)
    q = torch.randn(90, 8, 64, generator=torch.Generator().manual_seed(11)).half()
    check(attend(q, pools, table, lens, chunk=128), q, pools, table, lens)


def test_scales_of_any_size():
    """Scales that are no powers of two, far apart, zero: as given."""
    lens = torch.tensor([500, 77], dtype=i32)
    table, pages = rows_of(12, lens.tolist(), 32)
    k, v, ks, vs = cache(13, pages, 32, 16, 2, 128, I8)
    g = torch.Generator().manual_seed(14)
    ks = torch.rand(ks.shape, generator=g) * 0.02
    vs = torch.exp2(torch.randint(-40, 20, vs.shape, generator=g).float()) * (1 + torch.rand(vs.shape, generator=g))
    vs[torch.rand(vs.shape, generator=g) < 0.2] = 0
    ks[torch.rand(ks.shape, generator=g) < 0.2] = 0
    q = torch.randn(2, 8, 128, generator=g).to(torch.bfloat16)
    pools = (k, v, ks, vs)
    check(attend(q, pools, table, lens), q, pools, table, lens)


@pytest.mark.parametrize("scale", [0.0, 3.0, -0.5])
def test_sharp_and_flat_weights(scale):
    lens = torch.tensor([700, 3], dtype=i32)
    table, pages = rows_of(15, lens.tolist(), 64)
    pools = cache(16, pages, 64, 64, 2, 64, E4M3)
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(17)).half()
    check(attend(q, pools, table, lens, scale=scale), q, pools, table, lens, scale=scale)


def test_queries_of_any_size():
    """bf16 rows far outside fp16's range, rows of zeros."""
    lens = torch.tensor([300] * 5, dtype=i32)
    table, pages = rows_of(18, lens.tolist(), 64)
    pools = cache(19, pages, 64, 64, 1, 128, E4M3)
    q = torch.randn(5, 4, 128, generator=torch.Generator().manual_seed(20))
    q = (q * torch.tensor([1e-30, 1e-6, 0.0, 1.0, 1e4])[:, None, None]).to(torch.bfloat16)
    check(attend(q, pools, table, lens, scale=1e-4), q, pools, table, lens, scale=1e-4)


def test_pages_outside_the_pool_are_left_out():
    lens = torch.tensor([200, 200, 64], dtype=i32)
    table, pages = rows_of(21, lens.tolist(), 16)
    table[0, 3], table[0, 7], table[1, 0], table[1, 12], table[2, :4] = -1, pages, 2 ** 31 - 1, -2 ** 31, -9
    pools = cache(22, pages, 16, 16, 2, 128, E4M3)
    spoil(pools, table, lens)
    q = torch.randn(3, 8, 128, generator=torch.Generator().manual_seed(23)).half()
    got = attend(q, pools, table, lens)
    check(got, q, pools, table, lens)
    assert (got[2] == 0).all()
    q = torch.randn(3, 4, 8, 128, generator=torch.Generator().manual_seed(23)).half()
    check(attend(q, pools, table, lens), q, pools, table, lens)


def test_not_a_number_stays_visible():
    lens = torch.tensor([100, 100], dtype=i32)
    table, pages = rows_of(24, lens.tolist(), 64)
    k, v, ks, vs = cache(25, pages, 64, 64, 2, 64, E4M3)
    k.view(torch.uint8)[table[0, 0], 5, 0, 3] = 0x7f
    v.view(torch.uint8)[table[1, 1], 5, 1, 9] = 0x7f
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(26)).half()
    got = attend(q, (k, v, ks, vs), table, lens).cpu()
    assert got[0, :2].isnan().all() and got[0, 2:].isfinite().all()
    assert got[1, :2].isfinite().all() and got[1, 2:, 9].isnan().all()
    assert got[1, 2:].isnan().sum() == 2


def test_other_layouts():
    """Pools with heads outside tokens, with room between rows; strided and misaligned queries; int64 tables."""
    lens = torch.tensor([150, 33], dtype=i32)
    table, pages = rows_of(27, lens.tolist(), 32)
    k, v, ks, vs = cache(28, pages, 32, 16, 2, 64, I8)
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(29)).half()
    want = attend(q, (k, v, ks, vs), table, lens)
    check(want, q, (k, v, ks, vs), table, lens)
    heads_out = k.cuda().permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    roomy = torch.zeros(pages, 32, 2, 96, dtype=I8, device="cuda")[..., 16:80]
    roomy.copy_(v.cuda())
    scales = ks.cuda().permute(2, 0, 1).contiguous().permute(1, 2, 0)
    from tritonops_b200 import ops
    wide = torch.zeros(2, 4, 65, dtype=torch.float16, device="cuda")[..., 1:]
    wide.copy_(q.cuda())
    got = ops.paged_decode_8bit(wide, heads_out, roomy, scales, vs.cuda(), table.cuda().long(), lens.cuda().long())
    assert torch.equal(got, want)


def test_far_into_a_large_pool():
    """Pages whose bytes lie past 32-bit offsets."""
    from tritonops_b200 import ops
    page, heads, D = 64, 32, 128
    pages = (5 << 30) // (page * heads * D)
    lens = torch.tensor([130, 64], dtype=i32)
    table = torch.tensor([[pages - 1, 3, pages - 7], [pages - 2, -1, -1]], dtype=i32)
    pools = [torch.zeros(pages, page, heads, D, dtype=I8, device="cuda") for _ in range(2)]
    scales = [torch.zeros(pages, 4, heads, device="cuda") for _ in range(2)]
    g = torch.Generator().manual_seed(30)
    rows = [torch.randn(194, heads, D, generator=g).half() for _ in range(2)]
    ops.append_kv_8bit(*pools, *scales, rows[0].cuda(), rows[1].cuda(), table.cuda(),
                       torch.zeros(2, dtype=i32, device="cuda"), cu_new=torch.tensor([0, 130, 194], dtype=i32).cuda())
    q = torch.randn(2, 32, D, generator=g).half()
    got = ops.paged_decode_8bit(q.cuda(), *pools, *scales, table.cuda(), lens.cuda())
    near = sorted({pages - 1, 3, pages - 7, pages - 2})
    small = [t[torch.tensor(near).cuda()].cpu() for t in (*pools, *scales)]
    moved = torch.tensor([[near.index(e) if e >= 0 else -1 for e in r] for r in table.tolist()], dtype=i32)
    zero = [torch.zeros_like(t) for t in small]
    want = orc.append(*zero, *rows, moved, torch.zeros(2, dtype=i32), [130, 64])
    for a, b in zip(small, want):
        assert same_bits(a, b)
    check(got, q, small, moved, lens)


# ---------------------------------------------------------------------------- append
def append(pools, new_k, new_v, table, lens, cu=None):
    from tritonops_b200 import ops
    dev = [p.cuda() for p in pools]
    ops.append_kv_8bit(*dev, new_k.cuda(), new_v.cuda(), table.cuda(), lens.cuda(),
                       cu_new=None if cu is None else cu.cuda())
    return dev


def equal_cache(dev, want):
    for name, a, b in zip(("k", "v", "ks", "vs"), dev, want):
        assert same_bits(a, b), name


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("cdt", [E4M3, I8])
@pytest.mark.parametrize("D,heads,page,block", [(128, 2, 64, 64), (64, 3, 16, 16), (96, 1, 48, 16), (32, 5, 128, 32),
                                                (128, 9, 128, 128)])
def test_append(dtype, cdt, D, heads, page, block):
    """One row each and packed rows: fresh blocks, blocks already begun (with scales above and below
    what the new rows need), several blocks and pages, sequences without new rows."""
    g = torch.Generator().manual_seed(31)
    lens = torch.tensor([0, 1, 15, 16, 100, page - 1, page], dtype=i32)
    B = len(lens)
    for counts in ([1] * B, [0, 1, 2, 0, 70, 300, 17]):
        after = [n + m for n, m in zip(lens.tolist(), counts)]
        table, pages = rows_of(32, after, page)
        pools = cache(33, pages, page, block, heads, D, cdt)
        T = sum(counts)
        x = torch.randn(2, T, heads, D, generator=g) * torch.exp2(torch.randint(-3, 4, (2, T, 1, 1), generator=g).float())
        nk, nv = x.to(dtype)
        cu = None
        if counts != [1] * B:
            cu = torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=i32)
        dev = append(pools, nk, nv, table, lens, cu)
        want = orc.append(*pools, nk, nv, table, lens, counts)
        equal_cache(dev, want)
        if cu is None:      # the same rows as packed ones of one each
            equal_cache(append(pools, nk, nv, table, lens, torch.arange(B + 1, dtype=i32)), want)
        # again over what it wrote: nothing changes
        from tritonops_b200 import ops
        ops.append_kv_8bit(*dev, nk.cuda()[None] if cu is not None else nk.cuda(), nv.cuda()[None] if cu is not None else nv.cuda(),
                           table.cuda(), lens.cuda(), cu_new=None if cu is None else cu.cuda())
        equal_cache(dev, want)


@pytest.mark.parametrize("cdt", [E4M3, I8])
def test_append_odd_values(cdt):
    """Zeros, the smallest and largest numbers, infinities and NaN, foreign scales."""
    D, heads, page, block = 64, 1, 32, 16
    tiny = torch.finfo(torch.bfloat16).tiny
    tops = [0.0, tiny / 64, tiny, 1e-30, 448.0, 449.0, 127.0, 127.5, 1.0, 1.75, 1.76, 3.3e38, math.inf, -math.inf, math.nan]
    rows = torch.zeros(len(tops), heads, D)
    rows[:, 0, :] = torch.linspace(-1, 1, D)[None]
    rows = (rows * torch.tensor([1.0 if not math.isfinite(t) else min(t, 1e38) for t in tops])[:, None, None]).to(torch.bfloat16)
    rows[:, 0, 7] = torch.tensor(tops).to(torch.bfloat16)
    for start, foreign in ((0, None), (5, None), (5, 0.013), (5, 0.0), (5, math.nan), (5, 1e-40), (5, 2.0 ** 127)):
        lens = torch.full((len(tops),), start, dtype=i32)
        table, pages = rows_of(34, [start + 1] * len(tops), page)
        pools = cache(35, pages, page, block, heads, D, cdt)
        if foreign is not None:
            pools[2].fill_(foreign), pools[3].fill_(foreign)
            if foreign == 0.0:
                pools[0].view(torch.uint8).zero_(), pools[1].view(torch.uint8).zero_()
        dev = append(pools, rows, -rows, table, lens)
        equal_cache(dev, orc.append(*pools, rows, -rows, table, lens, [1] * len(tops)))


def test_append_token_by_token():
    """A sequence grown a token at a time holds what it holds when stored at once, in e4m3 (numbers that
    a larger scale does not push into the subnormals)."""
    g = torch.Generator().manual_seed(36)
    D, heads, page, block, n = 128, 2, 64, 64, 150
    x = (torch.rand(2, n, heads, D, generator=g) + 1) * torch.exp2(torch.randint(0, 3, (2, n, heads, 1), generator=g).float())
    nk, nv = x.half()
    table, pages = rows_of(37, [n], page)
    pools = cache(38, pages, page, block, heads, D, E4M3)
    at_once = append(pools, nk, nv, table, torch.tensor([0], dtype=i32), torch.tensor([0, n], dtype=i32))
    from tritonops_b200 import ops
    dev = [p.cuda() for p in pools]
    for t in range(n):
        ops.append_kv_8bit(*dev, nk[t:t + 1].cuda(), nv[t:t + 1].cuda(), table.cuda(), torch.tensor([t], dtype=i32).cuda())
    equal_cache(dev, [p.cpu() for p in at_once])


def test_append_rows_that_go_nowhere():
    """Past the row of the table, pages outside the pool, negative lengths, rows that cu_new does not
    count: nothing else changes."""
    D, heads, page, block = 64, 2, 16, 16
    pages = 12
    pools = cache(39, pages, page, block, heads, D, I8)
    table = torch.tensor([[0, 1], [2, -1], [pages, 3], [4, 5], [6, 7]], dtype=i32)
    lens = torch.tensor([30, 10, 0, -1, 2 ** 31 - 5], dtype=i32)
    counts = [7, 20, 20, 5, 10]
    g = torch.Generator().manual_seed(40)
    T = sum(counts) + 6
    nk, nv = torch.randn(2, T, heads, D, generator=g).half()
    cu = torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=i32)
    equal_cache(append(pools, nk, nv, table, lens, cu), orc.append(*pools, nk, nv, table, lens, counts))
    # more rows counted than given: the ones that exist
    cu2 = cu.clone()
    cu2[-1] = T + 100
    lens2 = torch.tensor([30, 10, 0, -1, 3], dtype=i32)
    want = orc.append(*pools, nk, nv, table, lens2, counts[:-1] + [T - int(cu[-2])])
    equal_cache(append(pools, nk, nv, table, lens2, cu2), want)
    # none at all
    equal_cache(append(pools, nk[:0], nv[:0], table, lens, torch.zeros(6, dtype=i32)), pools)


def test_append_many_sequences_and_layouts():
    """More sequences than a CTA has threads, many of them empty; strided rows and pools."""
    D, heads, page, block = 32, 2, 16, 16
    r = random.Random(41)
    counts = [r.choice([0, 0, 0, 1, 2, 5]) for _ in range(700)]
    lens = torch.tensor([r.randint(0, 40) for _ in counts], dtype=i32)
    table, pages = rows_of(42, [n + m for n, m in zip(lens.tolist(), counts)], page)
    pools = cache(43, pages, page, block, heads, D, E4M3)
    g = torch.Generator().manual_seed(44)
    T = sum(counts)
    nk, nv = torch.randn(2, T, heads, D, generator=g).to(torch.bfloat16)
    cu = torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=i32)
    want = orc.append(*pools, nk, nv, table, lens, counts)
    from tritonops_b200 import ops
    k = pools[0].cuda().view(torch.uint8).permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3).view(E4M3)
    qkv = torch.zeros(T, 3 * heads, D, dtype=torch.bfloat16, device="cuda")
    qkv[:, heads:2 * heads], qkv[:, 2 * heads:] = nk.cuda(), nv.cuda()
    dev = [k, pools[1].cuda(), pools[2].cuda().permute(2, 0, 1).contiguous().permute(1, 2, 0), pools[3].cuda()]
    ops.append_kv_8bit(*dev, qkv[:, heads:2 * heads], qkv[:, 2 * heads:], table.cuda(), lens.cuda(), cu_new=cu.cuda())
    equal_cache(dev, want)


# ---------------------------------------------------------------------------- together
@pytest.mark.parametrize("cdt", [E4M3, I8])
@pytest.mark.parametrize("graph", [False, True])
def test_a_server_step_by_step(cdt, graph):
    """Prompts stored, tokens generated, a sequence forked into beams, beams reordered, sequences
    ended, the pool compacted, more tokens: at every step what the cache holds and what attention
    over it gives are the oracle's.  With `graph` the steps of one token are a replayed graph."""
    from tritonops_b200 import ops
    D, Hq, Hkv, page, block, S, pages, width = 64, 8, 2, 32, 16, 6, 60, 8
    g = torch.Generator().manual_seed(45)
    host = cache(46, pages, page, block, Hkv, D, cdt)
    dev = [p.cuda() for p in host]
    table, lens, refs = torch.full((S, width), -1, dtype=i32), torch.zeros(S, dtype=i32), torch.zeros(pages, dtype=i32)
    state = [t.cuda() for t in (table, lens, refs)]
    counts = [70, 33, 1, 0, 64, 95]
    nk, nv = torch.randn(2, sum(counts), Hkv, D, generator=g).half()
    new = torch.tensor(counts, dtype=i32)
    cu = torch.tensor([0] + list(new.cumsum(0)), dtype=i32)

    t, r, missing = ops.grow_pages(*state, new.cuda(), page_size=page)
    assert int(missing) == 0
    ops.append_kv_8bit(*dev, nk.cuda(), nv.cuda(), t, state[1], cu_new=cu.cuda())
    state = [t, state[1] + new.cuda(), r]
    table, refs, _ = orc.grow(table, lens, refs, new, page)
    host = orc.append(*host, nk, nv, table, lens, counts)
    lens = lens + new

    fixed = [torch.empty_like(x) for x in state]
    rows = [torch.zeros(S, Hkv, D, dtype=torch.float16, device="cuda") for _ in range(2)]
    qd, one, par = torch.zeros(S, Hq, D, dtype=torch.float16, device="cuda"), torch.ones(S, dtype=i32, device="cuda"), \
        torch.zeros(S, dtype=i32, device="cuda")

    def step():
        t, n, r, short = ops.fork_pages(dev, *fixed, par, page_size=page)
        t, r, lacking = ops.grow_pages(t, n, r, one, page_size=page)
        ops.append_kv_8bit(*dev, *rows, t, n)
        o = ops.paged_decode_8bit(qd, *dev, t, n + 1, max_seqlen=width * page)
        return t, n + 1, r, short, lacking, o

    captured = None
    for parents in ([0, 1, 2, 3, 4, 5], [0, 0, 0, 0, 4, 5], [2, 1, 1, 3, 3, 5], [0, 0, 2, 3, 4, 4], [5, 4, 3, 2, 1, 0],
                    [0, 0, 0, 0, 0, 0]):
        x = torch.randn(2, S, Hkv, D, generator=g).half()
        q = torch.randn(S, Hq, D, generator=g).half()
        p = torch.tensor(parents, dtype=i32)
        for dst, src in zip((*rows, qd, par, *fixed), (x[0], x[1], q, p, *state)):
            dst.copy_(src)
        if graph and captured is None:
            keep = [d.clone() for d in dev]
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                step()
            torch.cuda.current_stream().wait_stream(s)
            for d, k in zip(dev, keep):
                d.copy_(k)
            captured = torch.cuda.CUDAGraph()
            with torch.cuda.graph(captured):
                out = step()
        if graph:
            captured.replay()
        else:
            out = step()
        table, lens, refs, short, host = orc.fork(host, table, lens, refs, p, page)
        table, refs, lacking = orc.grow(table, lens, refs, torch.ones(S, dtype=i32), page)
        host = orc.append(*host, x[0], x[1], table, lens, [1] * S)
        lens = lens + 1
        for a, b in zip(out[:5], (table, lens, refs, short, lacking)):
            assert torch.equal(a.cpu(), b)
        assert int(short) == 0 and int(lacking) == 0
        equal_cache(dev, host)
        check(out[5], q, host, table, lens)
        state = [a.clone() for a in out[:3]]

    p = torch.tensor([-1, 1, -1, 3, -1, -1], dtype=i32)
    state = list(ops.fork_pages(dev, *state, p.cuda(), page_size=page)[:3])
    t, r, live = ops.compact_pages(dev, state[0], state[2])
    table, lens, refs, _, host = orc.fork(host, table, lens, refs, p, page)
    table, refs, n, host = orc.compact(host, table, refs)
    assert torch.equal(t.cpu(), table) and torch.equal(r.cpu(), refs) and int(live) == int(n)
    equal_cache(dev, host)
    small = [d[:int(live)].clone() for d in dev]          # the pool can be cut there
    q = torch.randn(S, 3, Hq, D, generator=g).half()
    got = ops.paged_decode_8bit(q.cuda(), *small, t, state[1])
    check(got, q, [h[:int(n)] for h in host], table, lens)


def test_two_graphs_share_nothing():
    """Two captured calls replayed in turn and on two streams at once give what the eager calls give."""
    from tritonops_b200 import ops
    lens = torch.tensor([2000, 900, 1500], dtype=i32)
    table, pages = rows_of(50, lens.tolist(), 64)
    pools = [p.cuda() for p in cache(51, pages, 64, 64, 2, 128, E4M3)]
    qs = [torch.randn(3, 8, 128, generator=torch.Generator().manual_seed(i)).half().cuda() for i in (52, 53)]
    t, n = table.cuda(), lens.cuda()
    want = [ops.paged_decode_8bit(q, *pools, t, n) for q in qs]
    graphs, outs = [], []
    for q in qs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(ops.paged_decode_8bit(q, *pools, t, n))
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    for _ in range(3):
        for gr, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
    torch.cuda.synchronize()
    for a, b in zip(outs, want):
        assert torch.equal(a, b)


def test_refusals():
    from tritonops_b200 import ops
    lens = torch.tensor([20, 5], dtype=i32)
    table, pages = rows_of(54, lens.tolist(), 32)
    k, v, ks, vs = (p.cuda() for p in cache(55, pages, 32, 16, 2, 64, I8))
    q = torch.zeros(2, 4, 64, dtype=torch.float16, device="cuda")
    t, n = table.cuda(), lens.cuda()
    new = torch.zeros(2, 2, 64, dtype=torch.float16, device="cuda")
    bad = [
        lambda: ops.paged_decode_8bit(q.float(), k, v, ks, vs, t, n),
        lambda: ops.paged_decode_8bit(q, k.to(torch.uint8), v, ks, vs, t, n),
        lambda: ops.paged_decode_8bit(q, k, v.view(E4M3), ks, vs, t, n),
        lambda: ops.paged_decode_8bit(q[..., :32], k, v, ks, vs, t, n),
        lambda: ops.paged_decode_8bit(q[:, :3], k, v, ks, vs, t, n),
        lambda: ops.paged_decode_8bit(q, k, v, ks.half(), vs, t, n),
        lambda: ops.paged_decode_8bit(q, k, v, ks[:, :1].expand(-1, 3, -1), vs[:, :1].expand(-1, 3, -1), t, n),
        lambda: ops.paged_decode_8bit(q, k, v, ks[:-1], vs[:-1], t, n),
        lambda: ops.paged_decode_8bit(q, k, v, ks, vs, t[:1], n),
        lambda: ops.paged_decode_8bit(q, k, v, ks, vs, t, n[:1]),
        lambda: ops.paged_decode_8bit(q, k, v, ks, vs, t, n, chunk=100),
        lambda: ops.paged_decode_8bit(q, k[..., :24], v[..., :24], ks, vs, t, n),
        lambda: ops.append_kv_8bit(k, v, ks, vs, new.float(), new.float(), t, n),
        lambda: ops.append_kv_8bit(k, v, ks, vs, new, new[:1], t, n),
        lambda: ops.append_kv_8bit(k, v, ks, vs, new[:1], new[:1], t, n),
        lambda: ops.append_kv_8bit(k, v, ks, vs, new, new, t, n, cu_new=n),
        lambda: ops.append_kv_8bit(k, v, ks, vs, new[:, :1], new[:, :1], t, n),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.paged_decode_8bit(q.cpu(), k, v, ks, vs, t, n)
    assert ops.paged_decode_8bit(q[:0], k, v, ks, vs, t[:0], n[:0]).shape == (0, 4, 64)


def test_native_calls_equal_python_calls(monkeypatch):
    """Same bits from the native call path and the Python one, and who answered."""
    from tritonops_b200 import ops
    lens = torch.tensor([300, 17, 0], dtype=i32)
    table, pages = rows_of(56, [n + 40 for n in lens.tolist()], 32)
    host = cache(57, pages, 32, 16, 2, 64, I8)
    g = torch.Generator().manual_seed(58)
    q, rows = torch.randn(3, 2, 8, 64, generator=g).half().cuda(), torch.randn(2, 9, 2, 64, generator=g).half().cuda()
    t, n, cu = table.cuda(), lens.cuda(), torch.tensor([0, 4, 4, 9], dtype=i32).cuda()
    refs = torch.zeros(pages, dtype=i32)
    refs[table[table >= 0].long()] = 1
    refs, par, new = refs.cuda(), torch.tensor([0, 0, 2], dtype=i32).cuda(), torch.tensor([50, 0, 3], dtype=i32).cuda()

    def results():
        dev = [p.cuda() for p in host]
        out = [ops.paged_decode_8bit(q, *dev, t, n), ops.paged_decode_8bit(q[:, 0], *dev, t, n, max_seqlen=200, scale=0.3),
               ops.paged_decode_8bit(q[:, 1], *dev, t.long(), n, chunk=128),          # left to Python
               ops.paged_decode_8bit(q[..., 1:].contiguous()[..., :32], *(p[..., :32] if p.dim() == 4 else p for p in dev),
                                     t, n)]                                           # rows off 16 bytes: Python
        ops.append_kv_8bit(*dev, rows[0], rows[1], t, n, cu_new=cu)
        ops.append_kv_8bit(*dev, rows[0][:3], rows[1][:3], t, n + 20)
        ops.append_kv_8bit(*dev, rows[0][None], rows[1][None], t, n, cu_new=cu)       # left to Python
        out += [*ops.grow_pages(t, n, refs, new, page_size=32), *ops.fork_pages(dev, t, n, refs, par, page_size=32),
                *ops.fork_pages(iter(dev), t, n, refs, par, page_size=32),            # left to Python
                *ops.compact_pages(tuple(dev), t, refs)]
        return [bits(x).cpu() for x in out + dev]

    real, answered = ops._native, []

    def spy(name, *args):
        r = real(name, *args)
        answered.append((name, r is not None))
        return r

    monkeypatch.setattr(ops, "_native", spy)
    native = results()
    decode = [a for name, a in answered if name == "paged_decode_8bit"]
    assert decode == [True, True, False, False]
    assert [a for name, a in answered if name == "append_kv_8bit"] == [True, True, False]
    assert [a for name, a in answered if name.endswith("_pages")] == [True, True, False, True]
    monkeypatch.setattr(ops, "_native", lambda *a: None)
    for i, (a, b) in enumerate(zip(native, results())):
        assert same_bits(a, b), i


# ---------------------------------------------------------------------------- sizes past the kernels' own
def test_append_more_blocks_than_a_cta_lists():
    """One prompt of 620,000 rows beside a short one: what one call stores is, bit for bit, what calls of
    100,000 rows store (whole blocks, so their scales are the same)."""
    from tritonops_b200 import ops
    D, page, block = 32, 64, 16
    T, step = 620_000, 100_000
    pages = -(-T // page) + 3
    g = torch.Generator().manual_seed(57)
    x = (torch.randn(2, T + 5, 1, D, generator=g) * torch.exp2(torch.randint(-6, 7, (2, T + 5, 1, 1), generator=g).float())).half().cuda()
    table = torch.full((2, pages), -1, dtype=i32)
    order = torch.randperm(pages, generator=g).to(i32)
    table[0, :1], table[1, :pages - 2] = order[:1], order[1:pages - 1]
    table = table.cuda()

    def empty():
        return [torch.zeros(pages, page, 1, D, dtype=E4M3, device="cuda") for _ in range(2)] + \
               [torch.zeros(pages, page // block, 1, device="cuda") for _ in range(2)]

    def lengths(*n):
        return torch.tensor(n, dtype=i32, device="cuda")
    whole, parts = empty(), empty()
    ops.append_kv_8bit(*whole, x[0], x[1], table, lengths(0, 0), cu_new=lengths(0, 5, T + 5))
    ops.append_kv_8bit(*parts, x[0, :5], x[1, :5], table, lengths(0, 0), cu_new=lengths(0, 5, 5))
    for at in range(0, T, step):
        n = min(step, T - at)
        part = x[:, 5 + at:5 + at + n]
        ops.append_kv_8bit(*parts, part[0], part[1], table, lengths(5, at), cu_new=lengths(0, 0, n))
    for a, b in zip(whole, parts):
        assert torch.equal(bits(a), bits(b))
    # and a sample of the blocks are the oracle's
    some = [0, 1, 137 * 64 // block, T // block - 1]
    for blk in some:
        rows = x[:, 5 + blk * block:5 + (blk + 1) * block].cpu()
        k, v, ks, vs = [torch.zeros(1, block, 1, D).to(E4M3) for _ in range(2)] + [torch.zeros(1, 1, 1) for _ in range(2)]
        want = orc.append(k, v, ks, vs, rows[0], rows[1], torch.zeros(1, 1, dtype=i32), torch.zeros(1, dtype=i32), [block])
        pg, off = int(table[1, blk * block // page]), blk * block % page
        got = [whole[0][pg:pg + 1, off:off + block], whole[1][pg:pg + 1, off:off + block],
               whole[2][pg:pg + 1, off // block:off // block + 1], whole[3][pg:pg + 1, off // block:off // block + 1]]
        equal_cache(got, want)


@pytest.mark.parametrize("cdt", [E4M3, I8])
def test_a_thousand_ragged_sequences(cdt):
    lens = [random.Random(58 + i).choice([0, 1, 2, 15, 16, 17, 40, 129, 300]) for i in range(1100)]
    table, pages = rows_of(59, lens, 16)
    n = torch.tensor(lens, dtype=i32)
    pools = cache(60, pages, 16, 16, 2, 64, cdt)
    spoil(pools, table, n)
    q = torch.randn(len(lens), 2, 4, 64, generator=torch.Generator().manual_seed(61)).to(torch.bfloat16)
    check(attend(q, pools, table, n), q, pools, table, n)


def test_drafts_do_not_see_what_comes_after_them():
    """NaN and the largest numbers in the last drafted token reach its own query only."""
    lens = torch.tensor([200, 64, 5], dtype=i32)
    table, pages = rows_of(62, lens.tolist(), 16)
    pools = cache(63, pages, 16, 16, 2, 128, E4M3)
    q = torch.randn(3, 5, 10, 128, generator=torch.Generator().manual_seed(64)).half()
    before = attend(q, pools, table, lens).cpu()
    for b, n in enumerate(lens.tolist()):
        page, at = int(table[b, (n - 1) // 16]), (n - 1) % 16
        pools[0].view(torch.uint8)[page, at], pools[1].view(torch.uint8)[page, at] = 0x7f, 0x7f
    after = attend(q, pools, table, lens).cpu()
    assert torch.equal(after[:, :4], before[:, :4]) and after[:, 4].isnan().all()
    q[:, 1] = math.nan                       # a query's NaN stays its own as well
    odd = attend(q, pools, table, lens).cpu()
    assert odd[:, 1].isnan().all()
    assert torch.equal(odd[:, [0, 2, 3]], before[:, [0, 2, 3]])


def test_calls_on_two_streams_at_once():
    """Appends, attention and hand-outs of two caches, issued in turn on two streams."""
    from tritonops_b200 import ops
    lens = torch.tensor([700, 1300, 90], dtype=i32)
    jobs = []
    for i in (65, 66):
        table, pages = rows_of(i, [n + 40 for n in lens.tolist()], 32)
        g = torch.Generator().manual_seed(i)
        pools = cache(i, pages, 32, 32, 2, 128, I8)
        nk, nv = torch.randn(2, 3, 2, 128, generator=g).half()
        q = torch.randn(3, 16, 128, generator=g).half()
        refs = torch.randint(0, 2, (30000,), generator=g).to(i32)
        want = orc.append(*pools, nk, nv, table, lens, [1] * 3)
        jobs.append(dict(dev=[p.cuda() for p in pools], nk=nk.cuda(), nv=nv.cuda(), q=q, qd=q.cuda(), t=table.cuda(),
                         table=table, want=want, refs=refs, refs_d=refs.cuda(), s=torch.cuda.Stream()))
    n, one = lens.cuda(), torch.ones(3, dtype=i32, device="cuda")
    empty = torch.full((3, 200), -1, dtype=i32)
    ed, new = empty.cuda(), torch.tensor([1000, 50, 3000], dtype=i32)
    newd, zero = new.cuda(), torch.zeros(3, dtype=i32, device="cuda")
    torch.cuda.synchronize()
    for _ in range(3):
        for j in jobs:
            with torch.cuda.stream(j["s"]):
                ops.append_kv_8bit(*j["dev"], j["nk"], j["nv"], j["t"], n)
                j["o"] = ops.paged_decode_8bit(j["qd"], *j["dev"], j["t"], n + one)
                j["g"] = ops.grow_pages(ed, zero, j["refs_d"], newd, page_size=16)
    torch.cuda.synchronize()
    for j in jobs:
        equal_cache(j["dev"], j["want"])
        check(j["o"], j["q"], j["want"], j["table"], lens + 1)
        for a, b in zip(j["g"], orc.grow(empty, torch.zeros(3, dtype=i32), j["refs"], new, 16)):
            assert torch.equal(a.cpu().flatten(), b.flatten())


def test_expanded_pools_are_refused():
    from tritonops_b200 import ops
    k, v, ks, vs = [p.cuda() for p in cache(67, 4, 16, 16, 2, 64, I8)]
    t, n = torch.zeros(1, 2, dtype=i32, device="cuda"), torch.ones(1, dtype=i32, device="cuda")
    row = torch.zeros(1, 2, 64, dtype=torch.float16, device="cuda")
    q = torch.zeros(1, 4, 64, dtype=torch.float16, device="cuda")
    wide = k[:1].expand(4, -1, -1, -1)
    for call in (lambda: ops.append_kv_8bit(wide, v, ks, vs, row, row, t, n),
                 lambda: ops.append_kv_8bit(k, v, ks[:, :, :1].expand(-1, -1, 2), vs, row, row, t, n),
                 lambda: ops.paged_decode_8bit(q, wide, v, ks, vs, t, n)):
        with pytest.raises((ValueError, RuntimeError), match="STRIDE|stride"):
            call()


@pytest.mark.parametrize("chunk", [2 ** 31 - 128, 2 ** 30])
def test_one_chunk_of_any_size(chunk):
    lens = torch.tensor([700, 3], dtype=i32)
    table, pages = rows_of(68, lens.tolist(), 64)
    pools = cache(69, pages, 64, 64, 1, 64, E4M3)
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(70)).half()
    check(attend(q, pools, table, lens, chunk=chunk), q, pools, table, lens)


def test_counts_that_do_not_ascend_store_nothing_elsewhere():
    """cu_new that names rows again and again: pages of other rows of the table stay as they are."""
    D, heads, page, block = 32, 1, 16, 16
    S, T = 64, 4096
    pages = S + 4
    pools = cache(71, pages, page, block, heads, D, I8)
    table = torch.full((S, 1), -1, dtype=i32)
    table[:S // 2, 0] = torch.arange(S // 2, dtype=i32)
    cu = torch.tensor([0, T] * (S // 2) + [0], dtype=i32)
    nk, nv = torch.randn(2, T, heads, D, generator=torch.Generator().manual_seed(72)).half()
    dev = append(pools, nk, nv, table, torch.zeros(S, dtype=i32), cu)
    for a, b in zip(dev, pools):
        assert same_bits(a[S // 2:], b[S // 2:])
