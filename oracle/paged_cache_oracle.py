"""CPU oracle of the paged 8-bit cache: attention over it, the append that quantises into it, and the
bookkeeping of its pages, in plain Python and float64, one sequence after another.

The reference has no such cache; attention over one is its decoding mathematics
(flash_attn_triton/flash_attn_decoding.py:62-122) on the numbers the cache stands for."""
import math

import torch

MOST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def sequence_rows(pool, scales, row, n):
    """(positions, float64 rows [positions, H, D]) of the first n keys of a page-table row; keys on
    pages outside the pool are left out."""
    pages, size = pool.shape[:2]
    block = size // scales.shape[1]
    pos, rows = [], []
    for t in range(n):
        page, r = int(row[t // size]), t % size
        if 0 <= page < pages:
            pos.append(t)
            rows.append(pool[page, r].double() * scales[page, r // block].double()[:, None])
    if not rows:
        return torch.zeros(0, dtype=torch.long), torch.zeros(0, *pool.shape[2:], dtype=torch.float64)
    return torch.tensor(pos), torch.stack(rows)


def attend(q, k, v, ks, vs, table, lens, max_seqlen=None, scale=None):
    """(o float64 like q, sum of softmax weight x |v| like q): q [B, n, Hq, D] on the CPU."""
    B, n, Hq, D = q.shape
    Hkv, group = k.shape[2], Hq // k.shape[2]
    cap = table.shape[1] * k.shape[1]
    if max_seqlen is not None:
        cap = min(cap, max_seqlen)
    scale = D ** -0.5 if scale is None else scale
    o, mass = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for b in range(B):
        length = min(max(int(lens[b]), 0), cap)
        at, kr = sequence_rows(k, ks, table[b], length)
        _, vr = sequence_rows(v, vs, table[b], length)
        for i in range(n):
            seen = at < length - n + 1 + i
            if not seen.any():
                continue
            qi = q[b, i].double().view(Hkv, group, D)
            w = torch.softmax(torch.einsum("hgd,thd->hgt", qi, kr[seen]) * scale, -1)
            o[b, i] = torch.einsum("hgt,thd->hgd", w, vr[seen]).reshape(Hq, D)
            mass[b, i] = torch.einsum("hgt,thd->hgd", w, vr[seen].abs()).reshape(Hq, D)
    return o, mass


def scale_for(top, dtype):
    """Smallest power of two s with top <= s * (largest number); 0 for 0, NaN for what is not finite."""
    if not math.isfinite(top):
        return math.nan
    if top == 0:
        return 0.0
    s = 2.0 ** -126
    while top > s * MOST[dtype]:
        s *= 2
    return s


def to_8bit(x, dtype):
    """float64 -> nearest number of the type to the fp32 quotient, ties to even."""
    return x.float().to(dtype) if dtype == torch.float8_e4m3fn else x.float().round().clamp(-127, 127).to(dtype)


def append(k, v, ks, vs, new_k, new_v, table, lens, counts):
    """The cache after appending counts[b] rows to each sequence: (k, v, ks, vs), new tensors."""
    out = [t.clone() for t in (k, v, ks, vs)]
    pages, size = k.shape[:2]
    block = size // ks.shape[1]
    t0 = 0
    for b, m in enumerate(counts):
        start = int(lens[b])
        if start >= 0:
            done = 0
            while done < m:
                pos = start + done
                off, here = pos % block, min(block - pos % block, m - done)
                if pos // size < table.shape[1]:
                    page, idx = int(table[b, pos // size]), pos % size // block
                    if 0 <= page < pages:
                        for pool, scales, rows in ((out[0], out[2], new_k), (out[1], out[3], new_v)):
                            _append_block(pool[page, idx * block:(idx + 1) * block], scales[page, idx], off,
                                          rows[t0 + done:t0 + done + here].double())
                done += here
        t0 += m
    return out


def _append_block(held, scales, off, rows):
    dt = held.dtype
    for h in range(held.shape[1]):
        need = scale_for(float(rows[:, h].abs().max()), dt)
        before = float(scales[h]) if off else 0.0
        after = math.nan if math.isnan(need) or math.isnan(before) else max(need, before)
        scales[h] = after
        x = rows[:, h] / after if after > 0 else torch.zeros_like(rows[:, h])
        held[off:off + rows.shape[0], h] = to_8bit(x, dt)
        if off and after > before:
            # (rounded to fp32 first, as the ratio and the product are where `before` is no power of two)
            ratio = torch.tensor(before, dtype=torch.float32) / torch.tensor(after, dtype=torch.float32)
            held[:off, h] = to_8bit((held[:off, h].float() * ratio).double(), dt)


def _pages_of(row, pages):
    return [int(e) if 0 <= int(e) < pages else -1 for e in row]


def grow(table, lens, refs, new, page_size):
    table, refs = table.clone(), refs.clone()
    S, P = table.shape
    free = [i for i, r in enumerate(refs.tolist()) if r <= 0]
    missing = 0
    for b in range(S):
        row = _pages_of(table[b], len(refs))
        want = -(-(max(int(lens[b]), 0) + max(int(new[b]), 0)) // page_size)
        missing += max(want - P, 0)
        for i in range(min(want, P)):
            if row[i] < 0:
                if free:
                    row[i] = free.pop(0)
                    refs[row[i]] = 1
                else:
                    missing += 1
        table[b] = torch.tensor(row, dtype=torch.int32)
    return table, refs, torch.tensor([missing], dtype=torch.int32)


def fork(pools, table, lens, refs, parents, page_size):
    """(table, lens, refs, missing, pools), new tensors."""
    S, P = table.shape
    N = len(refs)
    rows = [_pages_of(r, N) for r in table]
    parents = parents.tolist()
    keeper = {}
    for b, p in enumerate(parents):
        if 0 <= p < S and (p not in keeper or p == b):
            keeper[p] = b
    refs = refs.tolist()
    for b, p in enumerate(parents):
        if p != b:
            for e in rows[b]:
                if e >= 0:
                    refs[e] -= 1
    out, out_lens, wants = [], [], []
    for b, p in enumerate(parents):
        if not 0 <= p < S:
            out.append([-1] * P)
            out_lens.append(0)
            continue
        n = min(max(int(lens[p]), 0), P * page_size)
        full = n // page_size
        row = list(rows[p]) if keeper[p] == b else [e if i < full else -1 for i, e in enumerate(rows[p])]
        if p != b:
            for e in row:
                if e >= 0:
                    refs[e] += 1
        if keeper[p] != b and n % page_size and rows[p][full] >= 0:
            wants.append((b, full, rows[p][full]))
        out.append(row)
        out_lens.append(n)
    free = [i for i, r in enumerate(refs) if r <= 0]
    pools = [p.clone() for p in pools]
    before = [p.clone() for p in pools]
    missing = 0
    for b, full, src in wants:
        if free:
            dst = free.pop(0)
            out[b][full] = dst
            refs[dst] = 1
            for new, old in zip(pools, before):
                new[dst] = old[src]
        else:
            out_lens[b] = full * page_size
            missing += 1
    i32 = torch.int32
    return (torch.tensor(out, dtype=i32), torch.tensor(out_lens, dtype=i32), torch.tensor(refs, dtype=i32),
            torch.tensor([missing], dtype=i32), pools)


def compact(pools, table, refs):
    """(table, refs, live, pools), new tensors."""
    N = len(refs)
    refs = refs.tolist()
    n = sum(r > 0 for r in refs)
    holes = [i for i in range(n) if refs[i] <= 0]
    movers = [i for i in range(n, N) if refs[i] > 0]
    to = {i: i for i in range(N) if refs[i] > 0}
    to.update(zip(movers, holes))
    pools = [p.clone() for p in pools]
    out = [0] * N
    for src, dst in to.items():
        out[dst] = refs[src]
        if src != dst:
            for p in pools:
                p[dst] = p[src]
    new = [[to.get(int(e), -1) for e in row] for row in table]
    i32 = torch.int32
    return torch.tensor(new, dtype=i32), torch.tensor(out, dtype=i32), torch.tensor([n], dtype=i32), pools
