"""The operators of a paged key/value cache held in 8 bits, as cases that can be timed and compared:
attention over the cache, the append that quantises into it, and the hand-out, forking and
compaction of its pages.

`run` computes them in plain torch; with `own` it makes the library's calls instead.  Lengths, page
tables and parents, which shape the work, come from the case itself (its `lens_seed`), tensors from
the seed given to `prepare`.

The cache.  Pools [pages, page, Hkv, D] hold e4m3 or int8 numbers, and a scale (fp32) stands for
each block of `block` tokens of a page and each head: [pages, page // block, Hkv].  A row of the
page table lists the pages of one sequence (slot), -1 where it holds none, and `refs` counts the
rows that hold a page, 0 for a free one."""
import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
CACHE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def listed():
    return [
        # One user's token against a short cache: what a call costs.
        dict(name="attend_small", kind="attend", batch=1, n=1, hq=8, hkv=2, d=64, page=16, block=16, lo=333, hi=333,
             lens_seed=1, dtype="fp16", cache="e4m3"),
        # A decoding step of a full serving batch, lengths as they come.
        dict(name="attend_batch", kind="attend", batch=64, n=1, hq=32, hkv=8, d=128, page=64, block=64, lo=1024,
             hi=8192, lens_seed=2, dtype="bf16", cache="e4m3"),
        # A few very long contexts, fine scales.
        dict(name="attend_long", kind="attend", batch=4, n=1, hq=32, hkv=8, d=128, page=64, block=16, lo=90001,
             hi=131072, lens_seed=3, dtype="bf16", cache="int8"),
        # Five drafted tokens for each sequence checked in one pass, small pages.
        dict(name="attend_drafts", kind="attend", batch=24, n=5, hq=32, hkv=8, d=128, page=16, block=16, lo=300,
             hi=6000, lens_seed=4, dtype="fp16", cache="int8"),
        # The step before attend_batch: one new token for each of 256 sequences.
        dict(name="append_step", kind="append", batch=256, new_lo=1, new_hi=1, lo=0, hi=1000, hkv=8, d=128, page=64,
             block=16, lens_seed=5, dtype="bf16", cache="e4m3"),
        # Prompts, and the later parts of prompts, stored in one call.
        dict(name="append_prompts", kind="append", batch=6, new_lo=37, new_hi=5000, lo=0, hi=700, hkv=8, d=128,
             page=64, block=64, lens_seed=6, dtype="fp16", cache="int8"),
        # One sequence forked into four beams, a small 16-bit cache.
        dict(name="fork_small", kind="fork", groups=1, beams=4, free=0.0, lo=400, hi=500, layers=2, hkv=4, d=64, page=32,
             block=0, spare=0.1, lens_seed=7, dtype="bf16", cache="bf16"),
        # A step of beam search over a batch, some sequences finished: rows shared, copied and freed.
        dict(name="fork_beams", kind="fork", groups=64, beams=4, free=0.1, lo=100, hi=1500, layers=4, hkv=8, d=128,
             page=64, block=64, spare=0.2, lens_seed=8, dtype="bf16", cache="e4m3"),
        # A handful of pages moved together in a small cache.
        dict(name="compact_small", kind="compact", slots=8, lo=50, hi=200, live=0.6, layers=1, hkv=2, d=64, page=16,
             block=0, lens_seed=9, dtype="fp16", cache="fp16"),
        # A pool half of whose sequences have ended, made dense again.
        dict(name="compact_pool", kind="compact", slots=256, lo=500, hi=2500, live=0.5, layers=2, hkv=8, d=128, page=64,
             block=16, lens_seed=10, dtype="bf16", cache="int8"),
        # Pages for the next token of a small batch.
        dict(name="grow_small", kind="grow", slots=8, lo=1, hi=1000, new_lo=1, new_hi=1, page=16, spare=0.2,
             lens_seed=11),
        # Pages for the coming prompts and tokens of a large server with small pages.
        dict(name="grow_server", kind="grow", slots=1024, lo=0, hi=8000, new_lo=0, new_hi=600, page=16, spare=0.3,
             lens_seed=12),
    ]


# ---------------------------------------------------------------------------- drawing
def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_HEADS = [(8, 8), (16, 4), (32, 8), (12, 12), (32, 32), (16, 1), (28, 4), (64, 8)]


def draw(rng):
    """A case of the ranges `listed` stands for; none costs more than the largest listed one."""
    most = max(work(c)["bytes"] for c in listed())
    for _ in range(500):
        c = _draw(rng)
        if work(c)["bytes"] <= most and _held(c) <= 6e9:
            return c
    return dict(kind="grow", slots=_log_int(rng, 1, 1024), lo=0, hi=_log_int(rng, 16, 8000), new_lo=0, new_hi=64,
                page=16, spare=0.3, lens_seed=rng.randrange(1 << 20))


def _draw(rng):
    kind = rng.choice(["attend"] * 4 + ["append"] * 3 + ["fork"] * 2 + ["compact"] * 2 + ["grow"])
    hq, hkv = rng.choice(_HEADS)
    page = rng.choice([16, 32, 48, 64, 128])
    block = rng.choice([b for b in (16, 32, 64, 128) if page % b == 0])
    c = dict(kind=kind, hkv=hkv, d=rng.choice([32, 64, 96, 128, 128]), page=page, block=block,
             dtype=rng.choice(["bf16", "fp16"]), cache=rng.choice(["e4m3", "int8"]), lens_seed=rng.randrange(1 << 20))
    if kind == "attend":
        hi = _log_int(rng, 8, 131072)
        c.update(hq=hq, batch=_log_int(rng, 1, 128), n=rng.choice([1, 1, 1, 1, 2, 3, 4, 7]),
                 lo=max(1, hi // rng.choice([1, 2, 8])), hi=hi)
    elif kind == "append":
        new = rng.choice([1, 1, 4, _log_int(rng, 8, 8192)])
        hi = _log_int(rng, 1, 4000)
        c.update(batch=_log_int(rng, 1, 256), new_lo=max(1, new // rng.choice([1, 2, 16])), new_hi=new,
                 lo=rng.choice([0, hi // 2]), hi=hi)
    elif kind == "fork":
        hi = _log_int(rng, 16, 4000)
        c.update(groups=_log_int(rng, 1, 64), beams=rng.choice([2, 2, 4, 5]), free=rng.choice([0.0, 0.1, 0.5]),
                 lo=max(1, hi // rng.choice([1, 2, 8])), hi=hi, layers=rng.randint(1, 6), spare=rng.choice([0.05, 0.3]))
    elif kind == "compact":
        hi = _log_int(rng, 16, 4000)
        c.update(slots=_log_int(rng, 1, 512), lo=max(1, hi // rng.choice([1, 2, 8])), hi=hi,
                 live=round(rng.uniform(0.2, 0.95), 2), layers=rng.randint(1, 6))
    else:
        hi = _log_int(rng, 16, 32768)
        c = dict(kind=kind, slots=_log_int(rng, 1, 1024), lo=rng.choice([0, hi // 2]), hi=hi, new_lo=rng.choice([0, 1]),
                 new_hi=_log_int(rng, 1, 2000), page=page, spare=rng.choice([0.0, 0.05, 0.5]),
                 lens_seed=c["lens_seed"])
    if kind in ("fork", "compact") and rng.random() < 0.3:     # the page operators serve 16-bit pools as well
        c.update(cache=c["dtype"], block=0)
    return c


def _held(c):
    """Bytes of the pools of a case."""
    if c["kind"] == "grow":
        return 0.0
    each = c["page"] * c["hkv"] * c["d"] * 2.0 * c.get("layers", 1) * (1 if c["cache"] in CACHE else 2)
    return each * _shape(c)["pages"]


# ---------------------------------------------------------------------------- the shape of the work
def _pages(n, page):
    return -(-n // page)


def _shape(c):
    """Lengths, page rows and so on of a case, as Python lists: the same for every seed."""
    r = random.Random(c["lens_seed"])
    kind, page = c["kind"], c["page"]
    s = {}
    if kind == "attend":
        s["lens"] = [r.randint(c["lo"], c["hi"]) for _ in range(c["batch"])]
        s["used"] = [_pages(n, page) for n in s["lens"]]
        s["pages"] = sum(s["used"])
    elif kind == "append":
        s["lens"] = [r.randint(c["lo"], c["hi"]) for _ in range(c["batch"])]
        s["new"] = [r.randint(c["new_lo"], c["new_hi"]) for _ in range(c["batch"])]
        s["used"] = [_pages(n + m, page) for n, m in zip(s["lens"], s["new"])]
        s["pages"] = sum(s["used"])
    elif kind == "fork":
        slots = c["groups"] * c["beams"]
        s["lens"] = [r.randint(c["lo"], c["hi"]) for _ in range(c["groups"]) for _ in range(c["beams"])]
        s["used"] = [_pages(n, page) for n in s["lens"]]
        gone = [r.random() < c["free"] for _ in range(c["groups"])]
        s["parents"] = [-1 if gone[b // c["beams"]] else b - b % c["beams"] + r.randrange(c["beams"])
                        for b in range(slots)]
        s["pages"] = sum(s["used"]) + int(c["spare"] * sum(s["used"])) + 1
    elif kind == "compact":
        s["lens"] = [r.randint(c["lo"], c["hi"]) for _ in range(c["slots"])]
        s["used"] = [_pages(n, page) for n in s["lens"]]
        s["pages"] = max(sum(s["used"]), int(sum(s["used"]) / c["live"]))
    else:
        s["lens"] = [r.randint(c["lo"], c["hi"]) for _ in range(c["slots"])]
        s["new"] = [r.randint(c["new_lo"], c["new_hi"]) for _ in range(c["slots"])]
        s["used"] = [_pages(n, page) for n in s["lens"]]
        s["pages"] = sum(s["used"]) + int(c["spare"] * sum(s["used"])) + 1
    s["order"] = random.Random(c["lens_seed"] + 1).sample(range(s["pages"]), sum(s["used"]))
    s["width"] = max(1, max(s["used"]))
    if kind == "fork":
        s["width"] += 1
    if kind == "grow":
        s["width"] = max(1, max(_pages(n + m, page) for n, m in zip(s["lens"], s["new"])))
    return s


def _rows(s):
    rows, at = [], 0
    for n in s["used"]:
        rows.append(s["order"][at:at + n] + [-1] * (s["width"] - n))
        at += n
    return rows


# ---------------------------------------------------------------------------- preparing
def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _pool(g, c, pages):
    """A pool whose numbers fill the range of their type as quantised rows do."""
    shape = (pages, c["page"], c["hkv"], c["d"])
    x = torch.empty(shape, device="cuda", dtype=torch.float16).normal_(generator=g)
    if c["cache"] == "e4m3":
        return (x * 90).clamp_(-448, 448).to(torch.float8_e4m3fn)
    if c["cache"] == "int8":
        return (x * 28).clamp_(-127, 127).to(torch.int8)
    return x.to(DTYPES[c["cache"]])


def _scale(g, c, pages):
    """Powers of two, as the append leaves them, for rows of standard deviation about one."""
    shape = (pages, c["page"] // c["block"], c["hkv"])
    up = torch.randint(-1, 2, shape, generator=g, device="cuda").float()
    return torch.exp2(up - (6 if c["cache"] == "e4m3" else 5))


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = _shape(c)
    s = {"case": dict(c), "lens": _ints(shape["lens"]), "pages": shape["pages"]}
    rows = _rows(shape)
    if c["kind"] in ("fork", "compact", "grow"):
        # the same rows over other pages for another seed
        perm = torch.randperm(shape["pages"], generator=g, device="cuda").int()
        table = _ints(rows)
        s["table"] = torch.where(table >= 0, perm[table.clamp(min=0).long()], -1).contiguous()
        s["refs"] = torch.zeros(shape["pages"] + 1, dtype=torch.int32, device="cuda")
        s["refs"].index_add_(0, torch.where(s["table"] >= 0, s["table"], shape["pages"]).flatten(),
                             torch.ones(s["table"].numel(), dtype=torch.int32, device="cuda"))
        s["refs"] = s["refs"][:-1].clone()
    else:
        s["table"] = _ints(rows)
    if c["kind"] == "grow":
        s["new"] = _ints(shape["new"])
        return s
    if c["kind"] in ("fork", "compact"):
        pools = []
        for _ in range(c["layers"]):
            pools += [_pool(g, c, shape["pages"]), _pool(g, c, shape["pages"])]
            if c["block"]:
                pools += [_scale(g, c, shape["pages"]), _scale(g, c, shape["pages"])]
        s["pools"] = pools
        if c["kind"] == "fork":
            s["parents"] = _ints(shape["parents"])
        return s
    s["k"], s["v"] = _pool(g, c, shape["pages"]), _pool(g, c, shape["pages"])
    s["ks"], s["vs"] = _scale(g, c, shape["pages"]), _scale(g, c, shape["pages"])
    dt = DTYPES[c["dtype"]]
    if c["kind"] == "attend":
        lead = (c["batch"],) if c["n"] == 1 else (c["batch"], c["n"])
        s["q"] = torch.randn(*lead, c["hq"], c["d"], generator=g, device="cuda").to(dt)
        s["max"] = max(shape["lens"])
        return s
    new = shape["new"]
    total = sum(new)
    s["new_k"], s["new_v"] = (torch.randn(total, c["hkv"], c["d"], generator=g, device="cuda").to(dt) for _ in range(2))
    s["one"] = c["new_lo"] == c["new_hi"] == 1
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    s["cu"] = _ints(cu)
    s["blocks"] = max(_pages(n + m, c["block"]) - n // c["block"] for n, m in zip(shape["lens"], new))
    return s


# ---------------------------------------------------------------------------- one pass
def run(state):
    s = state
    kind = s["case"]["kind"]
    if own:
        return _run_own(s, kind)
    return {"attend": _attend, "append": _append, "fork": _fork, "compact": _compact, "grow": _grow}[kind](s)


def _run_own(s, kind):
    from tritonops_b200 import ops
    c = s["case"]
    if kind == "attend":
        return ops.paged_decode_8bit(s["q"], s["k"], s["v"], s["ks"], s["vs"], s["table"], s["lens"],
                                     max_seqlen=s["max"])
    if kind == "append":
        ops.append_kv_8bit(s["k"], s["v"], s["ks"], s["vs"], s["new_k"], s["new_v"], s["table"], s["lens"],
                           cu_new=None if s["one"] else s["cu"])
        return s["k"], s["v"], s["ks"], s["vs"]
    if kind == "fork":
        return (*ops.fork_pages(s["pools"], s["table"], s["lens"], s["refs"], s["parents"], page_size=c["page"]),
                s["pools"])
    if kind == "compact":
        return (*ops.compact_pages(s["pools"], s["table"], s["refs"]), s["pools"])
    return ops.grow_pages(s["table"], s["lens"], s["refs"], s["new"], page_size=c["page"])


def _bytes(t):
    """8-bit pools are moved as bytes."""
    return t.view(torch.uint8) if t.element_size() == 1 else t


def _attend(s):
    c = s["case"]
    b, n, g = c["batch"], c["n"], c["hq"] // c["hkv"]
    at = s["table"].clamp(min=0).long()

    def rows(pool, scale):      # [B, Hkv, keys, D] in 32 bits
        x = _bytes(pool)[at].view(pool.dtype).float()
        x = x.unflatten(2, (-1, c["block"])) * scale[at][..., None, :, None]
        return x.flatten(1, 3).transpose(1, 2)

    q = s["q"].reshape(b, n, c["hkv"], g, c["d"]).float().permute(0, 2, 1, 3, 4).flatten(2, 3)
    scores = q @ rows(s["k"], s["ks"]).transpose(-1, -2) * c["d"] ** -0.5      # [B, Hkv, n * G, keys]
    t = torch.arange(scores.shape[-1], device="cuda")
    i = torch.arange(n, device="cuda").repeat_interleave(g)
    seen = t < (s["lens"][:, None] - n + 1 + i)[:, None, :, None]
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    v = rows(s["v"], s["vs"]).masked_fill((t >= s["lens"][:, None])[:, None, :, None], 0.0)
    o = p @ v / total.clamp(min=1e-30)
    return o.unflatten(2, (n, g)).permute(0, 2, 1, 3, 4).reshape(s["q"].shape).to(s["q"].dtype)


def _need(top, cache):
    """The smallest power of two s with top <= s * (largest number of the type): 0 for 0, NaN for a
    top that is not finite."""
    m, e = torch.frexp(torch.where(torch.isfinite(top), top, 1.0))
    e = e - torch.where(m <= (0.875 if cache == "e4m3" else 0.9921875), 0, -1)
    e = (e - (9 if cache == "e4m3" else 7)).clamp(min=-126)
    scale = ((e + 127).to(torch.int32) << 23).view(torch.float32)
    scale = torch.where(top == 0, 0.0, scale)
    return torch.where(torch.isfinite(top), scale, math.nan)


def _quantise(x, cache):
    return x.to(torch.float8_e4m3fn) if cache == "e4m3" else torch.round(x).to(torch.int8)


def _append(s):
    c = s["case"]
    bt, per = c["block"], c["page"] // c["block"]
    start, new = s["lens"].long(), (s["cu"][1:] - s["cu"][:-1]).long()
    blk = start[:, None] // bt + torch.arange(s["blocks"], device="cuda")            # [B, blocks]
    touched = blk * bt < (start + new)[:, None]
    page = s["table"].long().gather(1, (blk // per).clamp(max=s["table"].shape[1] - 1))
    at = (page * per + blk % per)[touched]                                           # blocks of the pool
    pos = blk[..., None] * bt + torch.arange(bt, device="cuda")                      # [B, blocks, bt]
    is_old = (pos < start[:, None, None])[touched][..., None, None]
    is_new = ((pos >= start[:, None, None]) & (pos < (start + new)[:, None, None]))[touched][..., None, None]
    src = (s["cu"][:-1].long()[:, None, None] + pos - start[:, None, None])[touched].clamp(0, s["new_k"].shape[0] - 1)

    def store(pool, scale, rows):
        flat = _bytes(pool).view(-1, bt, c["hkv"], c["d"])
        held = flat[at]                                                              # [blocks, bt, H, D]
        x = rows[src].float()
        need = _need(torch.where(is_new, x, 0.0).abs().amax((1, 3)), c["cache"])     # [blocks, H]
        before = torch.where(is_old.any(1)[..., 0], scale.view(-1, c["hkv"])[at], 0.0)
        after = torch.where(torch.isnan(before) | torch.isnan(need), math.nan, torch.maximum(before, need))
        one = torch.where(after > 0, after, 1.0)[:, None, :, None]
        fresh = torch.where((after > 0)[:, None, :, None], x / one, 0.0)
        kept = held.view(pool.dtype).float() * (before[:, None, :, None] / one)
        moved = is_old & (after > before)[:, None, :, None]
        q = _quantise(torch.where(is_new, fresh, torch.where(moved, kept, 0.0)), c["cache"])
        flat[at] = torch.where(is_new | moved, q.view(torch.uint8), held)
        scale.view(-1, c["hkv"])[at] = after

    store(s["k"], s["ks"], s["new_k"])
    store(s["v"], s["vs"], s["new_v"])
    return s["k"], s["v"], s["ks"], s["vs"]


def _free_pages(refs):
    """The free pages in ascending order, in the first places of a list as long as the pool (the rest -1)."""
    free = refs <= 0
    place = torch.where(free, free.cumsum(0) - 1, refs.numel())
    out = torch.full((refs.numel() + 1,), -1, dtype=torch.int32, device=refs.device)
    return out.scatter_(0, place, torch.arange(refs.numel(), dtype=torch.int32, device=refs.device))[:-1]


def _hand_out(refs, wanted):
    """The lowest free pages for the true places of `wanted`, in order: (pages, -1 elsewhere; refs; how many
    places got none)."""
    free = _free_pages(refs)
    rank = (wanted.flatten().cumsum(0) - 1).view(wanted.shape)
    got = torch.where(wanted & (rank < free.numel()), free[rank.clamp(0, free.numel() - 1)], -1)
    refs = torch.cat([refs, refs.new_zeros(1)]).scatter_(0, torch.where(got >= 0, got, refs.numel()).long().flatten(), 1)
    return got, refs[:-1].clone(), (wanted & (got < 0)).sum(dtype=torch.int32).view(1)


def _count(table, pages):
    """How many of the entries of `table` name each page."""
    out = torch.zeros(pages + 1, dtype=torch.int32, device=table.device)
    at = torch.where((table >= 0) & (table < pages), table, pages).flatten()
    return out.index_add_(0, at, torch.ones_like(at))[:-1]


def _move(pool, src, dst):
    flat = _bytes(pool)
    flat[dst] = flat[src]


def _fork(s):
    c, table, parents, pages = s["case"], s["table"], s["parents"].long(), s["pages"]
    slots, page = table.shape[0], c["page"]
    here = torch.arange(slots, device="cuda")
    ok = (parents >= 0) & (parents < slots)
    p = torch.where(ok, parents, 0)
    stays = ok & (parents == here)
    lens = torch.where(ok, s["lens"][p].clamp(0, table.shape[1] * page), 0)
    # who has the row whole: its own slot, else the lowest one that takes it
    first = torch.full((slots + 1,), slots, device="cuda").scatter_reduce_(
        0, torch.where(ok, p, slots), torch.where(stays, -1, here), "amin")[:-1]
    keeps = ok & ((first[p] == here) | stays)
    rows = torch.where(ok[:, None], table[p], -1)
    rows = torch.where((rows >= 0) & (rows < pages), rows, -1)
    i, full = torch.arange(table.shape[1], device="cuda"), (lens // page)[:, None]
    last = (i == full) & (lens % page != 0)[:, None] & (rows >= 0) & ~keeps[:, None]
    shared = torch.where(keeps[:, None] | (i < full), rows, -1)
    refs = s["refs"] - _count(torch.where(stays[:, None], -1, table), pages) \
        + _count(torch.where(stays[:, None], -1, shared), pages)
    got, refs, missing = _hand_out(refs, last)
    new = torch.where(last, got, shared).int()
    lens = torch.where((last & (got < 0)).any(1), lens // page * page, lens).int()
    done = last & (got >= 0)
    src, dst = rows[done].long(), got[done].long()
    [_move(pool, src, dst) for pool in s["pools"]]
    return new, lens, refs, missing, s["pools"]


def _compact(s):
    table, refs, pages = s["table"], s["refs"], s["pages"]
    live = refs > 0
    n = live.sum()
    at = torch.arange(pages, device="cuda")
    dst, src = at[~live & (at < n)], at[live & (at >= n)]
    to = torch.where(live, at, -1).scatter_(0, src, dst)
    new = torch.where((table >= 0) & (table < pages), to[table.clamp(0, pages - 1).long()], -1).int()
    counts = torch.where(live, refs, 0)
    counts[dst] = counts[src]
    counts = torch.where(at < n, counts, 0)
    [_move(pool, src, dst) for pool in s["pools"]]
    return new, counts, n.int().view(1), s["pools"]


def _grow(s):
    c, table = s["case"], s["table"]
    width = table.shape[1]
    tokens = s["lens"].clamp(min=0).long() + s["new"].clamp(min=0)
    want = (tokens + c["page"] - 1) // c["page"]
    held = (table >= 0) & (table < s["pages"])
    wanted = (torch.arange(width, device="cuda") < want[:, None]) & ~held
    got, refs, missing = _hand_out(s["refs"], wanted)
    over = (want - width).clamp(min=0).sum(dtype=torch.int32)
    return torch.where(held, table, got).int(), refs, missing + over


# ---------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    s = _shape(c)
    if c["kind"] == "attend":
        keys = sum(s["lens"])
        blocks = sum(_pages(n, c["block"]) for n in s["lens"])
        return {"bytes": 2.0 * keys * c["hkv"] * c["d"] + 8.0 * blocks * c["hkv"]
                + 4.0 * c["batch"] * c["n"] * c["hq"] * c["d"] + 4.0 * sum(s["used"]),
                "flops": 4.0 * c["d"] * c["hq"] * c["n"] * keys}
    if c["kind"] == "append":
        t = sum(s["new"])
        blocks = sum(_pages(n + m, c["block"]) - n // c["block"] for n, m in zip(s["lens"], s["new"]))
        return {"bytes": 6.0 * t * c["hkv"] * c["d"] + 8.0 * blocks * c["hkv"] + 4.0 * sum(s["used"]),
                "flops": 6.0 * t * c["hkv"] * c["d"]}
    books = 8.0 * len(s["lens"]) * s["width"] + 8.0 * s["pages"]
    if c["kind"] == "grow":
        return {"bytes": books + 8.0 * len(s["lens"]), "flops": 0.0}
    each = c["layers"] * 2.0 * (c["page"] * c["hkv"] * c["d"] * (1 if c["cache"] in CACHE else 2)
                                + (4 * (c["page"] // c["block"]) * c["hkv"] if c["block"] else 0))
    if c["kind"] == "fork":
        kept = set(b for b, p in enumerate(s["parents"]) if p == b)
        copies = 0
        for b, p in enumerate(s["parents"]):
            if p >= 0 and p != b:
                copies += p in kept and s["lens"][p] % c["page"] != 0
                kept.add(p)
        return {"bytes": books + 12.0 * len(s["lens"]) + 2.0 * each * copies, "flops": 0.0}
    live = sum(s["used"])
    return {"bytes": books + 2.0 * each * live * (s["pages"] - live) / s["pages"], "flops": 0.0}


# ---------------------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    """What `run(prepare(case, seed))` returns, a sequence at a time in 64 bits; the whole numbers of the page
    operators and of int8 pools have no such value."""
    c = case
    s = prepare(c, seed)
    shape = _shape(c)
    if c["kind"] == "attend":
        return _exact_attend(c, s, shape)
    if c["kind"] == "append":
        return _exact_append(c, s, shape)
    if c["kind"] == "grow" or c["cache"] == "int8":
        return None
    return _exact_pages(c, s, shape)


def _sequence(c, shape, b, *pools):
    """The rows of sequence b in each of `pools` (with their scales where they are pairs), in 64 bits."""
    n = shape["lens"][b]
    at = sum(shape["used"][:b])
    pages = torch.tensor(shape["order"][at:at + shape["used"][b]], device="cuda")
    out = []
    for pool, scale in pools:
        x = _bytes(pool)[pages].view(pool.dtype).double().flatten(0, 1)[:n]
        out.append(x * scale[pages].double().flatten(0, 1).repeat_interleave(c["block"], 0)[:n, :, None])
    return out


def _exact_attend(c, s, shape):
    n, g = c["n"], c["hq"] // c["hkv"]
    q = s["q"].view(c["batch"], n, c["hq"], c["d"]).double()
    o = torch.zeros_like(q)
    for b, length in enumerate(shape["lens"]):
        k, v = _sequence(c, shape, b, (s["k"], s["ks"]), (s["v"], s["vs"]))
        for i in range(n):
            m = length - n + 1 + i
            if m <= 0:
                continue
            x = torch.einsum("hgd,thd->hgt", q[b, i].view(c["hkv"], g, c["d"]), k[:m]) / math.sqrt(c["d"])
            o[b, i] = torch.einsum("hgt,thd->hgd", torch.softmax(x, -1), v[:m]).reshape(c["hq"], c["d"])
    return o.view(s["q"].shape)


def _exact_append(c, s, shape):
    bt, per = c["block"], c["page"] // c["block"]
    most = 448.0 if c["cache"] == "e4m3" else 127.0
    out, at, t0 = [], 0, 0
    pools = [(s["k"].double(), s["ks"].double(), s["new_k"].double()),
             (s["v"].double(), s["vs"].double(), s["new_v"].double())]
    for b, (n, m) in enumerate(zip(shape["lens"], shape["new"])):
        pages = torch.tensor(shape["order"][at:at + shape["used"][b]], device="cuda")
        first, end = n // bt, _pages(n + m, bt)
        blocks = torch.arange(first, end, device="cuda")
        where = (pages[blocks // per], blocks % per)
        for pool, scale, rows in pools:
            view = pool.view(-1, per, bt, c["hkv"], c["d"])
            x = view[where]                                                          # [blocks, bt, H, D]
            span = torch.zeros(x.shape[0] * bt, c["hkv"], c["d"], dtype=torch.float64, device="cuda")
            lo = n - first * bt
            span[lo:lo + m] = rows[t0:t0 + m]
            top = span.view(x.shape).abs().amax((1, 3)).cpu()
            need = torch.tensor([[0.0 if v == 0 else 2.0 ** max(-126, math.ceil(math.log2(v / most))) for v in r]
                                 for r in top.tolist()], dtype=torch.float64, device="cuda")
            before = torch.zeros_like(need)
            if lo:
                before[0] = scale[where][0]
            after = torch.maximum(before, need)
            held = x.flatten(0, 1)
            fine = span / after.repeat_interleave(bt, 0).clamp(min=2.0 ** -126)[..., None]
            fine[:lo] = held[:lo] * (before[0] / after[0].clamp(min=2.0 ** -126))[:, None]
            fine = fine.to(torch.float8_e4m3fn).double() if c["cache"] == "e4m3" else fine.round()
            held[:lo + m] = fine[:lo + m]
            view[where] = held.view(x.shape)
            scale[where] = after
        at += shape["used"][b]
        t0 += m
    for pool, scale, _ in pools:
        out.append((pool if c["cache"] == "e4m3" else None, scale))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def _exact_pages(c, s, shape):
    """The pools after the moves that the lists of the case, taken one slot after another, ask for."""
    rows = s["table"].tolist()
    refs = s["refs"].tolist()
    moves = []
    if c["kind"] == "compact":
        n = sum(r > 0 for r in refs)
        moves = list(zip([p for p in range(n, len(refs)) if refs[p] > 0], [p for p in range(n) if refs[p] <= 0]))
    else:
        parents = shape["parents"]
        owner = {}
        for b, p in enumerate(parents):
            if p >= 0 and (p not in owner or p == b):
                owner[p] = b
        want = []
        for b, p in enumerate(parents):
            if p != b:
                for e in rows[b]:
                    if e >= 0:
                        refs[e] -= 1
        for b, p in enumerate(parents):
            if p < 0 or p == b:
                continue
            full, part = divmod(shape["lens"][p], c["page"])
            for i, e in enumerate(rows[p]):
                if e >= 0 and (owner[p] == b or i < full):
                    refs[e] += 1
            if owner[p] != b and part:
                want.append(rows[p][full])
        free = [p for p, r in enumerate(refs) if r <= 0]
        moves = list(zip(want, free))
    pools = [p.double() for p in s["pools"]]
    if moves:
        src, dst = torch.tensor(moves, device="cuda").T
        for p in pools:
            p[dst] = p[src]
    return (None, None, None, None, pools) if c["kind"] == "fork" else (None, None, None, pools)
