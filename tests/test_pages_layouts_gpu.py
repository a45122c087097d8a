"""Pools whose heads lie outside their tokens, as attention and append take them, in the page operators: as the
tensors whose pages are one block of memory each."""
import pytest
import torch

from oracle import paged_cache_oracle as orc

pytestmark = pytest.mark.gpu
i32 = torch.int32


@pytest.mark.parametrize("outermost", [False, True])
def test_heads_outside_tokens(outermost):
    from tritonops_b200 import ops
    pages, page, heads, D = 24, 16, 2, 32
    g = torch.Generator().manual_seed(1)
    held = torch.randint(-127, 128, (heads, pages, page, D) if outermost else (pages, heads, page, D), generator=g, dtype=torch.int8)
    dev = held.cuda()
    pool = dev.permute(1, 2, 0, 3) if outermost else dev.transpose(1, 2)         # [pages, page, heads, D]
    blocks = [pool[:, :, h] for h in range(heads)] if outermost else [dev]
    before = pool.cpu().clone()
    table = torch.tensor([[20, 3, -1], [7, -1, -1], [-1, -1, -1]], dtype=i32)
    lens, par = torch.tensor([20, 9, 0], dtype=i32), torch.tensor([0, 0, 1], dtype=i32)
    refs = torch.zeros(pages, dtype=i32)
    refs[[20, 3, 7]] = 1
    got = ops.fork_pages(blocks, table.cuda(), lens.cuda(), refs.cuda(), par.cuda(), page_size=page)
    want = orc.fork([before], table, lens, refs, par, page)
    for x, y in zip((*got, pool), (*want[:4], want[4][0])):
        assert torch.equal(x.cpu(), y)
    got2 = ops.compact_pages(blocks, got[0], got[2])
    want2 = orc.compact(want[4], want[0], want[2])
    for x, y in zip((*got2, pool), (*want2[:3], want2[3][0])):
        assert torch.equal(x.cpu(), y)
    # what attention reads through the new table is what it read before
    scale = torch.full((pages, 1, heads), 2.0 ** -5, device="cuda")
    q = torch.randn(3, heads, D, generator=g).cuda().half()
    o = ops.paged_decode_8bit(q, pool, pool, scale, scale, got2[0], got[1])
    old = before.cuda()
    rows = torch.tensor([[20, 3, -1], [20, 3, -1], [7, -1, -1]], dtype=i32, device="cuda")
    assert torch.equal(o, ops.paged_decode_8bit(q, old, old, scale, scale, rows, got[1]))
