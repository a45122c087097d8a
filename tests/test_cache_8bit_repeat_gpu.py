"""Attention over the 8-bit cache is a pure function of its inputs: the same bits from every call, whoever takes over
which part of the work."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cdt", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("batch,n,page,lo,hi", [(1, 1, 16, 333, 333), (64, 1, 64, 1024, 8192), (2, 1, 64, 50000, 60000),
                                                (24, 5, 16, 300, 6000), (300, 3, 48, 1, 400)])
def test_same_bits_from_every_call(cdt, batch, n, page, lo, hi):
    from tritonops_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(1)
    lens = torch.randint(lo, hi + 1, (batch,), generator=g, device="cuda", dtype=torch.int32)
    width = -(-hi // page)
    pages = batch * width
    x = torch.empty(2, pages, page, 2, 128, device="cuda", dtype=torch.float16).normal_(generator=g) * 28
    k, v = x.to(cdt) if cdt != torch.int8 else x.clamp(-127, 127).to(cdt)
    s = torch.exp2(torch.randint(-7, -4, (2, pages, page // 16, 2), generator=g, device="cuda").float())
    table = torch.randperm(pages, generator=g, device="cuda").int().view(batch, width)
    q = torch.randn(batch, n, 8, 128, generator=g, device="cuda").bfloat16()
    first = ops.paged_decode_8bit(q, k, v, *s, table, lens)
    dirt = torch.empty(40 << 20, device="cuda")
    for i in range(8):
        dirt.fill_(float("nan"))       # (what a call finds in its scratch and in L2 is not what the last one left)
        assert torch.equal(ops.paged_decode_8bit(q, k, v, *s, table, lens), first)
