"""Operands that the kernels cannot address as they lie (a base or a stride that is no multiple of 16 bytes) are
copied, those among them that torch calls contiguous as well."""
import pytest
import torch


def odd_base(*shape, **kw):
    n = torch.Size(shape).numel()
    return torch.randn(n + 8, **kw)[1:n + 1].view(shape)


def odd_stride(heads, dim, **kw):
    return torch.randn(1, heads * dim + 4, **kw)[:, :heads * dim].view(1, heads, dim)


def test_copies_are_addressable():
    from tritonops_b200 import ops
    h = dict(dtype=torch.float16)
    for t in (odd_base(3, 4, 64, **h), odd_stride(4, 64, **h), torch.randn(64, 4, **h).t(), torch.randn(2, 3, 65, **h)[:, :, :64]):
        c = ops._rowmajor16(t)
        assert torch.equal(c, t) and c.data_ptr() % 16 == 0 and c.stride(-1) == 1 and all(s % 8 == 0 for s in c.stride()[:-1])
    t = torch.randn(2, 4, 64, **h)[:, 1:3]
    assert ops._rowmajor16(t) is t


@pytest.mark.gpu
@pytest.mark.parametrize("make", [lambda n, h, d: odd_base(n, h, d, device="cuda", dtype=torch.float16),
                                  lambda n, h, d: odd_stride(h, d, device="cuda", dtype=torch.float16)])
def test_calls_take_them(make):
    from tritonops_b200 import ops
    i32 = torch.int32
    table, lens = torch.arange(4, dtype=i32, device="cuda").view(1, 4), torch.tensor([50], dtype=i32, device="cuda")
    pools = [[torch.zeros(4, 16, 2, 64, dtype=torch.int8, device="cuda") for _ in range(2)]
             + [torch.zeros(4, 1, 2, device="cuda") for _ in range(2)] for _ in range(2)]
    rows, q = make(1, 2, 64), make(1, 4, 64)
    for cache, new in zip(pools, (rows, rows.clone(memory_format=torch.contiguous_format))):
        for at in range(50):
            ops.append_kv_8bit(*cache, new, new, table, torch.full_like(lens, at))
    assert all(torch.equal(a, b) for a, b in zip(*pools))
    same = q.clone(memory_format=torch.contiguous_format)
    assert torch.equal(ops.paged_decode_8bit(q, *pools[0], table, lens), ops.paged_decode_8bit(same, *pools[1], table, lens))
    k = torch.randn(1, 64, 2, 64, device="cuda", dtype=torch.float16)
    assert torch.equal(ops.decode(q, k, k, seqlens=lens), ops.decode(same, k, k, seqlens=lens))

