"""A call whose launch CUDA refuses answers with an error, and the next call knows nothing of it."""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu
i32 = torch.int32


def append(dev):
    from tritonops_b200 import ops
    k, v = (torch.zeros(2, 16, 1, 32, dtype=torch.int8, device=dev) for _ in range(2))
    ks, vs = (torch.zeros(2, 1, 1, device=dev) for _ in range(2))
    rows, at = torch.ones(1, 1, 32, dtype=torch.float16, device=dev), torch.zeros(1, 1, dtype=i32, device=dev)
    return lambda: ops.append_kv_8bit(k, v, ks, vs, rows, rows, at, at.view(1))


def grow(dev):
    from tritonops_b200 import ops
    table, n, refs = torch.full((2, 4), -1, dtype=i32, device=dev), torch.ones(2, dtype=i32, device=dev), torch.zeros(8, dtype=i32, device=dev)
    return lambda: ops.grow_pages(table, n, refs, n, page_size=16)


def norm(dev):
    from tritonops_b200 import ops
    x, w = (torch.ones(n, 4096, device=dev, dtype=torch.bfloat16) for n in (1024, 1))
    return lambda: ops.rmsnorm_fwd(x, w[0], 1e-6)


@pytest.mark.parametrize("make", [append, grow, norm])
def test_next_call_does_not_report_it(make):
    """The launch goes to a stream whose capture has been made invalid (by a synchronisation within it)."""
    rt = C.CDLL("libcudart.so.12")
    s = torch.cuda.Stream()
    call = make("cuda")
    with torch.cuda.stream(s):
        s.wait_stream(torch.cuda.default_stream())
        call()                                     # (the allocations of the next one are cached now)
        s.synchronize()
        stream, graph = C.c_void_p(s.cuda_stream), C.c_void_p()
        assert rt.cudaStreamBeginCapture(stream, 1) == 0
        assert rt.cudaStreamSynchronize(stream) != 0
        with pytest.raises(RuntimeError, match="a CUDA call failed"):
            call()
        assert rt.cudaStreamEndCapture(stream, C.byref(graph)) != 0
        rt.cudaGetLastError()
        call()
        s.synchronize()
