"""Calls from several host threads at once."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("backward", [False, True])
def test_wide_and_narrow_rows(backward):
    """The streaming kernels of two widths share a shared-memory limit: no call lowers it under another thread's launch."""
    from tritonops_b200 import ops
    raised, ready = [], threading.Barrier(8, timeout=60)

    def make(dim):
        x, w = torch.randn(1024, dim, device="cuda").bfloat16(), torch.ones(dim, device="cuda", dtype=torch.bfloat16)
        y, rstd = ops.rmsnorm_fwd(x, w, 1e-6)
        return (lambda: ops.rmsnorm_bwd(y, x, w, rstd)) if backward else (lambda: ops.rmsnorm_fwd(x, w, 1e-6))

    def loop(call):
        with torch.cuda.stream(torch.cuda.Stream()):
            ready.wait()
            try:
                for _ in range(20000):
                    call()
            except (RuntimeError, ValueError) as e:
                raised.append(str(e))

    calls = [make(dim) for dim in (1024, 4096 if backward else 5120)] * 4
    torch.cuda.synchronize()
    threads = [threading.Thread(target=loop, args=(call,)) for call in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not raised
