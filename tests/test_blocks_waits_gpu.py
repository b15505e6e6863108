"""The block-scaled products beside a device wait that runs out: what is in an output is right or was there before."""
import subprocess
import sys

import pytest
import torch
from test_blocks_gpu import operands

from h3b import _lib, ops

BF16 = torch.bfloat16
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,k", [(1, 5120, 5120), (40, 40960, 512), (100, 5120, 5120), (300, 9000, 512), (2000, 9999, 400)])
def test_products_beside_a_wait_that_gives_up(dev, m, n, k):
    """A barrier that nobody joins gives up after 10 ms while products run on another stream: a product that ends early
    leaves whole values only, the ones behind it leave their outputs alone, and all is well once the status is read."""
    a, w, sa, sb = operands(m, n, k, seed=m)
    want = ops.fp8_gemm_blocks(a, w, sa, sb)
    outs = [torch.full((m, n), 7.0, dtype=BF16, device=dev) for _ in range(8)]
    flags = [torch.zeros(8, dtype=torch.int32, device=dev) for _ in range(2)]
    side, lib = torch.cuda.Stream(), _lib.load()
    torch.cuda.synchronize()
    assert ops.device_status() == 0
    _lib.check(lib.h3b_set_wait_timeout_ns(10_000_000), "h3b_set_wait_timeout_ns")
    try:
        ops.p2p_signal_wait(flags, flags[0], 0, 7, side.cuda_stream)
        while not side.query():
            ops.fp8_gemm_blocks(a, w, sa, sb, out=outs[0])
        for y in outs[1:]:
            ops.fp8_gemm_blocks(a, w, sa, sb, out=y)
        torch.cuda.synchronize()
        assert ops.device_status() == _lib.H3B_ETIMEOUT
    finally:
        _lib.check(lib.h3b_set_wait_timeout_ns(4_000_000_000), "h3b_set_wait_timeout_ns")
    for y in outs:
        assert bool(((y == want) | (y == 7)).all())
    assert bool((outs[-1] == 7).all())
    assert ops.device_status() == 0
    assert torch.equal(ops.fp8_gemm_blocks(a, w, sa, sb), want)


def test_first_call_of_a_process_on_a_side_stream(dev):
    """The status words are allocated by the first product, whose kernel may not see them before they are zero."""
    code = ("import sys; sys.path[:0] = %r\n"
            "import torch\n"
            "from h3b import ops\n"
            "a = torch.ones(40, 256, device='cuda').to(torch.float8_e4m3fn)\n"
            "s, t = torch.ones(40, 2, device='cuda'), torch.ones(1, 2, device='cuda')\n"
            "torch.cuda.synchronize()\n"
            "with torch.cuda.stream(torch.cuda.Stream()):\n"
            "    y = ops.fp8_gemm_blocks(a, a, s, t)\n"
            "    z = ops.fp8_gemm_blocks(a, a, s, t)\n"
            "torch.cuda.synchronize()\n"
            "assert bool((y == 256).all()) and bool((z == 256).all())\n"
            "assert ops.device_status() == 0\n") % sys.path
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr
