"""Block-scaled operators captured: forms that first run inside a capture, and bounds that go bad between replays."""
import subprocess
import sys

import pytest
import torch
from test_blocks_gpu import bounds, check_product, operands

from h3b import ops

BF16 = torch.bfloat16
pytestmark = pytest.mark.gpu


def test_forms_that_first_run_in_a_capture(dev):
    """One product of one row, then a graph with every other form and quantiser, none of which the process has run."""
    code = ("import sys; sys.path[:0] = %r\n"
            "import torch\n"
            "from h3b import ops\n"
            "from test_blocks_gpu import operands, bounds\n"
            "x = torch.randn(70, 512, device='cuda').to(torch.bfloat16)\n"
            "jobs = [operands(m, n, k, seed=m) for m, n, k in ((1, 512, 512), (20, 512, 512), (60, 512, 512),\n"
            "        (100, 5120, 5120), (300, 20000, 272), (2000, 9999, 400), (513, 2568, 9216))]\n"
            "grouped = operands(640, 264, 512, seed=1, experts=6), bounds([100, 0, 40, 300, 100, 100])\n"
            "ops.fp8_gemm_blocks(*jobs[0])\n"
            "torch.cuda.synchronize()\n"
            "def run():\n"
            "    y = [ops.fp8_gemm_blocks(*j) for j in jobs] + [ops.fp8_gemm_grouped(*grouped[0], grouped[1])]\n"
            "    for fn in (ops.quant_blocks, ops.silu_mul_quant_blocks, ops.quant_weight_blocks):\n"
            "        q, s = fn(x)\n"
            "        y += [q.view(torch.uint8), s]\n"
            "    return y\n"
            "graph = torch.cuda.CUDAGraph()\n"
            "with torch.cuda.graph(graph):\n"
            "    y = run()\n"
            "graph.replay()\n"
            "torch.cuda.synchronize()\n"
            "assert all(torch.equal(a, b) for a, b in zip(y, run()))\n"
            "assert ops.device_status() == 0\n") % sys.path
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr


@pytest.mark.parametrize("rows,n,k", [(48, 4096, 512), (300, 520, 4096), (3000, 4096, 512)])
def test_bounds_that_go_bad_between_replays(dev, rows, n, k):
    a, w, sa, sb = operands(rows, n, k, seed=rows, experts=4)
    good = bounds([rows // 3, 0, rows // 3, rows - 2 * (rows // 3)])
    bad = good.clone()
    bad[1] = rows + 1
    off, out = good.clone(), torch.empty(rows, n, dtype=BF16, device=dev)
    want = ops.fp8_gemm_grouped(a, w, sa, sb, good)
    torch.cuda.synchronize()
    assert ops.device_status() == 0
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.fp8_gemm_grouped(a, w, sa, sb, off, out=out)
    for at in (good, bad, bad, good):
        off.copy_(at)
        out.fill_(7.0)
        graph.replay()
        first = 0 if at is good else rows // 3       # the groups on both sides of the bad bound are left out
        assert bool((out[:first] == 7).all()) and torch.equal(out[first:], want[first:])
    assert ops.device_status() == -1
    check_product(out[:rows // 3], a[:rows // 3], w[0], sa[:rows // 3], sb[0])
