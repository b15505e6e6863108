"""The block-scaled operators at sizes past 16 and 32 bits."""
import pytest
import torch
from test_blocks_gpu import operands

from h3b import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("experts,each", [(70_000, 1), (40_000, 16)])
def test_more_row_tiles_than_a_grid_axis_holds(dev, experts, each):
    rows, n, k = experts * each, 16, 32
    a, w, sa, sb = operands(rows, n, k, seed=experts, experts=experts)
    y = ops.fp8_gemm_grouped(a, w, sa, sb, torch.arange(0, rows + 1, each, dtype=torch.int32, device=dev))
    ad = a.double().view(experts, each, k) * sa.double().view(experts, each, 1)
    wd = w.double() * sb.double()
    ref, size = (torch.bmm(p, q.transpose(1, 2)).view(rows, n) for p, q in ((ad, wd), (ad.abs(), wd.abs())))
    acc = (128 + 1 + 4) * 2.0 ** -23 * size
    assert float(((y.double() - ref).abs() - acc - 2.0 ** -8 * (ref.abs() + acc)).max()) <= 0
    assert ops.device_status() == 0
