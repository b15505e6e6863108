"""Bad bounds of the grouped block-scaled product, in calls of many waves and in every form: each group that is served is
right, each row that is not keeps what it held, and neither the calls behind it nor those of another stream notice."""
import pytest
import torch
from test_blocks_gpu import bounds, check_product, operands

from h3b import ops

BF16 = torch.bfloat16
pytestmark = pytest.mark.gpu


def served(off, rows):
    """The rows that each group is served for: a group out of range or out of order has none, and one that begins below the end
    of an earlier group has those from that end on."""
    reach, got = 0, []
    for lo, hi in zip(off[:-1], off[1:]):
        if not 0 <= lo <= hi <= rows:
            got.append((0, 0))
            continue
        got.append((max(lo, reach), hi) if max(lo, reach) < hi else (0, 0))
        reach = max(reach, hi)
    return got


# narrow (16 and 64 rows a tile; whole K and K in parts), wide in rounds and wide with K in parts
FORMS = [(640, 64, 4096, 512), (700, 70, 200, 2048), (1400, 70, 4096, 512), (4800, 48, 4096, 512), (480, 6, 136, 4096),
         (9000, 40, 2000, 256), (1000, 70, 136, 128)]


def spoil(rows, experts, how):
    step = rows // experts
    off = [step * e for e in range(experts)] + [rows]
    if how == "late":
        off[experts - 1] = rows + 1
    elif how == "early":
        off[0] = -1
    elif how == "huge":
        off[2] = 2_000_000_000
    elif how == "down":
        off[3] = step // 2
    elif how == "edge":           # around the 32nd bound
        at = min(32, experts - 2)
        off[at] = off[at - 2] - 1
    elif how == "two":
        off[1], off[experts // 2] = -(1 << 31), rows + 7
    elif how == "again":          # every second group claims all rows
        off = [0 if e % 2 == 0 else rows for e in range(experts)] + [rows]
    return off


@pytest.mark.parametrize("how", ["late", "early", "huge", "down", "edge", "two", "again"])
@pytest.mark.parametrize("rows,experts,n,k", FORMS)
def test_bad_bounds_reach_no_other_group(dev, rows, experts, n, k, how):
    a, w, sa, sb = operands(rows, n, k, seed=rows, experts=experts)
    off = spoil(rows, experts, how)
    at = torch.tensor(off, dtype=torch.int64, device=dev)
    assert ops.device_status() == 0
    for _ in range(3):
        y = torch.full((rows, n), 7.0, dtype=BF16, device=dev)
        ops.fp8_gemm_grouped(a, w, sa, sb, at, out=y)
        left = torch.ones(rows, dtype=torch.bool)
        for e, (lo, hi) in enumerate(served(off, rows)):
            if lo < hi:
                check_product(y[lo:hi], a[lo:hi], w[e], sa[lo:hi], sb[e])
                left[lo:hi] = False
        assert bool((y[left.to(dev)] == 7).all())
    assert ops.device_status() == -1
    assert ops.device_status() == 0


def test_calls_after_bad_bounds_are_served(dev):
    """Until somebody reads the status the products, the per-token product and the attention go on, on every stream."""
    a, w, sa, sb = operands(300, 512, 512, seed=1, experts=3)
    bad, good = torch.tensor([0, 400, 20, 300], device=dev), bounds([100, 0, 200])
    a8 = torch.randn(256, 512, device=dev).to(torch.float8_e4m3fn)
    one = torch.ones(256, device=dev)
    qkv = torch.randn(3, 256, 2, 128, device=dev).to(BF16)

    def calls():
        return (ops.fp8_gemm_grouped(a, w, sa, sb, good), ops.fp8_gemm_blocks(a[:5], w[0], sa[:5], sb[0]),
                ops.fp8_gemm_blocks(a, w[1], sa, sb[1]), ops.fp8_gemm(a8, a8, one, one), ops.flash_attn(*qkv))

    want = calls()
    assert ops.device_status() == 0
    ops.fp8_gemm_grouped(a, w, sa, sb, bad)
    got, side = [calls()], torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.fp8_gemm_grouped(a, w, sa, sb, bad)
        got.append(calls())
    torch.cuda.synchronize()
    assert all(torch.equal(y, z) for ys in got for y, z in zip(ys, want))
    assert ops.device_status() == -1
    assert ops.device_status() == 0
