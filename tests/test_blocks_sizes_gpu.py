"""The block-scaled operators at sizes past 16 and 32 bits: many experts, tensors of 2^31 elements and more."""
import pytest
import torch
from test_blocks_gpu import bounds, check_product, codes, nb, operands, quant_oracle

from h3b import ops

BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn
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


LARGE = 1 << 31


def test_quantisers_past_2_31_elements(dev):
    """The last rows of a tensor of more than 2^31 elements give the bits that they give by themselves."""
    m, k = 420_003, 5136
    assert m * k > LARGE
    x = torch.randn(4099, k, device=dev, generator=torch.Generator(device=dev).manual_seed(1)).to(BF16).repeat(103, 1)[:m]
    tail = x[-70:].clone()
    q, s = ops.quant_blocks(x)
    for rows in (slice(0, 70), slice(m - 70, m)):
        rq, rs = quant_oracle(x[rows])
        assert torch.equal(s[rows], rs) and torch.equal(codes(q[rows]), codes(rq))
    want = ops.silu_mul_quant_blocks(tail)
    del q, s
    q, s = ops.silu_mul_quant_blocks(x)
    assert torch.equal(s[-70:], want[1]) and torch.equal(codes(q[-70:]), codes(want[0]))
    del q, s
    w = x.view(-1)[:67 * 6251 * 5136].view(67, 6251, 5136)
    assert w.numel() > LARGE
    q, s = ops.quant_weight_blocks(w)
    rq, rs = ops.quant_weight_blocks(w[66].contiguous())
    assert torch.equal(s[66], rs) and torch.equal(codes(q[66]), codes(rq))


def test_quantisers_with_rows_2_31_elements_apart(dev):
    held = torch.empty(LARGE + (1 << 20), dtype=BF16, device=dev)
    x = held.as_strided((3, 512), (1 << 30, 1))
    x.copy_(torch.randn(3, 512, device=dev, generator=torch.Generator(device=dev).manual_seed(2)))
    c = x.contiguous()
    for fn in (ops.quant_blocks, ops.silu_mul_quant_blocks, ops.quant_weight_blocks):
        (q, s), (rq, rs) = fn(x), fn(c)
        assert torch.equal(s, rs) and torch.equal(codes(q), codes(rq))


def test_products_past_2_31_elements(dev):
    """An output and a weight of more than 2^31 elements, and operands whose last rows lie that far from the first."""
    m, n, k = 70_001, 31_000, 144
    assert m * n > LARGE
    a, w, sa, sb = operands(m, n, k, seed=3)
    y = ops.fp8_gemm_blocks(a, w, sa, sb)
    for rows in (slice(0, 40), slice(m - 300, m)):
        check_product(y[rows], a[rows], w, sa[rows], sb)
    off = bounds([m - 301, 0, 301])
    three = torch.stack([w, w, w.view(torch.uint8).flip(0).view(E4M3)])
    y = ops.fp8_gemm_grouped(a, three, sa, torch.stack([sb] * 3), off, out=y)
    check_product(y[-301:], a[-301:], three[2], sa[-301:], sb)
    del y, three
    held = torch.empty(LARGE + (1 << 20), dtype=torch.uint8, device=dev)
    for rows in (3, 300):
        ld = (LARGE // (rows - 1) + 15) // 16 * 16
        far = held.as_strided((rows, k), (ld, 1)).view(E4M3)
        far.copy_(a[:rows])
        far_out = held.view(BF16).as_strided((rows, 200), (ld // 2, 1), 1024)
        want = ops.fp8_gemm_blocks(a[:rows], w[:200], sa[:rows], sb[:2])
        assert torch.equal(ops.fp8_gemm_blocks(far, w[:200], sa[:rows], sb[:2], out=far_out), want)
        assert torch.equal(ops.fp8_gemm_blocks(w[:200], far, sa[:1].expand(200, -1), sb[:-(-rows // 128)]),
                           ops.fp8_gemm_blocks(w[:200], a[:rows], sa[:1].expand(200, -1), sb[:-(-rows // 128)]))


def test_grouped_weight_past_2_31_elements(dev):
    e, n, k = 70, 6000, 5120
    assert e * n * k > LARGE
    w = torch.randint(0, 256, (n, k), dtype=torch.uint8, device=dev, generator=torch.Generator(device=dev).manual_seed(5))
    w = torch.where(w & 0x7F >= 0x78, w & 0x87, w).repeat(e, 1, 1)
    w[-1].copy_(w[-1].flip(0))
    w = w.view(E4M3)
    for each in (1, 200):
        a, _, sa, _ = operands(e * each, 16, k, seed=each)
        sb = torch.rand(e, nb(n), nb(k), device=dev) * 1e-3 + 1e-5
        y = ops.fp8_gemm_grouped(a, w, sa, sb, bounds([each] * e))
        for i in (0, e - 1):
            rows = slice(i * each, (i + 1) * each)
            check_product(y[rows], a[rows], w[i], sa[rows], sb[i])
