"""The block-scaled FP8 operators on the GPU against their formulas in 64 bits.

Bounds.  Quant: a scale is a correctly rounded quotient (2^-24); a code is off by at most half an e4m3 step.  silu(g) * u
in fp32 with the fast exponential and division: (6 + 1.2 |g|) * 2^-23 relative.  Products: e4m3 products are exact in
fp32; a block's 128 products and the blocks' scaled sums are added in fp32, each addition off by at most one unit in the
last place of a partial sum, which is at most S = sum |sa sb a w|: (128 + blocks + 4) * 2^-23 * S, and the output rounding
(half a step: 2^-8 bf16, 2^-11 f16 relative)."""
import pytest
import torch

from h3b import ops

BF16, F16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
B = 128
pytestmark = pytest.mark.gpu
HALF_STEP = {BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {BF16: 2.0 ** -133, F16: 2.0 ** -25}      # half of the smallest subnormal step


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def nb(n):
    return -(-n // B)


def spread(s, n, dim):
    """Each block's scale at each of its n places along dim."""
    return s.repeat_interleave(B, dim=dim).narrow(dim, 0, n)


def FP8_MAX(like):
    """448 as a tensor: torch divides by a Python number with its reciprocal, which is not the rounded quotient."""
    return torch.full((1,), 448.0, device=like.device)


def quant_oracle(x):
    """The eager fp32 formula (IEEE division), block by block of the last dimension."""
    rows, k = x.shape
    p = torch.nn.functional.pad(x.float(), (0, nb(k) * B - k)).view(rows, nb(k), B)
    s = torch.maximum(p.abs().amax(-1) / FP8_MAX(x), torch.tensor(1.0 / (448.0 * 512.0), device=x.device))
    q = (p * (torch.ones_like(s) / s)[..., None]).clamp(-448.0, 448.0)
    return q.view(rows, -1)[:, :k].to(E4M3), s


def codes(t):
    return t.contiguous().view(torch.uint8)


def half_step_e4m3(v):
    """Half the e4m3 step at |v| <= 448 (64-bit)."""
    _, e = torch.frexp(v)
    return torch.exp2((e.double() - 4).clamp_min(-9.0)) / 2


def check_product(y, a, w, sa, sb, bias=None):
    ad = a.double() * spread(sa.double(), a.shape[1], 1)
    wd = w.double() * spread(spread(sb.double(), w.shape[0], 0), w.shape[1], 1)
    ref, size = ad @ wd.t(), ad.abs() @ wd.abs().t()
    if bias is not None:
        ref, size = ref + bias.double(), size + bias.double().abs()
    acc = (B + sa.shape[1] + 4) * 2.0 ** -23 * size
    tol = acc + HALF_STEP[y.dtype] * (ref.abs() + acc) + TINY[y.dtype]
    bad = ((y.double() - ref).abs() - tol).max()
    assert bool(torch.isfinite(y).all()) and float(bad) <= 0, f"off by {float(bad)} beyond the bound"


def operands(m, n, k, seed=0, experts=None, scale_major="block"):
    g = gen(seed)
    a = (torch.randn(m, k, device="cuda", generator=g) * 100).clamp(-448, 448).to(E4M3)
    shape = (n, k) if experts is None else (experts, n, k)
    w = (torch.randn(shape, device="cuda", generator=g) * 100).clamp(-448, 448).to(E4M3)
    sa = torch.rand(m, nb(k), device="cuda", generator=g) * 0.02 + 1e-3
    if scale_major == "block":
        sa = sa.t().contiguous().t()
    sb = torch.rand((*shape[:-2], nb(n), nb(k)), device="cuda", generator=g) * 1e-3 + 1e-5
    return a, w, sa, sb


# ---------------------------------------------------------------------------------------------------------------
# quantisers
# ---------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("m,k", [(1, 1), (1, 8), (3, 120), (1, 128), (2, 129), (5, 136), (17, 1000), (64, 5120),
                                 (1, 5120), (129, 13824), (7, 1001)])
def test_quant_blocks_is_the_eager_formula(dev, m, k):
    x = (torch.randn(m, k, device=dev, generator=gen(m + k)) * 3).to(BF16)
    q, s = ops.quant_blocks(x)
    rq, rs = quant_oracle(x)
    assert q.shape == (m, k) and s.shape == (m, nb(k)) and s.dtype == torch.float32
    assert torch.equal(s, rs) and torch.equal(codes(q), codes(rq))
    full = spread(s.double(), k, 1)
    v = x.double() / full
    # the code rounds fl(x * fl(1/s)): two roundings of 2^-24 before it, 2^-23 |v|; with |v| < 2^e the half step is
    # 2^(e-5) or more, so that is at most 2^-18 of it
    assert float(((q.double() - v).abs() - half_step_e4m3(v) * (1 + 2.0 ** -18)).max()) <= 0


def test_quant_blocks_every_bf16_maximum(dev):
    """A block for each positive finite bf16 value as its maximum, and the whole tile of a weight likewise."""
    top = torch.arange(1, 0x7F80, dtype=torch.int32, device=dev).to(torch.int16).view(BF16)
    x = (torch.rand(top.numel(), 128, device=dev, generator=gen(1)) * 2 - 1) * top.float()[:, None]
    x = torch.where(x.abs() > top.float()[:, None], 0.0, x).to(BF16)
    x[:, 77] = -top
    q, s = ops.quant_blocks(x)
    rq, rs = quant_oracle(x)
    assert torch.equal(s, rs) and torch.equal(codes(q), codes(rq))
    tiles = x[:254].view(254, 1, 128).expand(254, 128, 128).contiguous()
    q, s = ops.quant_weight_blocks(tiles)
    assert torch.equal(s.view(-1), rs[:254, 0]) and torch.equal(codes(q[:, 5]), codes(rq[:254]))


def test_quant_blocks_special_rows(dev):
    """Zero blocks take the smallest scale; a NaN or an infinity marks its own block only; subnormals and the largest
    value keep the formula."""
    x = torch.randn(8, 384, device=dev, generator=gen(3)).to(BF16)
    x[0] = 0
    x[1, 5] = float("nan")
    x[2, 130] = float("inf")
    x[3, :128] = torch.finfo(BF16).max
    x[4] = 1e-40
    x[5, 256:] = float("-inf")
    x[6, 127] = -torch.finfo(BF16).max
    q, s = ops.quant_blocks(x)
    rq, rs = quant_oracle(x)
    # the eager maximum with the smallest scale propagates NaN as the kernel does
    assert torch.equal(torch.isnan(s), torch.isnan(rs))
    assert torch.equal(s[~torch.isnan(s)], rs[~torch.isnan(rs)])
    nan = torch.isnan(rq.float())
    assert torch.equal(torch.isnan(q.float()), nan)
    assert torch.equal(codes(q)[~nan], codes(rq)[~nan])
    assert float(s[0, 0]) == float(torch.tensor(1.0 / (448.0 * 512.0))) and bool((q[0].float() == 0).all())
    assert not bool(torch.isnan(s[1, 1:]).any()) and not bool(torch.isinf(s[2, [0, 2]]).any())


def test_quant_blocks_strided_rows_and_division_mode(dev):
    wide = torch.randn(33, 1000, device=dev, generator=gen(4)).to(BF16)
    for view in (wide[:, :512], wide[:, 3:700], wide[::2, 8:136], wide[5:6]):
        q, s = ops.quant_blocks(view)
        rq, rs = quant_oracle(view)
        assert torch.equal(s, rs) and torch.equal(codes(q), codes(rq))
    s_full = ops.quant_blocks(wide, div_mode=ops.DIV_FULL)[1]
    s_ieee = ops.quant_blocks(wide)[1]
    assert float(((s_full - s_ieee) / s_ieee).abs().max()) <= 2.0 ** -22   # div.full: 2 units in the last place


@pytest.mark.parametrize("shape", [(1, 1), (128, 128), (130, 144), (200, 1001), (1, 5120), (3, 100, 272), (4, 256, 640),
                                   (2, 129, 24)])
def test_quant_weight_blocks(dev, shape):
    w = (torch.randn(shape, device=dev, generator=gen(len(shape) + shape[-1])) * 0.02).to(BF16)
    q, s = ops.quant_weight_blocks(w)
    n, k = shape[-2:]
    assert q.shape == shape and s.shape == (*shape[:-2], nb(n), nb(k))
    three = w.view(-1, n, k).float()
    p = torch.nn.functional.pad(three, (0, nb(k) * B - k, 0, nb(n) * B - n)).view(-1, nb(n), B, nb(k), B)
    rs = (p.abs().amax(dim=(2, 4)) / FP8_MAX(w)).clamp_min(1.0 / (448.0 * 512.0))
    rq = (p * (torch.ones_like(rs) / rs)[:, :, None, :, None]).clamp(-448, 448).view(-1, nb(n) * B, nb(k) * B)[:, :n, :k].to(E4M3)
    assert torch.equal(s.view_as(rs), rs) and torch.equal(codes(q.view_as(rq)), codes(rq))


def test_quant_weight_blocks_strided(dev):
    big = torch.randn(3, 300, 400, device=dev, generator=gen(9)).to(BF16)
    view = big[:, 10:200, 8:264]
    q, s = ops.quant_weight_blocks(view)
    rq, rs = ops.quant_weight_blocks(view.contiguous())
    assert torch.equal(codes(q), codes(rq)) and torch.equal(s, rs)


@pytest.mark.parametrize("k", [256, 272, 264, 250])
@pytest.mark.parametrize("m", [8, 13, 130])
def test_quantisers_same_bits_for_any_alignment(dev, m, k):
    """32-byte, 16-byte and single-value accesses: columns of a larger tensor that start at 0, 8, 16 and 1 values."""
    base = (torch.randn(m, 2 * k, device=dev, generator=gen(m + k)) * 2).to(BF16)
    want = ops.quant_blocks(base), ops.silu_mul_quant_blocks(base), ops.quant_weight_blocks(base)
    for ld in (2 * k + 40, 2 * k + 48 - 2 * k % 16, 2 * k + 33):
        big = torch.full((m + 1, ld), float("nan"), dtype=BF16, device=dev)
        for first in (0, 8, 16, 1):
            x = big[:m, first:first + 2 * k]
            x.copy_(base)
            got = ops.quant_blocks(x), ops.silu_mul_quant_blocks(x), ops.quant_weight_blocks(x)
            for (q, s), (rq, rs) in zip(got, want):
                assert torch.equal(s, rs) and torch.equal(codes(q), codes(rq))
            big.fill_(float("nan"))


@pytest.mark.parametrize("m,f,gain", [(1, 128, 1.0), (3, 100, 1.0), (17, 13824, 1.5), (40, 136, 30.0), (5, 77, 4.0)])
def test_silu_mul_quant_blocks(dev, m, f, gain):
    x = (torch.randn(m, 2 * f, device=dev, generator=gen(f)) * gain).to(BF16)
    q, s = ops.silu_mul_quant_blocks(x)
    assert q.shape == (m, f) and s.shape == (m, nb(f))
    check_silu(q, s, x)


def test_silu_mul_quant_blocks_special_values(dev):
    """Gates far out on both sides, infinities and NaN give what g / (1 + exp(-g)) * u gives."""
    x = torch.ones(6, 512, device=dev, dtype=BF16)
    x[0, :256] = -1e4            # silu = -0
    x[1, :256] = 1e4
    x[2, 3] = float("nan")
    x[3, 200] = float("inf")
    x[4, 7] = float("-inf")      # -inf / inf
    x[5, 256 + 9] = float("nan")
    q, s = ops.silu_mul_quant_blocks(x)
    h = x[:, :256].float() / (1 + torch.exp(-x[:, :256].float())) * x[:, 256:].float()
    p = h.view(6, 2, 128).abs().amax(-1)
    assert torch.equal(torch.isnan(s), torch.isnan(p)) and torch.equal(torch.isinf(s), torch.isinf(p))
    fine = torch.isfinite(p)
    ref = (p[fine] / 448).clamp_min(1.0 / (448.0 * 512.0))
    assert float(((s[fine] - ref) / ref).abs().max()) < 1e-5
    assert bool((q[0].float() == 0).all()) and bool((q[1].float() == 448).all())


def test_empty_inputs(dev):
    for q, s in (ops.quant_blocks(torch.empty(0, 256, dtype=BF16, device=dev)),
                 ops.silu_mul_quant_blocks(torch.empty(0, 512, dtype=BF16, device=dev))):
        assert q.shape == (0, 256) and s.shape == (0, 2)
    q, s = ops.quant_blocks(torch.empty(3, 0, dtype=BF16, device=dev))
    assert q.shape == (3, 0) and s.shape == (3, 0)
    q, s = ops.quant_weight_blocks(torch.empty(2, 0, 64, dtype=BF16, device=dev))
    assert q.shape == (2, 0, 64) and s.shape == (2, 0, 1)
    a, w, sa, sb = operands(4, 100, 128)
    assert ops.fp8_gemm_blocks(a[:0], w, sa[:0], sb).shape == (0, 100)
    a, w, sa, sb = operands(4, 100, 128, experts=2)
    off = torch.zeros(3, dtype=torch.int32, device=dev)
    assert ops.fp8_gemm_grouped(a[:0], w, sa[:0], sb, off).shape == (0, 100)


# ---------------------------------------------------------------------------------------------------------------
# the product
# ---------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("k", [16, 128, 144, 1040])
@pytest.mark.parametrize("n", [1, 7, 128, 136, 300])
@pytest.mark.parametrize("m", [1, 2, 16, 17, 33, 64, 65, 128, 129, 257, 300])
def test_product_sizes(dev, m, n, k):
    a, w, sa, sb = operands(m, n, k, seed=m * 7 + n)
    check_product(ops.fp8_gemm_blocks(a, w, sa, sb), a, w, sa, sb)


@pytest.mark.parametrize("m,n,k", [(1, 5120, 5120), (8, 2816, 13824), (100, 5120, 5120), (777, 1544, 5120),
                                   (1000, 5120, 2048), (4097, 768, 1152)])
def test_product_larger(dev, m, n, k):
    a, w, sa, sb = operands(m, n, k, seed=k)
    check_product(ops.fp8_gemm_blocks(a, w, sa, sb), a, w, sa, sb)


@pytest.mark.parametrize("out_dtype", [BF16, F16])
@pytest.mark.parametrize("m,n,k", [(5, 300, 640), (200, 300, 640), (20, 256, 512)])
def test_product_bias_and_types(dev, m, n, k, out_dtype):
    a, w, sa, sb = operands(m, n, k, seed=5)
    bias = (torch.randn(n, device=dev, generator=gen(1)) * 3).to(BF16)
    check_product(ops.fp8_gemm_blocks(a, w, sa, sb, bias, out_dtype), a, w, sa, sb, bias)


@pytest.mark.parametrize("m", [3, 16, 40, 100, 128, 300, 513])
def test_product_is_exact_on_integers(dev, m):
    """Small integers with power-of-two scales: every partial sum is exact, so any order gives the same bits."""
    n, k = 392, 1424
    g = gen(m)
    a = torch.randint(-3, 4, (m, k), device=dev, generator=g).float().to(E4M3)
    w = torch.randint(-3, 4, (n, k), device=dev, generator=g).float().to(E4M3)
    sa = torch.exp2(torch.randint(-2, 3, (m, nb(k)), device=dev, generator=g).float())
    sb = torch.exp2(torch.randint(-2, 3, (nb(n), nb(k)), device=dev, generator=g).float())
    ref = (a.double() * spread(sa.double(), k, 1)) @ (w.double() * spread(spread(sb.double(), n, 0), k, 1)).t()
    assert torch.equal(ops.fp8_gemm_blocks(a, w, sa, sb), ref.to(BF16))


@pytest.mark.parametrize("m", [9, 70, 301])
def test_product_strided_operands_and_output(dev, m):
    n, k = 264, 640
    g = gen(m)
    big_a = (torch.randn(m, k + 48, device=dev, generator=g) * 60).to(E4M3)
    big_w = (torch.randn(n + 5, k + 32, device=dev, generator=g) * 60).to(E4M3)
    a, w = big_a[:, 16:16 + k], big_w[5:, :k]
    sa = (torch.rand(m, 2 * nb(k), device=dev, generator=g) + 0.1)[:, ::2]          # row-major, every second column
    sb = (torch.rand(nb(k), nb(n), device=dev, generator=g) + 0.1).t()
    want = ops.fp8_gemm_blocks(a.contiguous(), w.contiguous(), sa.contiguous(), sb.contiguous())
    check_product(want, a, w, sa, sb)
    assert torch.equal(ops.fp8_gemm_blocks(a, w, sa, sb), want)
    for ld, first in ((n + 8, 0), (n + 3, 0), (n + 16, 8), (n + 8, 3)):              # aligned rows, odd rows, odd start
        buf = torch.full((m, ld + 8), 7.0, dtype=BF16, device=dev)
        out = buf[:, first:first + n]
        assert ops.fp8_gemm_blocks(a, w, sa, sb, out=out) is out
        assert torch.equal(out, want)
        assert bool((buf[:, :first] == 7).all()) and bool((buf[:, first + n:] == 7).all())


@pytest.mark.parametrize("m", [4, 90, 400])
def test_product_nan_stays_in_its_row(dev, m):
    """A NaN or infinite scale or value of one row reaches that row only."""
    a, w, sa, sb = operands(m, 200, 384, seed=2)
    want = ops.fp8_gemm_blocks(a, w, sa, sb)
    a2, sa2 = a.clone(), sa.clone()
    a2.view(torch.uint8)[0, 5] = 0x7F
    sa2[m - 1, 1] = float("inf")
    y = ops.fp8_gemm_blocks(a2, w, sa2, sb)
    assert bool(torch.isnan(y[0]).all()) and not bool(torch.isfinite(y[m - 1]).any())
    assert torch.equal(y[1:m - 1], want[1:m - 1])


# many columns: the wide form with single CTAs (300, 65 rows), with pairs (512, 2,000) and with K in parts (100, 200, 513)
WIDE = [(300, 20001, 272), (65, 40000, 144), (512, 9400, 512), (2000, 9999, 400), (100, 5120, 5120), (200, 5128, 5120),
        (513, 2568, 9216)]


@pytest.mark.parametrize("out_dtype", [BF16, F16])
@pytest.mark.parametrize("m,n,k", WIDE)
def test_wide_product_bias_and_outputs(dev, m, n, k, out_dtype):
    a, w, sa, sb = operands(m, n, k, seed=3)
    bias = (torch.randn(n, device=dev, generator=gen(1)) * 3).to(BF16)
    want = ops.fp8_gemm_blocks(a, w, sa, sb, bias, out_dtype)
    check_product(want, a, w, sa, sb, bias)
    for ld, first in ((n + 24 - n % 8, 8), (n + 13, 3)):                             # aligned rows, odd rows
        buf = torch.full((m + 2, ld), 7.0, dtype=out_dtype, device=dev)
        out = buf[1:m + 1, first:first + n]
        ops.fp8_gemm_blocks(a, w, sa, sb, bias, out=out)
        assert torch.equal(out, want)
        out.fill_(7.0)
        assert bool((buf == 7).all())


@pytest.mark.parametrize("first", [0, 1, 2, 4])
@pytest.mark.parametrize("m,n,k", [*WIDE, (40, 300, 1024), (3, 129, 2048)])
def test_outputs_of_every_alignment(dev, m, n, k, first):
    """Rows that start 16, 8, 4 or 2 bytes aligned, all alike or in turn, and nothing written around them."""
    a, w, sa, sb = operands(m, n, k, seed=4)
    want = ops.fp8_gemm_blocks(a, w, sa, sb)
    for ld in (n + 16 - n % 8, n + 12 - n % 4 + 4 * (n // 4 % 2), n + 10 - n % 2 + 2 * (n // 2 % 2), n + 9 + n % 2):
        buf = torch.full((m + 2, ld), 7.0, dtype=BF16, device=dev)
        out = buf[1:m + 1, first:first + n]
        ops.fp8_gemm_blocks(a, w, sa, sb, out=out)
        assert torch.equal(out, want)
        out.fill_(7.0)
        assert bool((buf == 7).all())


@pytest.mark.parametrize("m,n,k", WIDE)
def test_wide_product_is_exact_on_integers(dev, m, n, k):
    g = gen(m)
    a = torch.randint(-2, 3, (m, k), device=dev, generator=g).float().to(E4M3)
    w = torch.randint(-2, 3, (n, k), device=dev, generator=g).float().to(E4M3)
    sa = torch.exp2(torch.randint(-1, 2, (m, nb(k)), device=dev, generator=g).float())
    sb = torch.exp2(torch.randint(-1, 2, (nb(n), nb(k)), device=dev, generator=g).float())
    ref = (a.double() * spread(sa.double(), k, 1)) @ (w.double() * spread(spread(sb.double(), n, 0), k, 1)).t()
    assert torch.equal(ops.fp8_gemm_blocks(a, w, sa, sb), ref.to(BF16))


@pytest.mark.parametrize("m,n,k", WIDE)
def test_wide_product_nan_stays_in_its_row(dev, m, n, k):
    a, w, sa, sb = operands(m, n, k, seed=2)
    want = ops.fp8_gemm_blocks(a, w, sa, sb)
    a2, sa2 = a.clone(), sa.clone()
    a2.view(torch.uint8)[0, 5] = 0x7F
    sa2[m - 1, 1] = float("nan")
    y = ops.fp8_gemm_blocks(a2, w, sa2, sb)
    assert bool(torch.isnan(y[0]).all()) and bool(torch.isnan(y[m - 1]).all())
    assert torch.equal(y[1:m - 1], want[1:m - 1])


def test_product_repeats_bit_for_bit(dev):
    for m, n, k in ((1, 512, 5120), (40, 1024, 4096), (600, 1024, 2048)):
        a, w, sa, sb = operands(m, n, k, seed=m)
        first = ops.fp8_gemm_blocks(a, w, sa, sb)
        for _ in range(5):
            assert torch.equal(ops.fp8_gemm_blocks(a, w, sa, sb), first)


# ---------------------------------------------------------------------------------------------------------------
# grouped by expert
# ---------------------------------------------------------------------------------------------------------------


def bounds(sizes, first=0, dtype=torch.int32):
    return torch.tensor([first, *(first + sum(sizes[:i + 1]) for i in range(len(sizes)))], dtype=dtype, device="cuda")


SIZES = [
    [1], [0, 1], [1, 0, 0], [5, 0, 3], [16, 17, 15], [0, 0, 40, 0], [129, 0, 1, 255], [300, 200, 100],
    [0, 600, 1, 0, 30], [256, 256], [1] * 40, [0] * 33 + [9] + [0] * 31 + [2], [3, 50, 0, 128, 65, 1, 7, 0, 33],
    [1000, 1, 1, 1], list(range(0, 70)),
]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{sum(s)}")
@pytest.mark.parametrize("n,k", [(200, 400), (264, 128)])
def test_grouped_sizes(dev, sizes, n, k):
    e, t = len(sizes), sum(sizes)
    a, w, sa, sb = operands(t, n, k, seed=t, experts=e)
    off = bounds(sizes)
    y = ops.fp8_gemm_grouped(a, w, sa, sb, off)
    at = 0
    for i, m in enumerate(sizes):
        if m:
            check_product(y[at:at + m], a[at:at + m], w[i], sa[at:at + m], sb[i])
        at += m
    assert torch.equal(ops.fp8_gemm_grouped(a, w, sa, sb, off.long(), out_dtype=BF16), y)
    assert ops.device_status() == 0


@pytest.mark.parametrize("sizes", [[3, 0, 4], [40, 70, 0, 5], [200, 300], [0, 0], [130]])
@pytest.mark.parametrize("n", [256, 201])
def test_grouped_leaves_other_rows(dev, sizes, n):
    """Rows before the first and behind the last bound keep what they held, and may hold anything in the inputs."""
    k, first, behind = 256, 6, 37
    t = first + sum(sizes) + behind
    a, w, sa, sb = operands(t, n, k, seed=1, experts=len(sizes))
    a.view(torch.uint8)[:first] = 0x7F
    a.view(torch.uint8)[t - behind:] = 0xFF
    sa[t - behind:] = float("nan")
    out = torch.full((t, n), 7.0, dtype=F16, device=dev)
    assert ops.fp8_gemm_grouped(a, w, sa, sb, bounds(sizes, first), out=out) is out
    assert bool((out[:first] == 7).all()) and bool((out[t - behind:] == 7).all())
    at = first
    for i, m in enumerate(sizes):
        if m:
            check_product(out[at:at + m], a[at:at + m], w[i], sa[at:at + m], sb[i])
        at += m


@pytest.mark.parametrize("rows", [30, 600])
@pytest.mark.parametrize("off", [[0, 10, 5, 30], [-3, 10, 20, 30], [0, 10, 20, 10_000], [0, 2_000_000_000, 20, 30]])
def test_grouped_bad_bounds_are_recorded(dev, off, rows):
    """Bounds out of order or out of range: nothing outside the output is touched, and the status word says so."""
    a, w, sa, sb = operands(rows, 136, 256, experts=3)
    buf = torch.full((rows + 400, 136), 7.0, dtype=BF16, device=dev)
    assert ops.device_status() == 0
    ops.fp8_gemm_grouped(a, w, sa, sb, torch.tensor(off, dtype=torch.int64, device=dev), out=buf[200:200 + rows])
    assert ops.device_status() == -1
    assert ops.device_status() == 0
    assert bool((buf[:200] == 7).all()) and bool((buf[200 + rows:] == 7).all())
    good = bounds([10, 10, rows - 20])
    y = ops.fp8_gemm_grouped(a, w, sa, sb, good)                   # and the next call works
    check_product(y[:10], a[:10], w[0], sa[:10], sb[0])


@pytest.mark.parametrize("rows", [20, 480, 560, 9000])
def test_grouped_overlapping_bounds_are_recorded(dev, rows):
    """Every second group claims all rows, the ones between are out of order: more row tiles than correct bounds can make
    (K is split over clusters in the middle cases), no wait that runs out, and the next call works."""
    a, w, sa, sb = operands(rows, 136, 2048, experts=8)
    buf = torch.full((rows + 400, 136), 7.0, dtype=BF16, device=dev)
    assert ops.device_status() == 0
    off = torch.tensor([0, rows, 0, rows, 0, rows, 0, rows, rows], device=dev)
    ops.fp8_gemm_grouped(a, w, sa, sb, off, out=buf[200:200 + rows])
    assert ops.device_status() == -1
    assert bool((buf[:200] == 7).all()) and bool((buf[200 + rows:] == 7).all())
    y = ops.fp8_gemm_grouped(a, w, sa, sb, bounds([rows] + [0] * 7))
    check_product(y, a, w[0], sa, sb[0])


@pytest.mark.parametrize("rows", [1, 128 * 70])
def test_grouped_bad_bounds_behind_the_last_tile(dev, rows):
    """Good groups that use up all row tiles of the launch, and a bad bound far behind them."""
    e = 128
    a, w, sa, sb = operands(rows, 64, 128, experts=e)
    off = torch.full((e + 1,), rows, dtype=torch.int32, device=dev)
    off[0], off[e] = 0, rows + 4
    assert ops.device_status() == 0
    y = ops.fp8_gemm_grouped(a, w, sa, sb, off)
    assert ops.device_status() == -1
    check_product(y, a, w[0], sa, sb[0])


@pytest.mark.parametrize("rows", [48, 700])
def test_grouped_equals_the_dense_product(dev, rows):
    """One expert with all rows: the same bits as the dense product when both take the same form."""
    a, w, sa, sb = operands(rows, 392, 656, experts=1)
    y = ops.fp8_gemm_grouped(a, w, sa, sb, bounds([rows]))
    assert torch.equal(y, ops.fp8_gemm_blocks(a, w[0], sa, sb[0]))


def test_grouped_strided(dev):
    sizes, n, k = [30, 0, 150], 136, 384
    g = gen(8)
    big = (torch.randn(3, n + 9, k + 64, device=dev, generator=g) * 50).to(E4M3)
    w = big[:, 3:3 + n, 16:16 + k]
    a = (torch.randn(sum(sizes), 2 * k, device=dev, generator=g) * 50).to(E4M3)[:, k:]
    sa = torch.rand(sum(sizes), nb(k), device=dev, generator=g)
    sb = torch.rand(3, nb(k), 2 * nb(n), device=dev, generator=g)[:, :, ::2].transpose(1, 2)
    y = ops.fp8_gemm_grouped(a, w, sa, sb, bounds(sizes))
    assert torch.equal(y, ops.fp8_gemm_grouped(a.contiguous(), w.contiguous(), sa, sb.contiguous(), bounds(sizes)))
    check_product(y[30:], a[30:], w[2], sa[30:], sb[2])


def test_many_experts(dev):
    g = gen(0)
    e, t, n, k = 300, 500, 128, 128
    sizes = torch.bincount(torch.randint(0, e, (t,), device=dev, generator=g), minlength=e).tolist()
    a, w, sa, sb = operands(t, n, k, experts=e)
    y = ops.fp8_gemm_grouped(a, w, sa, sb, bounds(sizes))
    at = 0
    for i, m in enumerate(sizes):
        if m:
            check_product(y[at:at + m], a[at:at + m], w[i], sa[at:at + m], sb[i])
        at += m


# ---------------------------------------------------------------------------------------------------------------
# together, captured, on other streams
# ---------------------------------------------------------------------------------------------------------------


def ffn(x, w1, s1, w2, s2, off=None):
    """An FFN as it is served: quant, fc1 (gate | up), silu-mul quant, fc2; every stage's tensors."""
    q, s = ops.quant_blocks(x)
    h = ops.fp8_gemm_blocks(q, w1, s, s1) if off is None else ops.fp8_gemm_grouped(q, w1, s, s1, off)
    q2, sh = ops.silu_mul_quant_blocks(h)
    y = ops.fp8_gemm_blocks(q2, w2, sh, s2) if off is None else ops.fp8_gemm_grouped(q2, w2, sh, s2, off)
    return x, q, s, h, q2, sh, y


def ffn_weights(hidden, f, experts=None):
    shape = (lambda *s: s) if experts is None else (lambda *s: (experts, *s))
    w1 = (torch.randn(shape(2 * f, hidden), device="cuda", generator=gen(1)) * hidden ** -0.5).to(BF16)
    w2 = (torch.randn(shape(hidden, f), device="cuda", generator=gen(2)) * f ** -0.5).to(BF16)
    return (*ops.quant_weight_blocks(w1), *ops.quant_weight_blocks(w2))


def check_silu(q, s, x):
    """q, s of silu_mul_quant_blocks(x) within the bounds of the fast arithmetic and of the roundings."""
    m, f = x.shape[0], x.shape[1] // 2
    g, u = x[:, :f].double(), x[:, f:].double()
    h = g * torch.sigmoid(g) * u
    err = h.abs() * (6 + 1.2 * g.abs()) * 2.0 ** -23 + 1e-36     # values below the normal range may flush to zero
    pad = (0, nb(f) * B - f)
    amax = torch.nn.functional.pad(h.abs(), pad).view(m, -1, B).amax(-1)
    amax_err = torch.nn.functional.pad(err, pad).view(m, -1, B).amax(-1)
    ref = (amax / 448).clamp_min(1.0 / (448.0 * 512.0))
    assert float(((s.double() - ref).abs() - amax_err / 448 - ref * 2.0 ** -23).max()) <= 0
    full = spread(s.double(), f, 1)
    v = h / full
    assert float(((q.double() - v).abs() - half_step_e4m3(v.clamp(-448, 448)) * (1 + 2.0 ** -18) - err / full * 1.001
                  - (v.abs() - 448).clamp_min(0)).max()) <= 0


def check_ffn(stages, w1, s1, w2, s2, rows=slice(None)):
    """Every stage of the run against its formula on what the stage before it gave."""
    x, q, s, h, q2, sh, y = (t[rows] for t in stages)
    rq, rs = quant_oracle(x)
    assert torch.equal(s, rs) and torch.equal(codes(q), codes(rq))
    check_product(h, q, w1, s, s1)
    check_silu(q2, sh, h)
    check_product(y, q2, w2, sh, s2)


@pytest.mark.parametrize("m", [1, 30, 300])
def test_ffn_run(dev, m):
    x = torch.randn(m, 512, device=dev, generator=gen(m)).to(BF16)
    packed = ffn_weights(512, 640)
    check_ffn(ffn(x, *packed), *packed)


def test_expert_ffn_run(dev):
    sizes = [0, 17, 200, 1, 0, 64]
    x = torch.randn(sum(sizes), 512, device=dev, generator=gen(7)).to(BF16)
    packed = ffn_weights(512, 384, experts=6)
    stages = ffn(x, *packed, bounds(sizes))
    at = 0
    for e, m in enumerate(sizes):
        if m:
            check_ffn(stages, *(t[e] for t in packed), rows=slice(at, at + m))
        at += m


def test_captured_with_new_inputs_and_sizes(dev):
    """One graph serves other rows and other group sizes: they are read on the device."""
    packed = ffn_weights(512, 384, experts=4)
    x = torch.randn(64, 512, device=dev, generator=gen(1)).to(BF16)
    off = bounds([10, 20, 30, 4])
    ffn(x, *packed, off)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ffn(x, *packed, off)[-1]
    for seed, sizes in ((2, [0, 64, 0, 0]), (3, [64, 0, 0, 0]), (4, [1, 2, 3, 58])):
        x.copy_(torch.randn(64, 512, device=dev, generator=gen(seed)).to(BF16))
        off.copy_(bounds(sizes))
        graph.replay()
        assert torch.equal(y, ffn(x, *packed, off)[-1])


def test_captured_behind_copies_and_a_joined_stream(dev):
    """The launches' programmatic edges where the node before is a copy or a memset, or there are two of them."""
    packed = ffn_weights(512, 384)
    src = torch.randn(40, 512, device=dev, generator=gen(1)).to(BF16)
    x, y2 = torch.empty_like(src), torch.empty(40, 512, dtype=BF16, device=dev)
    a, w, sa, sb = operands(40, 512, 640)
    ffn(src, *packed)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        x.zero_()
        x.copy_(src)
        y = ffn(x, *packed)[-1]
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        with torch.cuda.stream(side):
            ops.fp8_gemm_blocks(a, w, sa, sb, out=y2)
            q2, s2 = ops.quant_blocks(y2)
        q1, s1 = ops.quant_blocks(y)
        here.wait_stream(side)
        z = ops.fp8_gemm_blocks(q1, w[:, :512].contiguous(), s1, sb[:, :4].contiguous())
        z2 = ops.fp8_gemm_blocks(q2, w[:, :512].contiguous(), s2, sb[:, :4].contiguous())
        x.zero_()
    for seed in (5, 6):
        src.copy_(torch.randn(40, 512, device=dev, generator=gen(seed)).to(BF16))
        graph.replay()
        want = ffn(src, *packed)[-1]
        assert torch.equal(y, want)
        assert torch.equal(z, ops.fp8_gemm_blocks(*_as_product(want, w, sb)))
        assert torch.equal(z2, ops.fp8_gemm_blocks(*_as_product(ops.fp8_gemm_blocks(a, w, sa, sb), w, sb)))
        assert bool((x == 0).all())


def _as_product(y, w, sb):
    q, s = ops.quant_blocks(y)
    return q, w[:, :512].contiguous(), s, sb[:, :4].contiguous()


def test_back_to_back_launches_see_each_other(dev):
    """Every kernel may start before the one ahead of it on the stream ends: chains through the same buffers, with other
    kernels in between, give what launches one at a time give."""
    packed = ffn_weights(512, 384)
    xs = [torch.randn(m, 512, device=dev, generator=gen(m)).to(BF16) for m in (1, 40, 300, 17, 2000, 3)]
    want = []
    for x in xs:
        stages = ffn(x, *packed)
        torch.cuda.synchronize()
        want.append(ffn(stages[-1] * 0.5, *packed)[-1].clone())
        torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for x in xs:
            y = ffn(x, *packed)[-1]
            y.mul_(0.5)
            y = ffn(y, *packed)[-1]
            got.append(y.clone())
            y.fill_(float("nan"))          # the next call's buffers may be this one's
        for g, w in zip(got, want):
            assert torch.equal(g, w)


@pytest.mark.parametrize("m", [1, 20, 64, 300])
def test_weight_written_by_the_kernel_before(dev, m):
    """The product's weight comes from the launch just ahead of it, at the same address every time."""
    n, k = 2048, 2560
    ws = [(torch.randn(n, k, device=dev, generator=gen(i)) * 0.05).to(BF16) for i in range(4)]
    a, _, sa, _ = operands(m, 16, k)
    want = []
    for w in ws:
        wq, sb = ops.quant_weight_blocks(w)
        torch.cuda.synchronize()
        want.append(ops.fp8_gemm_blocks(a, wq, sa, sb))
        check_product(want[-1], a, wq, sa, sb)
    packed = [ops.quant_weight_blocks(w) for w in ws]
    held, held_s = torch.empty_like(packed[0][0]), torch.empty_like(packed[0][1])
    torch.cuda.synchronize()
    for i in range(40):
        wq, sb = ops.quant_weight_blocks(ws[i % 4])
        y = ops.fp8_gemm_blocks(a, wq, sa, sb)
        del wq, sb
        held.view(torch.uint8).copy_(packed[(i + 1) % 4][0].view(torch.uint8))
        held_s.copy_(packed[(i + 1) % 4][1])
        z = ops.fp8_gemm_blocks(a, held, sa, held_s)
        assert torch.equal(y, want[i % 4]) and torch.equal(z, want[(i + 1) % 4])


def test_two_streams_at_once(dev):
    a, w, sa, sb = operands(40, 1024, 2048, seed=3)
    b, v, sc, sd = operands(500, 1024, 2048, seed=4)
    want = ops.fp8_gemm_blocks(a, w, sa, sb), ops.fp8_gemm_blocks(b, v, sc, sd)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        with torch.cuda.stream(streams[0]):
            got[0].append(ops.fp8_gemm_blocks(a, w, sa, sb))
        with torch.cuda.stream(streams[1]):
            got[1].append(ops.fp8_gemm_blocks(b, v, sc, sd))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[0]) for y in got[0]) and all(torch.equal(y, want[1]) for y in got[1])


def test_threads_and_other_kernels_at_once(dev):
    """Four host threads with a stream each: products of every form beside the per-token product and the attention."""
    import threading

    shapes = [(3, 1024, 2048), (40, 5120, 1024), (300, 9000, 512), (200, 5128, 2048)]
    jobs = []
    for m, n, k in shapes:
        x = torch.randn(m, k, device=dev, generator=gen(m)).to(BF16)
        w = ops.quant_weight_blocks((torch.randn(n, k, device=dev, generator=gen(n)) * 0.02).to(BF16))
        q, s = ops.quant_blocks(x)
        jobs.append((x, w, ops.fp8_gemm_blocks(q, w[0], s, w[1])))
    a8 = torch.randn(512, 512, device=dev, generator=gen(1)).to(E4M3)
    one = torch.ones(512, device=dev)
    want8 = ops.fp8_gemm(a8, a8, one, one)
    qkv = torch.randn(3, 512, 4, 128, device=dev, generator=gen(2)).to(BF16)
    want_o = ops.flash_attn(qkv[0], qkv[1], qkv[2])
    torch.cuda.synchronize()
    wrong = []

    def work(job):
        x, w, want = job
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                q, s = ops.quant_blocks(x)
                y = ops.fp8_gemm_blocks(q, w[0], s, w[1])
                y8 = ops.fp8_gemm(a8, a8, one, one)
                o = ops.flash_attn(qkv[0], qkv[1], qkv[2])
                torch.cuda.current_stream().synchronize()
                if not (torch.equal(y, want) and torch.equal(y8, want8) and torch.equal(o, want_o)):
                    wrong.append(x.shape)

    threads = [threading.Thread(target=work, args=(j,)) for j in jobs]
    for th in threads:
        th.start()
    for th in threads:
        th.join(60)
    assert not wrong and not any(th.is_alive() for th in threads)
    assert ops.device_status() == 0


def test_torch_ops(dev):
    x = torch.randn(20, 512, device=dev, generator=gen(1)).to(BF16)
    q, s = torch.ops.h3b.quant_blocks(x)
    w, sw = torch.ops.h3b.quant_weight_blocks((torch.randn(2, 256, 512, device=dev, generator=gen(2))).to(BF16))
    off = bounds([15, 5])
    y = torch.ops.h3b.fp8_gemm_grouped(q, w, s, sw, off, BF16)
    out = torch.empty_like(y)
    torch.ops.h3b.fp8_gemm_grouped_out(q, w, s, sw, off, out)
    assert torch.equal(out, y)
    d = torch.ops.h3b.fp8_gemm_blocks(q, w[0], s, sw[0], None, BF16)
    torch.ops.h3b.fp8_gemm_blocks_out(q, w[0], s, sw[0], None, out)
    assert torch.equal(out, d) and torch.equal(d[:15], y[:15])
    assert torch.ops.h3b.silu_mul_quant_blocks(y)[0].shape == (20, 128)
