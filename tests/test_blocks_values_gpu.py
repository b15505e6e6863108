"""Block quant of silu(gate) * up against 64 bits where fp32 runs out: far negative gates and large ups.

Bounds.  silu(g) * u within (5 + 0.75 |g|) * 2^-23 of its size, as the kernel states, and half an fp32 subnormal step for results
below the normal range.  A scale is a quotient by 448, rounded (2^-24); a code is a product by a rounded inverse, two roundings
of 2^-24 ahead of e4m3's."""
import pytest
import torch
from test_blocks_gpu import B, half_step_e4m3, nb, spread

from h3b import ops

BF16 = torch.bfloat16
pytestmark = pytest.mark.gpu


def check(q, s, x):
    m, f = x.shape[0], x.shape[1] // 2
    g, u = x[:, :f].double(), x[:, f:].double()
    h = g * torch.sigmoid(g) * u
    err = h.abs() * (5 + 0.75 * g.abs()) * 2.0 ** -23 + 2.0 ** -150
    pad = (0, nb(f) * B - f)
    amax, amax_err = (torch.nn.functional.pad(t, pad).view(m, -1, B).amax(-1) for t in (h.abs(), err))
    ref = (amax / 448).clamp_min(1.0 / (448.0 * 512.0))
    assert float(((s.double() - ref).abs() - (amax_err / 448 + ref * 2.0 ** -24) * (1 + 2.0 ** -20)).max()) <= 0
    full = spread(s.double(), f, 1)
    v = h / full
    over = (v.abs() - 448).clamp_min(0)       # a maximum whose scale came out small by its error: cut at 448
    assert float(((q.double() - v).abs() - half_step_e4m3(v.clamp(-448, 448)) * (1 + 2.0 ** -18) - err / full * (1 + 2.0 ** -20)
                  - over).max()) <= 0


@pytest.mark.parametrize("m,f,gain", [(1, 128, 1.0), (3, 100, 1.0), (17, 13824, 1.5), (40, 136, 30.0), (5, 77, 4.0),
                                      (300, 1000, 60.0)])
def test_silu_within_the_stated_bound(dev, m, f, gain):
    g = torch.Generator(device=dev).manual_seed(f)
    x = (torch.randn(m, 2 * f, device=dev, generator=g) * gain).to(BF16)
    check(*ops.silu_mul_quant_blocks(x), x)


GATES = [-60.0, -86.0, -86.5, -87.0, -87.5, -88.0, -88.5, -89.0, -92.0, -100.0, -103.5, -104.0, -110.0, -120.0, -131.0, -140.0,
         -200.0, -1000.0]


@pytest.mark.parametrize("f", [1024, 1032, 1025])     # every way that values move
def test_silu_of_far_negative_gates(dev, f):
    """exp(-g) or its reciprocal leaves fp32 from g = -87.5 on, but the product with a large up is well within it."""
    g = torch.Generator(device=dev).manual_seed(f)
    x = torch.empty(len(GATES), 2 * f, device=dev, dtype=BF16)
    x[:, :f] = torch.tensor(GATES, device=dev, dtype=BF16)[:, None]
    sign = torch.where(torch.rand(len(GATES), f, device=dev, generator=g) < 0.5, -1.0, 1.0)
    size = torch.tensor([3e38, 1e38, 1e37, 1e35, 1e32, 1e28, 1e10, 1.0, 1.0], device=dev).repeat_interleave(B)[:f]
    x[:, f:] = (sign * size * torch.rand(len(GATES), f, device=dev, generator=g)).to(BF16)
    q, s = ops.silu_mul_quant_blocks(x)
    check(q, s, x)
    assert bool((s[:9, 0] > 1e-5).all()) and bool((q[:12, :128].float() != 0).any(1).all())      # nothing was flushed
    mixed = x.clone()                                 # and among ordinary gates
    mixed[:, 1:f:2] = torch.randn(len(GATES), f // 2, device=dev, generator=g).to(BF16)
    mixed[:, f:] = mixed[:, f:].float().clamp(-1e36, 1e36).to(BF16)
    check(*ops.silu_mul_quant_blocks(mixed), mixed)
