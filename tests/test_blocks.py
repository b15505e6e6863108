"""The block-scaled FP8 operators without a GPU: what the tensor wrappers and the C entry points refuse before a launch,
and the shapes and strides of the ops' fake kernels."""
import pytest
import torch

from h3b import _lib, ops

BF16, F16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


@pytest.fixture
def calls(monkeypatch):
    made = []
    monkeypatch.setattr(ops, "_need_cuda", lambda *ts: None)
    monkeypatch.setattr(ops, "_stream", lambda t: 0)
    monkeypatch.setattr(_lib, "call", lambda name, *a: made.append((name, a)))
    return made


def refused(calls, exc, fn, match=None):
    n = len(calls)
    with pytest.raises(exc, match=match):
        fn()
    assert len(calls) == n, "a refused call reached the library"


def operands(m=5, n=200, k=272, e=None, ks=None):
    kb = -(-k // 128) if ks is None else ks
    lead = () if e is None else (e,)
    return (torch.zeros(m, k).to(E4M3), torch.zeros(*lead, n, k).to(E4M3), torch.ones(m, kb),
            torch.ones(*lead, -(-n // 128), kb))


def test_cpu_tensors_raise():
    x = torch.zeros(4, 128, dtype=BF16)
    a, w, sa, sb = operands()
    for fn in (lambda: ops.quant_blocks(x), lambda: ops.silu_mul_quant_blocks(x), lambda: ops.quant_weight_blocks(x),
               lambda: ops.fp8_gemm_blocks(a, w, sa, sb),
               lambda: ops.fp8_gemm_grouped(a, w[None], sa, sb[None], torch.tensor([0, 5]))):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            fn()


def test_quantisers(calls):
    x = torch.zeros(6, 512, dtype=BF16)
    for fn in (ops.quant_blocks, ops.silu_mul_quant_blocks, ops.quant_weight_blocks):
        refused(calls, TypeError, lambda fn=fn: fn(x.float()), "dtype")
        refused(calls, ValueError, lambda fn=fn: fn(x.t()), "unit innermost")
        refused(calls, ValueError, lambda fn=fn: fn(x[0]))
    refused(calls, ValueError, lambda: ops.quant_blocks(x[None]), "dimensions")
    refused(calls, ValueError, lambda: ops.silu_mul_quant_blocks(x[:, :511]), "2F")
    refused(calls, ValueError, lambda: ops.quant_weight_blocks(x[None, None]))
    q, s = ops.quant_blocks(x[:, :300])
    assert q.shape == (6, 300) and s.shape == (6, 3) and s.stride() == (1, 8)
    q, s = ops.silu_mul_quant_blocks(x)
    assert q.shape == (6, 256) and s.shape == (6, 2)
    q, s = ops.quant_weight_blocks(x)
    assert s.shape == (1, 4)
    q, s = ops.quant_weight_blocks(torch.zeros(3, 130, 129, dtype=BF16))
    assert q.shape == (3, 130, 129) and s.shape == (3, 2, 2)
    assert [c[0] for c in calls] == ["h3b_quant_blocks_e4m3", "h3b_silu_mul_quant_blocks_e4m3"] + \
        ["h3b_quant_weight_blocks_e4m3"] * 2


@pytest.mark.parametrize("e", [None, 3])
def test_products(calls, e):
    a, w, sa, sb = operands(e=e)
    off = torch.tensor([0, 1, 2, 5], dtype=torch.int32)

    def run(a=a, w=w, sa=sa, sb=sb, off=off, **kw):
        if e is None:
            return ops.fp8_gemm_blocks(a, w, sa, sb, **kw)
        return ops.fp8_gemm_grouped(a, w, sa, sb, off, **kw)

    refused(calls, TypeError, lambda: run(a=a.float()), "dtype")
    refused(calls, TypeError, lambda: run(w=w.float()), "dtype")
    refused(calls, TypeError, lambda: run(sa=sa.double()), "fp32")
    refused(calls, TypeError, lambda: run(sb=sb.to(BF16)), "fp32")
    refused(calls, ValueError, lambda: run(a=a[:, :256]), "same K")
    refused(calls, ValueError, lambda: run(a=a[:, :264], w=w[..., :264]), "multiple of 16")
    refused(calls, ValueError, lambda: run(a=a[:, :0], w=w[..., :0]))
    refused(calls, ValueError, lambda: run(sa=sa[:4]), "sa must be")
    refused(calls, ValueError, lambda: run(sa=sa[:, :2]), "sa must be")
    refused(calls, ValueError, lambda: run(sb=sb[..., :1, :]), "sb")
    refused(calls, ValueError, lambda: run(w=w[..., None]), "dimensions")
    refused(calls, ValueError, lambda: run(w=w.transpose(-1, -2).contiguous().transpose(-1, -2)), "unit innermost")
    refused(calls, TypeError, lambda: run(out_dtype=torch.float32), "out_dtype")
    refused(calls, TypeError, lambda: run(out=torch.empty(5, 200)), "dtype")
    refused(calls, ValueError, lambda: run(out=torch.empty(5, 199, dtype=BF16)), "out must be")
    refused(calls, ValueError, lambda: run(out=torch.empty(200, 5, dtype=BF16).t()), "out must be")
    refused(calls, ValueError, lambda: run(out=torch.empty(1, 200, dtype=BF16).expand(5, 200)), "overlap")
    assert run().dtype == BF16 and run(out_dtype=F16).shape == (5, 200)
    out = torch.empty(5, 256, dtype=F16)[:, 3:203]
    assert run(out=out) is out
    assert run(a=a[:1], sa=sa[:1], off=off.clamp_max(1)).shape == (1, 200)
    assert calls[-1][1][1] == 272                       # a single row's stride is its length
    assert {c[0] for c in calls} == {"h3b_fp8_gemm_blocks" if e is None else "h3b_fp8_gemm_grouped"}


def test_bias_and_offsets(calls):
    a, w, sa, sb = operands()
    refused(calls, TypeError, lambda: ops.fp8_gemm_blocks(a, w, sa, sb, torch.zeros(200)), "bias")
    refused(calls, ValueError, lambda: ops.fp8_gemm_blocks(a, w, sa, sb, torch.zeros(100, dtype=BF16)), "bias")
    a, w, sa, sb = operands(e=3)
    refused(calls, TypeError, lambda: ops.fp8_gemm_grouped(a, w, sa, sb, torch.zeros(4)), "offsets")
    refused(calls, ValueError, lambda: ops.fp8_gemm_grouped(a, w, sa, sb, torch.tensor([0, 1, 2])), "offsets")
    refused(calls, ValueError, lambda: ops.fp8_gemm_grouped(a, w, sa, sb, torch.tensor([[0, 1, 2, 5]])), "offsets")
    ops.fp8_gemm_grouped(a, w, sa, sb, torch.tensor([0, 1, 2, 5]))
    assert calls[-1][1][13] == 1                        # int64 bounds are read as such


def test_tensors_on_two_devices_are_refused(calls):
    a, w, sa, sb = operands()
    refused(calls, ValueError, lambda: ops.fp8_gemm_blocks(a, w, sa.to("meta"), sb), "tensors on")
    refused(calls, ValueError, lambda: ops.fp8_gemm_blocks(a, w, sa, sb, out=torch.empty(5, 200, dtype=BF16,
                                                                                          device="meta")), "tensors on")


def test_fake_kernels():
    m = lambda *s, dt=BF16: torch.empty(s, dtype=dt, device="meta")  # noqa: E731
    for rows in (1, 6, 300):
        q, s = torch.ops.h3b.quant_blocks(m(rows, 300))
        real = ops._quant_outputs(rows, 300, torch.device("cpu"))[1]
        assert q.shape == (rows, 300) and q.dtype == E4M3 and s.shape == real.shape and s.stride() == real.stride()
    q, s = torch.ops.h3b.silu_mul_quant_blocks(m(6, 600))
    assert q.shape == (6, 300) and s.shape == (6, 3)
    q, s = torch.ops.h3b.quant_weight_blocks(m(4, 200, 300))
    assert q.shape == (4, 200, 300) and s.shape == (4, 2, 3) and s.dtype == torch.float32
    a, w, f = m(6, 256, dt=E4M3), m(200, 256, dt=E4M3), torch.float32
    assert torch.ops.h3b.fp8_gemm_blocks(a, w, m(6, 2, dt=f), m(2, 2, dt=f), None, F16).dtype == F16
    y = torch.ops.h3b.fp8_gemm_grouped(a, m(3, 200, 256, dt=E4M3), m(6, 2, dt=f), m(3, 2, 2, dt=f),
                                       m(4, dt=torch.int32), BF16)
    assert y.shape == (6, 200) and y.dtype == BF16
    out = m(6, 200)
    assert torch.ops.h3b.fp8_gemm_blocks_out(a, w, m(6, 2, dt=f), m(2, 2, dt=f), None, out) is None


def _gemm(L, a=16, lda=32, w=16, ldw=32, sa=16, sar=1, sab=1, sb=16, sbr=1, sbb=1, y=16, ldy=64, m=4, n=64, k=32, dt=0):
    return L.h3b_fp8_gemm_blocks(a, lda, w, ldw, sa, sar, sab, sb, sbr, sbb, None, y, ldy, m, n, k, dt, None)


def _grouped(L, a=16, lda=32, w=16, wexp=2048, ldw=32, off=16, rows=4, e=2, n=64, k=32, ldy=64, sbe=1):
    return L.h3b_fp8_gemm_grouped(a, lda, w, wexp, ldw, 16, 1, 1, 16, sbe, 1, 1, off, 0, 16, ldy, rows, e, n, k, 0, None)


EINVAL, EALIGN, EUNSUPPORTED = _lib.H3B_EINVAL, _lib.H3B_EALIGN, _lib.H3B_EUNSUPPORTED


@pytest.mark.parametrize("call,status", [
    (lambda L: L.h3b_quant_blocks_e4m3(16, -1, 8, 8, 16, 16, 1, 1, 0, None), EINVAL),
    (lambda L: L.h3b_quant_blocks_e4m3(16, 1, 8, 8, 16, 16, 1, 1, 2, None), EINVAL),
    (lambda L: L.h3b_quant_blocks_e4m3(None, 1, 8, 8, 16, 16, 1, 1, 0, None), EINVAL),
    (lambda L: L.h3b_quant_blocks_e4m3(16, 1, 8, -8, 16, 16, 1, 1, 0, None), EINVAL),
    (lambda L: L.h3b_quant_blocks_e4m3(None, 0, 8, 8, None, None, 1, 1, 0, None), _lib.H3B_OK),
    (lambda L: L.h3b_quant_blocks_e4m3(16, 1 << 31, 8, 8, 16, 16, 1, 1, 0, None), EUNSUPPORTED),
    (lambda L: L.h3b_silu_mul_quant_blocks_e4m3(16, 1, -8, 8, 16, 16, 1, 1, 0, None), EINVAL),
    (lambda L: L.h3b_quant_weight_blocks_e4m3(16, 1, 8, -1, 0, 8, 16, 16, 0, None), EINVAL),
    (lambda L: L.h3b_quant_weight_blocks_e4m3(16, 1, 8, 8, 0, 8, None, 16, 0, None), EINVAL),
    (lambda L: L.h3b_quant_weight_blocks_e4m3(16, 1 << 31, 8, 8, 0, 8, 16, 16, 0, None), EUNSUPPORTED),
    (lambda L: L.h3b_quant_weight_blocks_e4m3(None, 0, 8, 8, 0, 8, None, None, 0, None), _lib.H3B_OK),
    (lambda L: _gemm(L, m=-1), EINVAL), (lambda L: _gemm(L, n=0), EINVAL), (lambda L: _gemm(L, k=0), EINVAL),
    (lambda L: _gemm(L, m=0, a=None), _lib.H3B_OK), (lambda L: _gemm(L, a=None), EINVAL),
    (lambda L: _gemm(L, sb=None), EINVAL), (lambda L: _gemm(L, y=None), EINVAL), (lambda L: _gemm(L, dt=2), EINVAL),
    (lambda L: _gemm(L, k=24), EUNSUPPORTED), (lambda L: _gemm(L, lda=16), EALIGN), (lambda L: _gemm(L, ldw=40), EALIGN),
    (lambda L: _gemm(L, a=24), EALIGN), (lambda L: _gemm(L, w=8), EALIGN), (lambda L: _gemm(L, ldy=63), EINVAL),
    (lambda L: _gemm(L, sar=-1), EINVAL), (lambda L: _gemm(L, m=1 << 31), EUNSUPPORTED),
    (lambda L: _grouped(L, e=0), EINVAL), (lambda L: _grouped(L, off=None), EINVAL),
    (lambda L: _grouped(L, rows=0, off=None), _lib.H3B_OK), (lambda L: _grouped(L, wexp=0), EINVAL),
    (lambda L: _grouped(L, wexp=2056), EALIGN), (lambda L: _grouped(L, sbe=-1), EINVAL),
])
def test_c_entry_points_refuse_before_any_launch(call, status):
    lib = _lib.load()
    assert call(lib) == status
    if status != _lib.H3B_OK:
        assert lib.h3b_last_error()
