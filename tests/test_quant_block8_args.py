"""Refusals of the block-scaled FP8 operators: at the C entries (before any CUDA call, so they run without a GPU; the addresses are
never touched) and at the Python functions."""
import pytest
import torch

A = 1 << 20          # a 16-byte aligned address that is not looked at


@pytest.fixture(scope="module")
def L():
    from gigaslop_b200 import build, lib
    build.build()
    return lib()


def quant(L, x=A, dt=0, ldx=256, q=A, ldq=256, s=A, lds=2, M=4, K=256, rows=1):
    return L.gsb200_block_quantize_fp8(x, dt, ldx, q, ldq, s, lds, M, K, rows, None)


@pytest.mark.parametrize("bad", [dict(x=None), dict(q=None), dict(s=None), dict(dt=3), dict(dt=-1), dict(ldx=255), dict(ldq=255), dict(lds=1), dict(M=-1), dict(K=0),
                                 dict(K=-5), dict(rows=2), dict(rows=0), dict(rows=64), dict(x=A + 1), dict(s=A + 2), dict(K=2 ** 30 + 1, ldx=2 ** 31, ldq=2 ** 31, lds=2 ** 30)])
def test_quantize_refuses(L, bad):
    assert quant(L, **bad) == -1


def test_nothing_to_do_is_no_error(L):
    assert quant(L, M=0, x=None, q=None, s=None) == 0
    assert gemm(L, M=0, a=None, c=None) == 0


def dequant(L, q=A, ldq=256, s=A, lds=2, x=A, dt=0, ldx=256, M=4, K=256, rows=1):
    return L.gsb200_block_dequantize_fp8(q, ldq, s, lds, x, dt, ldx, M, K, rows, None)


@pytest.mark.parametrize("bad", [dict(x=None), dict(q=None), dict(s=None), dict(dt=7), dict(ldx=255), dict(ldq=255), dict(lds=1), dict(M=-1), dict(K=0), dict(rows=3), dict(x=A + 1)])
def test_dequantize_refuses(L, bad):
    assert dequant(L, **bad) == -1


def gemm(L, a=A, lda=256, sa=A, ldsa=2, b=A, ldb=256, sb=A, ldsb=2, c=A, ldc=64, ct=0, M=4, N=64, K=256, flags=0):
    return L.gsb200_gemm_fp8_block(a, lda, sa, ldsa, b, ldb, sb, ldsb, c, ldc, ct, M, N, K, flags, None)


@pytest.mark.parametrize("bad", [dict(a=None), dict(sa=None), dict(b=None), dict(sb=None), dict(c=None), dict(a=A + 8), dict(b=A + 1), dict(lda=264), dict(ldb=264), dict(lda=240),
                                 dict(ldb=240), dict(ldc=63), dict(ct=3), dict(ct=1, c=A + 2), dict(c=A + 1), dict(ldsa=1), dict(ldsb=1), dict(sa=A + 1), dict(sb=A + 2), dict(M=-1),
                                 dict(N=0), dict(K=0), dict(N=-4), dict(flags=1), dict(flags=4), dict(flags=16, ldb=48), dict(flags=16, N=300, ldb=304, ldc=300, ldsb=2),
                                 dict(M=2 ** 31)])
def test_gemm_refuses(L, bad):
    assert gemm(L, **bad) == -1


def wgrad(L, dy=A, dt=0, lddy=64, q=A, ldq=256, s=A, lds=2, dw=A, lddw=256, acc=0, ws=A, wsb=1 << 40, M=100, N=64, K=256):
    return L.gsb200_gemm_fp8_block_wgrad(dy, dt, lddy, q, ldq, s, lds, dw, lddw, acc, ws, wsb, M, N, K, None)


@pytest.mark.parametrize("bad", [dict(dy=None), dict(q=None), dict(s=None), dict(dw=None), dict(dt=1), dict(dt=5), dict(dy=A + 8), dict(q=A + 8), dict(lddy=56), dict(lddy=68),
                                 dict(ldq=264), dict(ldq=240), dict(lds=1), dict(lddw=255), dict(dw=A + 2), dict(s=A + 1), dict(M=-1), dict(N=0), dict(K=0)])
def test_wgrad_refuses(L, bad):
    assert wgrad(L, **bad) == -1


def test_wgrad_workspace(L):
    f = L.gsb200_gemm_fp8_block_wgrad_workspace_bytes
    assert f(64, 64, 64) == 0 and f(-1, 64, 64) == 0 and f(64, 0, 64) == 0 and f(0, 64, 64) == 0
    need = f(65536, 512, 512)
    assert need > 0 and need % (512 * 512 * 4) == 0
    assert f(65536, 512, 512) == need


def swiglu(L, g=A, ldg=256, u=A, ldu=256, dt=0, out=(A,) * 6, ldq=256, lds=2, M=4, F=256):
    return L.gsb200_swiglu_fp8_block(g, ldg, u, ldu, dt, *out, ldq, lds, M, F, None)


@pytest.mark.parametrize("bad", [dict(g=None), dict(u=None), dict(dt=3), dict(ldg=255), dict(ldu=255), dict(ldq=255), dict(lds=1), dict(M=-1), dict(F=0), dict(g=A + 1), dict(u=A + 1)]
                         + [dict(out=tuple(None if i == j else A for j in range(6))) for i in range(6)])
def test_swiglu_refuses(L, bad):
    assert swiglu(L, **bad) == -1


def bwd(L, dh=A, dt=0, lddh=256, gq=A, ldgq=256, gs=A, ldgs=2, uq=A, lduq=256, us=A, ldus=2, dg=A, lddg=256, du=A, lddu=256, out=(None,) * 4, ldq=0, lds=0, M=4, F=256):
    return L.gsb200_swiglu_fp8_block_bwd(dh, dt, lddh, gq, ldgq, gs, ldgs, uq, lduq, us, ldus, dg, lddg, du, lddu, *out, ldq, lds, M, F, None)


@pytest.mark.parametrize("bad", [dict(dh=None), dict(gq=None), dict(gs=None), dict(uq=None), dict(us=None), dict(dg=None), dict(du=None), dict(dt=4), dict(lddh=255), dict(ldgq=255),
                                 dict(lduq=255), dict(ldgs=1), dict(ldus=1), dict(lddg=255), dict(lddu=255), dict(F=0), dict(M=-2), dict(dh=A + 1),
                                 dict(out=(A, A, A, None), ldq=256, lds=2), dict(out=(A,) * 4, ldq=255, lds=2), dict(out=(A,) * 4, ldq=256, lds=1), dict(out=(A, A + 1, A, A), ldq=256, lds=2)])
def test_swiglu_bwd_refuses(L, bad):
    assert bwd(L, **bad) == -1


def test_cpu_tensors_are_refused():
    import gigaslop_b200 as g
    x, s = torch.zeros(4, 128), torch.ones(4, 1)
    q = x.to(torch.float8_e4m3fn)
    for call in (lambda: g.fp8_block_quantize(x), lambda: g.fp8_block_dequantize(q, s), lambda: g.gemm_fp8_block(q, q, s, s[:1]), lambda: g.gemm_fp8_block_wgrad(x.half(), q, s),
                 lambda: g.swiglu_fp8_block(x, x), lambda: g.swiglu_fp8_block_bwd(x, q, s, q, s)):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()


@pytest.mark.gpu
def test_python_refusals():
    import gigaslop_b200 as g
    z = lambda *sh, dt=torch.float16: torch.zeros(*sh, dtype=dt, device="cuda")
    f8 = torch.float8_e4m3fn
    q, s, w, sw = z(40, 256, dt=torch.uint8).view(f8), z(40, 2, dt=torch.float32), z(64, 256, dt=torch.uint8).view(f8), z(1, 2, dt=torch.float32)
    x, dy = z(40, 256), z(40, 64)
    bad = [
        (TypeError, lambda: g.fp8_block_quantize(x.to(torch.int32))), (TypeError, lambda: g.fp8_block_quantize(x.double())), (ValueError, lambda: g.fp8_block_quantize(x.view(-1))),
        (ValueError, lambda: g.fp8_block_quantize(x.t())), (ValueError, lambda: g.fp8_block_quantize(x, rows=64)), (ValueError, lambda: g.fp8_block_quantize(x, out=q[:, :255])),
        (ValueError, lambda: g.fp8_block_quantize(x, out_scale=s[:, :1])), (TypeError, lambda: g.fp8_block_quantize(x, out_scale=s.double())),
        (ValueError, lambda: g.fp8_block_quantize(x[:1].expand(40, 256))),
        (ValueError, lambda: g.fp8_block_dequantize(q, s[:, :1])), (ValueError, lambda: g.fp8_block_dequantize(q, s, rows=128)), (TypeError, lambda: g.fp8_block_dequantize(q, s, dtype=torch.int8)),
        (TypeError, lambda: g.fp8_block_dequantize(x, s)), (ValueError, lambda: g.fp8_block_dequantize(q, s, out=x[:39])),
        (ValueError, lambda: g.gemm_fp8_block(q, w[:, :240], s, sw)), (ValueError, lambda: g.gemm_fp8_block(q, w, s[:, :1], sw)), (ValueError, lambda: g.gemm_fp8_block(q, w, s, sw.t())),
        (ValueError, lambda: g.gemm_fp8_block(q, w, s, sw, b_transposed=True)), (TypeError, lambda: g.gemm_fp8_block(x, w, s, sw)), (TypeError, lambda: g.gemm_fp8_block(q, w, s, sw, dtype=torch.int32)),
        (ValueError, lambda: g.gemm_fp8_block(q, w, s, sw, out=dy[:39])), (TypeError, lambda: g.gemm_fp8_block(q, w, s.half(), sw)),
        (RuntimeError, lambda: g.gemm_fp8_block(q[:, :250].contiguous(), w[:, :250], s, sw)),             # rows that TMA cannot address
        (RuntimeError, lambda: g.gemm_fp8_block(q[:, 1:129], w[:, :128], s[:, :1], sw[:, :1])),
        (TypeError, lambda: g.gemm_fp8_block_wgrad(dy.float(), q, s)), (ValueError, lambda: g.gemm_fp8_block_wgrad(dy[:39], q, s)), (ValueError, lambda: g.gemm_fp8_block_wgrad(dy, q, s, accumulate=True)),
        (TypeError, lambda: g.gemm_fp8_block_wgrad(dy, q, s, out=z(64, 256))), (ValueError, lambda: g.gemm_fp8_block_wgrad(dy, q, s, out=z(64, 255, dt=torch.float32))),
        (RuntimeError, lambda: g.gemm_fp8_block_wgrad(z(40, 63), q, s)),
        (ValueError, lambda: g.swiglu_fp8_block(x, x[:, :255])), (TypeError, lambda: g.swiglu_fp8_block(x, x.float())),
        (ValueError, lambda: g.swiglu_fp8_block(x.t(), x.t())),
        (ValueError, lambda: g.swiglu_fp8_block_bwd(x, q[:39], s[:39], q, s)), (ValueError, lambda: g.swiglu_fp8_block_bwd(x, q, s[:, :1], q, s)), (TypeError, lambda: g.swiglu_fp8_block_bwd(x, x, s, q, s)),
    ]
    for i, (err, call) in enumerate(bad):
        with pytest.raises(err):
            call()
            pytest.fail(f"call {i} was not refused")
    torch.cuda.synchronize()
