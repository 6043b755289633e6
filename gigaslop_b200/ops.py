"""PyTorch-facing host functions over the C ABI.  torch supplies device memory
and streams; every byte of compute happens in libgigaslop_b200.so.

Function names and argument meaning follow the reference's host helpers
(``quantize_tensor``, ``fp8_quantize_per_token``) and kernels.

An operator that has a ``_checked_*`` function first offers the call to the native path (``_lib.native``, csrc/binding.cpp),
which takes it when every argument is a plain CUDA tensor of the current device that passes the operator's checks, and
answers None otherwise; then the ``_checked_*`` function decides: it raises what is wrong with the arguments, or makes the
call through ctypes.  The others (``gemm_i8_i32``, ``gemm_f16``, ``quantize_gemm_i8_rotary``) go through ctypes always.
"""
import functools

import torch

from . import _lib
from ._lib import check, lib


def _stream(t=None):
    """Current stream of ``t``'s device (of the current device without ``t``: inside an ``@_on_device`` function
    that is the tensors' device)."""
    return torch.cuda.current_stream(t.device if t is not None else None).cuda_stream


def same_device(*ts):
    """The one device all given tensors live on.  CPU tensors raise (there is no CPU path); tensors spread over
    several devices raise (the library launches on one device and would reach the others through peer pointers,
    with the wrong device's kernel attributes, SM count and static scratch)."""
    dev = None
    for t in ts:
        if t is None:
            continue
        if t.device.type != "cuda":
            raise RuntimeError("gigaslop_b200 operates on CUDA tensors only (no CPU fallback)")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError(f"all tensors of one call must live on one device (got {dev} and {t.device})")
    return dev


_need_cuda = same_device


def _on_device(fn):
    """Run ``fn`` with the device of its tensor arguments current: the C side keys its per-device state on the
    current device, and ``_stream()`` then returns that device's current stream."""
    @functools.wraps(fn)
    def wrapped(*args, **kwargs):
        dev = same_device(*[a for a in args if isinstance(a, torch.Tensor)],
                          *[a for a in kwargs.values() if isinstance(a, torch.Tensor)])
        if dev is None or dev.index == torch.cuda.current_device():      # the common case costs no context switch
            return fn(*args, **kwargs)
        with torch.cuda.device(dev):
            return fn(*args, **kwargs)
    return wrapped


def _rowmajor(t, name):
    if t.dim() != 2 or t.stride(1) != 1:
        raise ValueError(f"{name} must be 2-D with unit inner stride")
    return t


def _dt(t):
    if t.dtype == torch.float16:
        return _lib.F16
    if t.dtype == torch.float32:
        return _lib.F32
    raise TypeError("activations must be float16 or float32")


def quantize_tensor(t, dim=-1, out=None, out_scale=None):
    """Per-row symmetric absmax INT8 quantiser; same contract as the reference's
    ``quantize_tensor`` (cute/bench_quant_i8.py:15-31): returns (int8 [M,K], fp32 dequant scale [M])."""
    n = _lib.native
    if n is not None and (dim == -1 or dim == 1):
        r = n.quantize(0, t, out, out_scale)
        if r is not None:
            return r
    return _checked_quantize_tensor(t, dim, out, out_scale)


@_on_device
def _checked_quantize_tensor(t, dim, out, out_scale):
    if dim not in (-1, t.dim() - 1):
        raise ValueError("only per-row (last-dim) quantisation is on the hot path")
    _need_cuda(t)
    x = _rowmajor(t, "t")
    M, K = x.shape
    q = out if out is not None else torch.empty((M, K), dtype=torch.int8, device=x.device)
    s = out_scale if out_scale is not None else torch.empty((M,), dtype=torch.float32, device=x.device)
    check(lib().gsb200_ptq_int8(x.data_ptr(), _dt(x), x.stride(0), q.data_ptr(), q.stride(0), s.data_ptr(),
                                M, K, _stream()), "quantize_tensor")
    return q, s


def fp8_quantize_per_token(x, torch_formulation=True, out=None, out_scale=None):
    """Per-row E4M3 quantiser (fly/rdna_fp8_preshuffle_gemm.py:57-70); ``torch_formulation=False``
    selects the device-kernel arithmetic of fly/rdna_fp8_per_token_quantize.py."""
    n = _lib.native
    if n is not None:
        r = n.quantize(2 if torch_formulation else 1, x, out, out_scale)
        if r is not None:
            return r
    return _checked_fp8_quantize_per_token(x, torch_formulation, out, out_scale)


@_on_device
def _checked_fp8_quantize_per_token(x, torch_formulation, out, out_scale):
    _need_cuda(x)
    x = _rowmajor(x, "x")
    M, K = x.shape
    q = out if out is not None else torch.empty((M, K), dtype=torch.float8_e4m3fn, device=x.device)
    s = out_scale if out_scale is not None else torch.empty((M,), dtype=torch.float32, device=x.device)
    check(lib().gsb200_ptq_fp8(x.data_ptr(), _dt(x), x.stride(0), q.data_ptr(), q.stride(0), s.data_ptr(),
                               M, K, 1 if torch_formulation else 0, _stream()), "fp8_quantize_per_token")
    return q, s


def _check_ab(A, B, dtypes):
    _need_cuda(A, B)
    _rowmajor(A, "A"); _rowmajor(B, "B")
    if A.dtype not in dtypes or B.dtype not in dtypes:
        raise TypeError(f"operands must be one of {dtypes}")
    if A.shape[1] != B.shape[1]:
        raise ValueError("A is [M,K], B is [N,K]: K mismatch")
    return A.shape[0], B.shape[0], A.shape[1]


_I8 = (torch.int8,)
_F8 = (torch.float8_e4m3fn, torch.uint8)


@_on_device
def gemm_i8_i32(A, B, out=None):
    """Exact int32 ``A[M,K] . B[N,K]^T`` (cute/ampere_gemm_i8.py TensorOpGemmI8, int32 output)."""
    M, N, K = _check_ab(A, B, _I8)
    C = out if out is not None else torch.empty((M, N), dtype=torch.int32, device=A.device)
    check(lib().gsb200_gemm_i8_i32(A.data_ptr(), A.stride(0), B.data_ptr(), B.stride(0), C.data_ptr(), C.stride(0),
                                   M, N, K, _stream()), "gemm_i8_i32")
    return C


def _gemm_f16(fn, name, A, B, scale_a, scale_b, out, flags, dtypes):
    M, N, K = _check_ab(A, B, dtypes)
    _need_cuda(scale_a, scale_b)
    C = out if out is not None else torch.empty((M, N), dtype=torch.float16, device=A.device)
    check(fn(A.data_ptr(), A.stride(0), B.data_ptr(), B.stride(0), C.data_ptr(), C.stride(0),
             scale_a.data_ptr(), scale_b.data_ptr(), M, N, K, flags, _stream()), name)
    return C


def gemm_i8(A, B, scale_a, scale_b, out=None, flags=0):
    """W8A8 GEMM with per-token x per-channel dequant to fp16 (cute/ampere_gemm_i8_quant_rmem.py)."""
    n = _lib.native
    if n is not None:
        r = n.gemm(0, A, B, scale_a, scale_b, out, flags)
        if r is not None:
            return r
    return _checked_gemm_i8(A, B, scale_a, scale_b, out, flags)


@_on_device
def _checked_gemm_i8(A, B, scale_a, scale_b, out, flags):
    return _gemm_f16(lib().gsb200_gemm_i8_f16, "gemm_i8", A, B, scale_a, scale_b, out, flags, _I8)


def gemm_fp8(A, B, scale_a, scale_b, out=None, flags=0):
    """FP8 GEMM, ``B`` K-major ``[N,K]`` (fly/rdna_fp8_preshuffle_gemm.py compile_fp8_gemm)."""
    n = _lib.native
    if n is not None:
        r = n.gemm(1, A, B, scale_a, scale_b, out, flags)
        if r is not None:
            return r
    return _checked_gemm_fp8(A, B, scale_a, scale_b, out, flags)


@_on_device
def _checked_gemm_fp8(A, B, scale_a, scale_b, out, flags):
    return _gemm_f16(lib().gsb200_gemm_fp8_f16, "gemm_fp8", A, B, scale_a, scale_b, out, flags, _F8)


def _rotary(fn, name, A, B, scale_a, scale_b, sin_buf, cos_buf, nhead, head_dim, rotary_dim, seqlen,
            row_offset, out, flags, dtypes):
    M, N, K = _check_ab(A, B, dtypes)
    _need_cuda(scale_a, scale_b, sin_buf, cos_buf)
    if sin_buf.dtype != torch.float32 or not sin_buf.is_contiguous() or not cos_buf.is_contiguous():
        raise ValueError("sin/cos must be contiguous float32 [seqlen, rotary_dim/2]")
    if sin_buf.shape[0] < seqlen or sin_buf.shape[1] != rotary_dim // 2:
        raise ValueError("sin/cos table smaller than seqlen")
    C = out if out is not None else torch.empty((M, N), dtype=torch.float16, device=A.device)
    check(fn(A.data_ptr(), A.stride(0), B.data_ptr(), B.stride(0), C.data_ptr(), C.stride(0),
             scale_a.data_ptr(), scale_b.data_ptr(), sin_buf.data_ptr(), cos_buf.data_ptr(),
             M, N, K, nhead, head_dim, rotary_dim, seqlen, row_offset, flags, _stream()), name)
    return C


def gemm_i8_rotary(A, B, scale_a, scale_b, sin_buf, cos_buf, nhead, head_dim, rotary_dim, seqlen,
                   row_offset=0, out=None, flags=0):
    """QKV GEMM + rotary epilogue (cute/ampere_gemm_i8_rotary.py TensorOpGemmI8Rotary)."""
    n = _lib.native
    if n is not None:
        r = n.rotary(0, A, B, scale_a, scale_b, sin_buf, cos_buf, nhead, head_dim, rotary_dim, seqlen, row_offset, out, flags)
        if r is not None:
            return r
    return _checked_gemm_i8_rotary(A, B, scale_a, scale_b, sin_buf, cos_buf, nhead, head_dim, rotary_dim, seqlen, row_offset, out, flags)


@_on_device
def _checked_gemm_i8_rotary(A, B, scale_a, scale_b, sin_buf, cos_buf, nhead, head_dim, rotary_dim, seqlen, row_offset, out, flags):
    return _rotary(lib().gsb200_gemm_i8_rotary_f16, "gemm_i8_rotary", A, B, scale_a, scale_b, sin_buf, cos_buf,
                   nhead, head_dim, rotary_dim, seqlen, row_offset, out, flags, _I8)


@_on_device
def quantize_gemm_i8_rotary(x, B, scale_b, sin_buf, cos_buf, nhead, head_dim, rotary_dim, seqlen,
                            row_offset=0, out=None, out_scale=None, flags=0):
    """``gemm_i8_rotary(*quantize_tensor(x), ...)`` in one launch: fp16 ``x`` [M, K] in, the int8 operand is made on
    chip.  Same bytes as the two calls.  ``out_scale`` (optional, [M] fp32) receives the token scales."""
    _need_cuda(x, B, scale_b, sin_buf, cos_buf)
    if x.dtype != torch.float16 or B.dtype != torch.int8 or x.dim() != 2 or B.dim() != 2 or x.shape[1] != B.shape[1]:
        raise ValueError("x must be fp16 [M, K] and B int8 [N, K]")
    if x.stride(1) != 1 or B.stride(1) != 1:
        raise ValueError("rows must be contiguous")
    if sin_buf.dtype != torch.float32 or not sin_buf.is_contiguous() or not cos_buf.is_contiguous():
        raise ValueError("sin/cos must be contiguous float32 [seqlen, rotary_dim/2]")
    if sin_buf.shape[0] < seqlen or sin_buf.shape[1] != rotary_dim // 2:
        raise ValueError("sin/cos table smaller than seqlen")
    M, K = x.shape
    N = B.shape[0]
    C = out if out is not None else torch.empty((M, N), dtype=torch.float16, device=x.device)
    if out_scale is not None and (out_scale.dtype != torch.float32 or out_scale.numel() < M or not out_scale.is_cuda):
        raise ValueError("out_scale must be a CUDA float32 tensor of at least M elements")
    check(lib().gsb200_ptq_gemm_i8_rotary_f16(
        x.data_ptr(), x.stride(0), B.data_ptr(), B.stride(0), C.data_ptr(), C.stride(0),
        out_scale.data_ptr() if out_scale is not None else None, scale_b.data_ptr(), sin_buf.data_ptr(),
        cos_buf.data_ptr(), M, N, K, nhead, head_dim, rotary_dim, seqlen, row_offset, flags, _stream()),
        "quantize_gemm_i8_rotary")
    return C


def gemm_fp8_rotary(A, B, scale_a, scale_b, sin_buf, cos_buf, nhead, head_dim, rotary_dim, seqlen,
                    row_offset=0, out=None, flags=0):
    """FP8 QKV GEMM + rotary (fly/rdna_fp8_gemm_rotary.py compile_fp8_gemm_rotary)."""
    n = _lib.native
    if n is not None:
        r = n.rotary(1, A, B, scale_a, scale_b, sin_buf, cos_buf, nhead, head_dim, rotary_dim, seqlen, row_offset, out, flags)
        if r is not None:
            return r
    return _checked_gemm_fp8_rotary(A, B, scale_a, scale_b, sin_buf, cos_buf, nhead, head_dim, rotary_dim, seqlen, row_offset, out, flags)


@_on_device
def _checked_gemm_fp8_rotary(A, B, scale_a, scale_b, sin_buf, cos_buf, nhead, head_dim, rotary_dim, seqlen, row_offset, out, flags):
    return _rotary(lib().gsb200_gemm_fp8_rotary_f16, "gemm_fp8_rotary", A, B, scale_a, scale_b, sin_buf, cos_buf,
                   nhead, head_dim, rotary_dim, seqlen, row_offset, out, flags, _F8)


def _check_dual(A, Bg, Bu, dtypes):
    M, N, K = _check_ab(A, Bg, dtypes)
    _check_ab(A, Bu, dtypes)
    if Bu.shape != Bg.shape or Bu.stride(0) != Bg.stride(0):      # the library describes both with one N and one stride
        raise ValueError("gate and up weights must share shape and row stride")
    return M, N, K


def _dual(fn, name, A, Bg, Bu, scale_a, sbg, sbu, out, flags, dtypes):
    M, N, K = _check_dual(A, Bg, Bu, dtypes)
    _need_cuda(scale_a, sbg, sbu)
    C = out if out is not None else torch.empty((M, N), dtype=torch.float16, device=A.device)
    check(fn(A.data_ptr(), A.stride(0), Bg.data_ptr(), Bu.data_ptr(), Bg.stride(0), C.data_ptr(), C.stride(0),
             scale_a.data_ptr(), sbg.data_ptr(), sbu.data_ptr(), M, N, K, flags, _stream()), name)
    return C


def dual_gemm_i8_silu(A, B_gate, B_up, scale_a, scale_b_gate, scale_b_up, out=None, flags=0):
    """``silu(A.Bg^T) * (A.Bu^T)`` (cute/ampere_dual_gemm_i8_silu.py TensorOpDualGemmI8Silu)."""
    n = _lib.native
    if n is not None:
        r = n.dual(0, A, B_gate, B_up, scale_a, scale_b_gate, scale_b_up, out, flags)
        if r is not None:
            return r
    return _checked_dual_gemm_i8_silu(A, B_gate, B_up, scale_a, scale_b_gate, scale_b_up, out, flags)


@_on_device
def _checked_dual_gemm_i8_silu(A, B_gate, B_up, scale_a, scale_b_gate, scale_b_up, out, flags):
    return _dual(lib().gsb200_dual_gemm_i8_silu_f16, "dual_gemm_i8_silu", A, B_gate, B_up, scale_a,
                 scale_b_gate, scale_b_up, out, flags, _I8)


def dual_gemm_fp8_silu(A, B_gate, B_up, scale_a, scale_b_gate, scale_b_up, out=None, flags=0):
    """FP8 SwiGLU dual GEMM (fly/rdna_fp8_dual_gemm_silu.py compile_fp8_dual_gemm_silu)."""
    n = _lib.native
    if n is not None:
        r = n.dual(1, A, B_gate, B_up, scale_a, scale_b_gate, scale_b_up, out, flags)
        if r is not None:
            return r
    return _checked_dual_gemm_fp8_silu(A, B_gate, B_up, scale_a, scale_b_gate, scale_b_up, out, flags)


@_on_device
def _checked_dual_gemm_fp8_silu(A, B_gate, B_up, scale_a, scale_b_gate, scale_b_up, out, flags):
    return _dual(lib().gsb200_dual_gemm_fp8_silu_f16, "dual_gemm_fp8_silu", A, B_gate, B_up, scale_a,
                 scale_b_gate, scale_b_up, out, flags, _F8)


def mxfp8_quantize(x, out=None, out_scale=None):
    """Activations [M,K] fp16/fp32 -> (float8_e4m3fn [M,K], uint8 E8M0 scales [M,K/32]); one scale per 32 elements."""
    n = _lib.native
    if n is not None:
        r = n.quantize_mx(x, out, out_scale)
        if r is not None:
            return r
    return _checked_mxfp8_quantize(x, out, out_scale)


@_on_device
def _checked_mxfp8_quantize(x, out, out_scale):
    _need_cuda(x)
    x = _rowmajor(x, "x")
    M, K = x.shape
    q = out if out is not None else torch.empty((M, K), dtype=torch.float8_e4m3fn, device=x.device)
    s = out_scale if out_scale is not None else torch.empty((M, K // 32), dtype=torch.uint8, device=x.device)
    check(lib().gsb200_ptq_mxfp8(x.data_ptr(), _dt(x), x.stride(0), q.data_ptr(), q.stride(0), s.data_ptr(),
                                 s.stride(0), M, K, _stream()), "mxfp8_quantize")
    return q, s


def dual_gemm_fp8_silu_mxfp8(A, B_gate, B_up, scale_a, scale_b_gate, scale_b_up, out=None, out_scale=None, flags=0):
    """FP8 SwiGLU dual GEMM emitting MXFP8 (elements + E8M0 scale per 32 output columns); the interface of
    fp8_dual_silu_mxfp8_wrapper (fly/export_fp8_dual_gemm_silu_mxfp8.py:206-236)."""
    n = _lib.native
    if n is not None:
        r = n.dual_mx(A, B_gate, B_up, scale_a, scale_b_gate, scale_b_up, out, out_scale, flags)
        if r is not None:
            return r
    return _checked_dual_gemm_fp8_silu_mxfp8(A, B_gate, B_up, scale_a, scale_b_gate, scale_b_up, out, out_scale, flags)


@_on_device
def _checked_dual_gemm_fp8_silu_mxfp8(A, B_gate, B_up, scale_a, scale_b_gate, scale_b_up, out, out_scale, flags):
    M, N, K = _check_dual(A, B_gate, B_up, _F8)
    _need_cuda(scale_a, scale_b_gate, scale_b_up)
    q = out if out is not None else torch.empty((M, N), dtype=torch.float8_e4m3fn, device=A.device)
    s = out_scale if out_scale is not None else torch.empty((M, N // 32), dtype=torch.uint8, device=A.device)
    check(lib().gsb200_dual_gemm_fp8_silu_mxfp8(
        A.data_ptr(), A.stride(0), B_gate.data_ptr(), B_up.data_ptr(), B_gate.stride(0), q.data_ptr(), q.stride(0),
        s.data_ptr(), s.stride(0), scale_a.data_ptr(), scale_b_gate.data_ptr(), scale_b_up.data_ptr(), M, N, K, flags,
        _stream()), "dual_gemm_fp8_silu_mxfp8")
    return q, s


@_on_device
def gemm_f16(A, B, scale_a=None, scale_b=None, out=None, flags=0):
    """``(A_f16 . B_f16^T) * sA * sB`` -> fp16, scales optional (compile_f16_down_proj,
    fly/rdna_fp8_factored_gemm.py:660-843, is this with no scales and B = dn ``[R, C]``)."""
    M, N, K = _check_ab(A, B, (torch.float16,))
    C = out if out is not None else torch.empty((M, N), dtype=torch.float16, device=A.device)
    check(lib().gsb200_gemm_f16_f16(A.data_ptr(), A.stride(0), B.data_ptr(), B.stride(0), C.data_ptr(), C.stride(0),
                                    scale_a.data_ptr() if scale_a is not None else None,
                                    scale_b.data_ptr() if scale_b is not None else None, M, N, K, flags, _stream()),
          "gemm_f16")
    return C


def fp8_down_proj(x_fp8, scale_x, dn_fp8_rc, scale_dn, out=None):
    """``x_down_f16[M,R] = (x_fp8 . dn_fp8^T) * sx[m] * s_dn`` with a single scalar weight scale
    (compile_fp8_down_proj, fly/rdna_fp8_factored_gemm.py:442-651); ``dn`` K-major ``[R, C]``."""
    return gemm_fp8(x_fp8, dn_fp8_rc, scale_x, scale_dn, out=out, flags=_lib.FLAG_SCALAR_SCALE_B)


def fp8_factored_gemm(x_fp8, scale_x, dn_fp8_rc, scale_dn, up_f16_nr, bias, out=None):
    """Hoisted low-rank input projection ``ih = f16(f16((x . dn^T) * sx * s_dn) . up^T + bias)`` in one call
    (compile_fp8_factored_gemm, fly/rdna_fp8_factored_gemm.py:86-435).  ``dn`` ``[R, C]`` E4M3 and ``up``
    ``[N, R]`` fp16, both K-major; the intermediate needs no memory of the caller."""
    n = _lib.native
    if n is not None:
        r = n.fac_gemm(x_fp8, scale_x, dn_fp8_rc, scale_dn, up_f16_nr, bias, out)
        if r is not None:
            return r
    return _checked_fp8_factored_gemm(x_fp8, scale_x, dn_fp8_rc, scale_dn, up_f16_nr, bias, out)


@_on_device
def _checked_fp8_factored_gemm(x_fp8, scale_x, dn_fp8_rc, scale_dn, up_f16_nr, bias, out):
    _need_cuda(x_fp8, scale_x, dn_fp8_rc, scale_dn, up_f16_nr, bias)
    _rowmajor(x_fp8, "x"); _rowmajor(dn_fp8_rc, "dn"); _rowmajor(up_f16_nr, "up")
    if x_fp8.dtype != torch.float8_e4m3fn or dn_fp8_rc.dtype != torch.float8_e4m3fn or up_f16_nr.dtype != torch.float16:
        raise TypeError("x and dn must be float8_e4m3fn, up float16")
    M, C = x_fp8.shape
    R, C2 = dn_fp8_rc.shape
    N, R2 = up_f16_nr.shape
    if C2 != C or R2 != R or bias.numel() != N or scale_x.numel() != M:
        raise ValueError("shape mismatch")
    ih = out if out is not None else torch.empty((M, N), dtype=torch.float16, device=x_fp8.device)
    check(lib().gsb200_fac_gemm_fp8_f16(x_fp8.data_ptr(), x_fp8.stride(0), scale_x.data_ptr(), dn_fp8_rc.data_ptr(),
                                        dn_fp8_rc.stride(0), scale_dn.data_ptr(), up_f16_nr.data_ptr(),
                                        up_f16_nr.stride(0), bias.data_ptr(), ih.data_ptr(), ih.stride(0), M, C, R, N,
                                        _stream()), "fp8_factored_gemm")
    return ih


def factored_lstm_step(h_fp8_out, c_inout, hh_down, up_hh, bias_hh, x_down, up_ih, bias_ih):
    """One step of the low-rank hard-gate LSTM cell; argument order of fp8_factored_lstm_wrapper
    (fly/export_fp8_factored_lstm.py:158-182).  ``up_hh`` ``[4H, K_hh]`` and ``up_ih`` ``[4H, R]`` fp16 K-major."""
    n = _lib.native
    if n is not None:
        r = n.fac_step(h_fp8_out, c_inout, hh_down, up_hh, bias_hh, x_down, up_ih, bias_ih)
        if r is not None:
            return h_fp8_out, c_inout
    return _checked_factored_lstm_step(h_fp8_out, c_inout, hh_down, up_hh, bias_hh, x_down, up_ih, bias_ih)


@_on_device
def _checked_factored_lstm_step(h_fp8_out, c_inout, hh_down, up_hh, bias_hh, x_down, up_ih, bias_ih):
    _need_cuda(h_fp8_out, c_inout, hh_down, up_hh, x_down, up_ih)
    B, K_hh = hh_down.shape
    H = up_hh.shape[0] // 4
    R = x_down.shape[1]
    for t in (hh_down, up_hh, x_down, up_ih, c_inout, h_fp8_out):
        if not t.is_contiguous():
            raise ValueError("factored_lstm_step takes contiguous tensors")
    check(lib().gsb200_factored_lstm_step(h_fp8_out.data_ptr(), c_inout.data_ptr(), hh_down.data_ptr(), up_hh.data_ptr(),
                                          bias_hh.data_ptr() if bias_hh is not None else None, x_down.data_ptr(),
                                          up_ih.data_ptr(), bias_ih.data_ptr() if bias_ih is not None else None,
                                          B, H, K_hh, R, _stream()), "factored_lstm_step")
    return h_fp8_out, c_inout


def mx_scales_to_tiled(scales, K):
    """Row-major E8M0 scales ``[rows, K/32]`` -> the 128 x 4 tile order the block-scaled GEMMs take."""
    n = _lib.native
    if n is not None:
        r = n.mx_tile(scales, K)
        if r is not None:
            return r
    return _checked_mx_scales_to_tiled(scales, K)


@_on_device
def _checked_mx_scales_to_tiled(scales, K):
    _need_cuda(scales)
    rows = scales.shape[0]
    out = torch.empty(int(lib().gsb200_mx_tiled_scale_bytes(rows, K)), dtype=torch.uint8, device=scales.device)
    check(lib().gsb200_mx_scales_to_tiled(scales.data_ptr(), scales.stride(0), rows, K, out.data_ptr(), _stream()),
          "mx_scales_to_tiled")
    return out


def gemm_mxfp8(A, sfa_tiled, B, sfb_tiled, out=None):
    """Block-scaled MXFP8 GEMM ``A[M,K] . B[N,K]^T`` (E8M0 scale per 32 K elements on both operands) -> fp16."""
    n = _lib.native
    if n is not None:
        r = n.mx_gemm(A, sfa_tiled, B, sfb_tiled, out)
        if r is not None:
            return r
    return _checked_gemm_mxfp8(A, sfa_tiled, B, sfb_tiled, out)


@_on_device
def _checked_gemm_mxfp8(A, sfa_tiled, B, sfb_tiled, out):
    M, N, K = _check_ab(A, B, _F8)
    C = out if out is not None else torch.empty((M, N), dtype=torch.float16, device=A.device)
    check(lib().gsb200_gemm_mxfp8_f16(A.data_ptr(), A.stride(0), sfa_tiled.data_ptr(), B.data_ptr(), B.stride(0),
                                      sfb_tiled.data_ptr(), C.data_ptr(), C.stride(0), M, N, K, _stream()), "gemm_mxfp8")
    return C


def dual_gemm_mxfp8_silu(A, sfa_tiled, B_gate, B_up, sfb_gate_tiled, sfb_up_tiled, out=None):
    """Block-scaled MXFP8 SwiGLU dual GEMM ``silu(A.Bg^T) * (A.Bu^T)`` -> fp16."""
    n = _lib.native
    if n is not None:
        r = n.mx_dual(A, sfa_tiled, B_gate, B_up, sfb_gate_tiled, sfb_up_tiled, out)
        if r is not None:
            return r
    return _checked_dual_gemm_mxfp8_silu(A, sfa_tiled, B_gate, B_up, sfb_gate_tiled, sfb_up_tiled, out)


@_on_device
def _checked_dual_gemm_mxfp8_silu(A, sfa_tiled, B_gate, B_up, sfb_gate_tiled, sfb_up_tiled, out):
    M, N, K = _check_dual(A, B_gate, B_up, _F8)
    C = out if out is not None else torch.empty((M, N), dtype=torch.float16, device=A.device)
    check(lib().gsb200_dual_gemm_mxfp8_silu_f16(A.data_ptr(), A.stride(0), sfa_tiled.data_ptr(), B_gate.data_ptr(),
                                                B_up.data_ptr(), B_gate.stride(0), sfb_gate_tiled.data_ptr(),
                                                sfb_up_tiled.data_ptr(), C.data_ptr(), C.stride(0), M, N, K, _stream()),
          "dual_gemm_mxfp8_silu")
    return C


# ---- block-scaled FP8: one fp32 scale per 128 elements of a row, or per 128 x 128 tile ---------------------------------
# The backward operators are calls of their own: as everywhere in this package, autograd sees none of it, and results are detached whatever their inputs
# require.
BLOCK = 128
_BLOCK_DT = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}


def _block_dt(t, name, allowed=(torch.float16, torch.bfloat16, torch.float32)):
    dt = t if isinstance(t, torch.dtype) else t.dtype
    if dt not in allowed:
        raise TypeError(f"{name} must be one of {tuple(allowed)}, not {dt}")
    return _BLOCK_DT[dt]


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def _rows16(m, n, dtype, device):
    """An [m, n] output whose rows start on 16-byte boundaries: what the tensor cores read, and the fast stores."""
    per = 16 // dtype.itemsize
    ld = (n + per - 1) // per * per
    return torch.empty((m, n), dtype=dtype, device=device) if ld == n else torch.empty_strided((m, n), (ld, 1), dtype=dtype, device=device)


def _given(t, shape, dtypes, name):
    """A tensor argument of this shape and one of these types, rows of unit stride that do not overlap."""
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, not {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {list(shape)}, not {list(t.shape)}")
    if shape[0] == 0 or shape[1] == 0:
        return t
    if (shape[1] > 1 and t.stride(1) != 1) or (shape[0] > 1 and t.stride(0) < shape[1]):
        raise ValueError(f"{name} must have unit inner stride and rows that do not overlap")
    return t


def _ld(t):
    """Row stride for the library; of a single row it says nothing, so the least that is aligned for any use."""
    return t.stride(0) if t.shape[0] > 1 else (t.shape[1] + 15) // 16 * 16


def _f8_scaled(q, s, rows, name):
    if q.dim() != 2:
        raise ValueError(f"{name} must be 2-D")
    _given(q, q.shape, _F8, name)
    _given(s, (_blocks(q.shape[0]) if rows == BLOCK else q.shape[0], _blocks(q.shape[1])), (torch.float32,), f"scale of {name}")


def _2d(t, name):
    if t.dim() != 2:
        raise ValueError(f"{name} must be 2-D")
    return _given(t, t.shape, (t.dtype,), name)


def fp8_block_quantize(x, rows=1, out=None, out_scale=None):
    """``x`` [M,K] fp16/bf16/fp32 -> (float8_e4m3fn [M,K], fp32 scales): one scale per 128 elements of a row (``rows=1``, activations,
    gradients and checkpoints: scales [M, ceil(K/128)]) or per 128 x 128 tile (``rows=128``, weights: [ceil(M/128), ceil(K/128)]).
    Scales are the smallest powers of two with ``max|x| <= 448 * scale``.  The elements' rows start on 16-byte boundaries, as the
    products want them."""
    n = _lib.native
    if n is not None:
        r = n.block_quantize(x, rows, out, out_scale)
        if r is not None:
            return r
    return _checked_fp8_block_quantize(x, rows, out, out_scale)


@_on_device
def _checked_fp8_block_quantize(x, rows, out, out_scale):
    _need_cuda(x)
    _2d(x, "x")
    dt = _block_dt(x, "x")
    if rows not in (1, BLOCK):
        raise ValueError("a block is 1 or 128 rows")
    M, K = x.shape
    sshape = (_blocks(M) if rows == BLOCK else M, _blocks(K))
    q = _given(out, (M, K), _F8, "out") if out is not None else _rows16(M, K, torch.float8_e4m3fn, x.device)
    s = _given(out_scale, sshape, (torch.float32,), "out_scale") if out_scale is not None else torch.empty(sshape, dtype=torch.float32, device=x.device)
    check(lib().gsb200_block_quantize_fp8(x.data_ptr(), dt, _ld(x), q.data_ptr(), _ld(q), s.data_ptr(), max(_ld(s), sshape[1]), M, K, rows, _stream()),
          "fp8_block_quantize")
    return q, s


def fp8_block_dequantize(q, scale, rows=1, dtype=torch.bfloat16, out=None):
    """The values ``q * scale`` of a block-scaled tensor as fp16, bf16 or fp32 (a checkpoint restored, for a backward pass of the
    caller's own).  Exact in bf16 and fp32 for scales that are powers of two."""
    n = _lib.native
    if n is not None:
        r = n.block_dequantize(q, scale, rows, _BLOCK_DT.get(dtype, -1), out)
        if r is not None:
            return r
    return _checked_fp8_block_dequantize(q, scale, rows, dtype, out)


@_on_device
def _checked_fp8_block_dequantize(q, scale, rows, dtype, out):
    _need_cuda(q, scale)
    if rows not in (1, BLOCK):
        raise ValueError("a block is 1 or 128 rows")
    _f8_scaled(q, scale, rows, "q")
    M, K = q.shape
    if out is not None:
        _2d(out, "out")
        dtype = out.dtype
    dt = _block_dt(dtype, "out")
    x = _given(out, (M, K), (dtype,), "out") if out is not None else _rows16(M, K, dtype, q.device)
    check(lib().gsb200_block_dequantize_fp8(q.data_ptr(), _ld(q), scale.data_ptr(), _ld(scale), x.data_ptr(), dt, _ld(x), M, K, rows, _stream()),
          "fp8_block_dequantize")
    return x


def gemm_fp8_block(A, B, scale_a, scale_b, out=None, dtype=torch.float16, b_transposed=False):
    """``A[M,K] . B[N,K]^T`` over block-scaled FP8 operands -> fp16, bf16 or fp32: ``scale_a`` [M, ceil(K/128)], ``scale_b``
    [ceil(N/128), ceil(K/128)].  ``b_transposed``: B is [K,N] with scales [ceil(K/128), ceil(N/128)], which is the input gradient
    ``dY . W`` with the weight as the forward pass has it.  Sums and scales in fp32, one rounding: a product of two scales has to be a
    normal fp32 number, or 0."""
    n = _lib.native
    if n is not None:
        r = n.block_gemm(A, B, scale_a, scale_b, out, _BLOCK_DT.get(dtype, -1), b_transposed)
        if r is not None:
            return r
    return _checked_gemm_fp8_block(A, B, scale_a, scale_b, out, dtype, b_transposed)


@_on_device
def _checked_gemm_fp8_block(A, B, scale_a, scale_b, out, dtype, b_transposed):
    _need_cuda(A, B, scale_a, scale_b)
    _f8_scaled(A, scale_a, 1, "A")
    _f8_scaled(B, scale_b, BLOCK, "B")
    M, K = A.shape
    Kb, N = B.shape if b_transposed else B.shape[::-1]
    if Kb != K:
        raise ValueError(f"A is [M,K] with K = {K}, B {'[K,N]' if b_transposed else '[N,K]'} with K = {Kb}")
    if out is not None:
        _2d(out, "out")
        dtype = out.dtype
    dt = _block_dt(dtype, "out")
    C = _given(out, (M, N), (dtype,), "out") if out is not None else _rows16(M, N, dtype, A.device)
    check(lib().gsb200_gemm_fp8_block(A.data_ptr(), _ld(A), scale_a.data_ptr(), _ld(scale_a), B.data_ptr(), _ld(B), scale_b.data_ptr(),
                                      _ld(scale_b), C.data_ptr(), _ld(C), dt, M, N, K, _lib.FLAG_B_KN if b_transposed else 0, _stream()),
          "gemm_fp8_block")
    return C


def gemm_fp8_block_wgrad(dy, q, scale, out=None, accumulate=False):
    """Weight gradient ``dY^T . X`` [N,K] fp32 from ``dy`` [M,N] fp16/bf16 and the block-scaled 8-bit checkpoint ``q`` [M,K],
    ``scale`` [M, ceil(K/128)] of the layer's input.  ``accumulate`` adds to ``out``.  Rows of ``dy`` on 16-byte boundaries.  The
    checkpoint is restored to ``dy``'s significand, without loss for scales that are powers of two, whatever their size."""
    n = _lib.native
    if n is not None:
        r = n.block_wgrad(dy, q, scale, out, accumulate)
        if r is not None:
            return r
    return _checked_gemm_fp8_block_wgrad(dy, q, scale, out, accumulate)


@_on_device
def _checked_gemm_fp8_block_wgrad(dy, q, scale, out, accumulate):
    _need_cuda(dy, q, scale)
    _2d(dy, "dy")
    dt = _block_dt(dy, "dy", (torch.float16, torch.bfloat16))
    _f8_scaled(q, scale, 1, "q")
    (M, N), K = dy.shape, q.shape[1]
    if q.shape[0] != M:
        raise ValueError(f"dy has {M} rows, the checkpoint {q.shape[0]}")
    if accumulate and out is None:
        raise ValueError("accumulate needs the tensor to add to as out")
    dw = _given(out, (N, K), (torch.float32,), "out") if out is not None else torch.empty((N, K), dtype=torch.float32, device=dy.device)
    need = int(lib().gsb200_gemm_fp8_block_wgrad_workspace_bytes(M, N, K))
    ws = torch.empty(need, dtype=torch.uint8, device=dy.device) if need else None
    check(lib().gsb200_gemm_fp8_block_wgrad(dy.data_ptr(), dt, _ld(dy), q.data_ptr(), _ld(q), scale.data_ptr(), _ld(scale), dw.data_ptr(), _ld(dw),
                                            1 if accumulate else 0, ws.data_ptr() if need else None, need, M, N, K, _stream()),
          "gemm_fp8_block_wgrad")
    return dw


def swiglu_fp8_block(gate, up):
    """``gate * sigmoid(gate) * up`` as a block-scaled FP8 tensor, with 8-bit checkpoints of both inputs: ``((h, scale), (gate, scale),
    (up, scale))``, each what ``fp8_block_quantize`` makes (of ``h``: from its fp32 values)."""
    n = _lib.native
    if n is not None:
        r = n.block_swiglu(gate, up)
        if r is not None:
            return r
    return _checked_swiglu_fp8_block(gate, up)


@_on_device
def _checked_swiglu_fp8_block(gate, up):
    _need_cuda(gate, up)
    _2d(gate, "gate")
    dt = _block_dt(gate, "gate")
    _given(up, gate.shape, (gate.dtype,), "up")
    M, F = gate.shape
    q = [_rows16(M, F, torch.float8_e4m3fn, gate.device) for _ in range(3)]
    s = [torch.empty((M, _blocks(F)), dtype=torch.float32, device=gate.device) for _ in range(3)]
    check(lib().gsb200_swiglu_fp8_block(gate.data_ptr(), _ld(gate), up.data_ptr(), _ld(up), dt, q[0].data_ptr(), s[0].data_ptr(), q[1].data_ptr(),
                                        s[1].data_ptr(), q[2].data_ptr(), s[2].data_ptr(), q[0].stride(0), s[0].stride(0), M, F, _stream()),
          "swiglu_fp8_block")
    return (q[0], s[0]), (q[1], s[1]), (q[2], s[2])


def swiglu_fp8_block_bwd(dh, gate_q, gate_scale, up_q, up_scale, quantize=False):
    """Gradients of SwiGLU from the checkpoints: ``(dgate, dup)`` in ``dh``'s type.  ``quantize``: also ``(q, scale)`` of each, as
    ``fp8_block_quantize`` makes of them, in the same pass: ``(dgate, dup, (q, scale), (q, scale))``."""
    n = _lib.native
    if n is not None and not quantize:
        r = n.block_swiglu_bwd(dh, gate_q, gate_scale, up_q, up_scale)
        if r is not None:
            return r
    return _checked_swiglu_fp8_block_bwd(dh, gate_q, gate_scale, up_q, up_scale, quantize)


@_on_device
def _checked_swiglu_fp8_block_bwd(dh, gate_q, gate_scale, up_q, up_scale, quantize):
    _need_cuda(dh, gate_q, gate_scale, up_q, up_scale)
    _2d(dh, "dh")
    dt = _block_dt(dh, "dh")
    _f8_scaled(gate_q, gate_scale, 1, "gate_q")
    _f8_scaled(up_q, up_scale, 1, "up_q")
    M, F = dh.shape
    if tuple(gate_q.shape) != (M, F) or tuple(up_q.shape) != (M, F):
        raise ValueError(f"dh is {[M, F]}, the checkpoints {list(gate_q.shape)} and {list(up_q.shape)}")
    dg, du = (_rows16(M, F, dh.dtype, dh.device) for _ in range(2))
    q = [_rows16(M, F, torch.float8_e4m3fn, dh.device) for _ in range(2 if quantize else 0)]
    s = [torch.empty((M, _blocks(F)), dtype=torch.float32, device=dh.device) for _ in q]
    extra = (q[0].data_ptr(), s[0].data_ptr(), q[1].data_ptr(), s[1].data_ptr(), q[0].stride(0), s[0].stride(0)) if quantize else (None, None, None, None, 0, 0)
    check(lib().gsb200_swiglu_fp8_block_bwd(dh.data_ptr(), dt, _ld(dh), gate_q.data_ptr(), _ld(gate_q), gate_scale.data_ptr(), _ld(gate_scale),
                                            up_q.data_ptr(), _ld(up_q), up_scale.data_ptr(), _ld(up_scale), dg.data_ptr(), dg.stride(0),
                                            du.data_ptr(), du.stride(0), *extra, M, F, _stream()), "swiglu_fp8_block_bwd")
    return (dg, du, (q[0], s[0]), (q[1], s[1])) if quantize else (dg, du)
