"""Oracle: block-scaled FP8 (E4M3 elements, one fp32 scale per 128 elements of a row or per 128 x 128 tile) in 64 bits.

Test infrastructure only.  Not in the reference project; the definitions are the public header's.
"""
import torch

BLOCK = 128


def spread(s, rows, m, k):
    """The scale of every element, float64."""
    i = torch.arange(m, device=s.device) // rows
    j = torch.arange(k, device=s.device) // BLOCK
    return s.double()[i[:, None], j[None, :]]


def quantize(x, rows=1):
    """(elements as float64 in units of their scale, scales float64): scale 2^t with the least t >= -126 that keeps every finite
    |x| <= 448 2^t, 1 for a block of zeros; elements nearest (half to even) in E4M3, NaN for what is not finite."""
    m, k = x.shape
    x = x.double()
    fin = torch.isfinite(x)
    mag = torch.where(fin, x.abs(), 0.0)
    mb, kb = -(-m // rows), -(-k // BLOCK)
    pad = torch.zeros(mb * rows, kb * BLOCK, dtype=torch.float64, device=x.device)
    pad[:m, :k] = mag
    top = pad.view(mb, rows, kb, BLOCK).amax(dim=(1, 3))
    mant, e = torch.frexp(top)                                     # top = mant 2^e, 1/2 <= mant < 1; 448 = 7/8 2^9
    t = (e - 9 + (mant > 0.875)).clamp(min=-126)
    s = torch.where(top > 0, torch.ldexp(torch.ones_like(top), t), torch.ones_like(top))
    v = torch.where(fin, x, 0.0) / spread(s, rows, m, k)
    step = torch.ldexp(torch.ones_like(v), torch.frexp(v.abs().clamp(min=2.0 ** -6))[1] - 4)     # spacing of E4M3 at v
    q = torch.round(v / step) * step
    return torch.where(fin, q, float("nan")), s


def values(q, s, rows=1):
    return (q.double() if q.dtype != torch.uint8 else q.view(torch.float8_e4m3fn).double()) * spread(s, rows, *q.shape)


def gemm(A, sa, B, sb, transposed=False):
    """(C, sum of the magnitudes of the products) float64."""
    a, b = values(A, sa), values(B, sb, BLOCK)
    b = b if transposed else b.t()
    return a @ b, a.abs() @ b.abs()


def wgrad(dy, q, s):
    d, x = dy.double(), values(q, s)
    return d.t() @ x, d.abs().t() @ x.abs()


def swiglu(g, u):
    return g * torch.sigmoid(g) * u


def swiglu_bwd(dh, g, u):
    """(dgate, dup) float64 of float64 values."""
    sig = torch.sigmoid(g)
    return dh * u * sig * (1 + g * torch.sigmoid(-g)), dh * g * sig
