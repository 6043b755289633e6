"""GPU parity of the block-scaled FP8 operators against 64-bit statements of them.

Tolerances.  eps / 2 of the output type is its rounding.  A sum of n products in fp32, each addition off by at most 2^-23 of
the magnitudes summed so far (a tensor core may truncate), is within n 2^-23 of the sum of the magnitudes.  The block products add
128 terms per block, one multiply-add per block and one product of two scales."""
import math

import pytest
import torch

from oracle import block8
from util import need_lib

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn
TYPES = [torch.float16, torch.bfloat16, torch.float32]
SIZES = [(1, 1), (1, 128), (3, 127), (5, 129), (130, 256), (257, 1001), (70, 2049), (33, 640), (129, 8)]


def eps(dt):
    return torch.finfo(dt).eps / 2


def rnd(gen, *shape):
    return torch.randn(*shape, generator=gen)


def check_quantized(q, s, x, rows):
    want_q, want_s = block8.quantize(x.cpu(), rows)
    assert torch.equal(s.cpu().double(), want_s)
    got = q.cpu().view(torch.float8_e4m3fn).double()
    same = (got == want_q) | (got.isnan() & want_q.isnan())
    assert bool(same.all()), f"{int((~same).sum())} elements differ"
    assert torch.equal(torch.signbit(got[~want_q.isnan()]), torch.signbit(want_q[~want_q.isnan()]))


@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m,k", SIZES)
def test_quantize_is_exact(m, k, dt, rows):
    g = need_lib()
    gen = torch.Generator().manual_seed(m * 1000 + k)
    x = (rnd(gen, m, k) * torch.exp(3 * rnd(gen, m, 1))).to(dt)
    q, s = g.fp8_block_quantize(x.cuda(), rows=rows)
    check_quantized(q, s, x, rows)
    for out_t in TYPES:
        back = g.fp8_block_dequantize(q, s, rows=rows, dtype=out_t)
        want = block8.values(q.cpu(), s.cpu(), rows).to(out_t)
        assert torch.equal(back.cpu(), want)


@pytest.mark.parametrize("dt", TYPES)
def test_quantize_at_the_borders_of_the_scale(dt):
    """Block maxima at 448 2^t and its neighbours, at every power of two, subnormal, zero; NaN and infinities beside them."""
    g = need_lib()
    fi = torch.finfo(dt)
    tops = [0.0, fi.smallest_normal, float(torch.tensor(fi.smallest_normal, dtype=torch.float64) * fi.eps), fi.max]
    for t in range(-20, 7):
        v = torch.tensor(448.0 * 2.0 ** t).to(dt)
        tops += [float(v), float(torch.nextafter(v, torch.tensor(math.inf, dtype=dt))), float(torch.nextafter(v, torch.tensor(0.0, dtype=dt)))]
    gen = torch.Generator().manual_seed(5)
    x = torch.zeros(len(tops), 300, dtype=torch.float64)
    for i, t in enumerate(tops):
        x[i] = t * (2 * torch.rand(300, generator=gen, dtype=torch.float64) - 1)
        x[i, 7] = t
        x[i, 200] = -t
    x = x.to(dt)
    q, s = g.fp8_block_quantize(x.cuda())
    check_quantized(q, s, x, 1)
    x[3, 5], x[4, 130], x[5, 131], x[6, :] = math.nan, math.inf, -math.inf, math.nan
    x[7, :128] = math.inf
    for rows in (1, 128):
        q, s = g.fp8_block_quantize(x.cuda(), rows=rows)
        check_quantized(q, s, x, rows)


@pytest.mark.parametrize("k", [100, 128, 250, 512, 300])
@pytest.mark.parametrize("dt", TYPES)
def test_quantize_many_short_rows(k, dt):
    g = need_lib()
    gen = torch.Generator().manual_seed(k)
    x = rnd(gen, 16391, k).to(dt)
    check_quantized(*g.fp8_block_quantize(x.cuda()), x, 1)
    pad = torch.zeros(16391, (k + 7) // 8 * 8, dtype=dt, device="cuda")[:, :k]
    pad.copy_(x)
    check_quantized(*g.fp8_block_quantize(pad), x, 1)


def test_quantize_every_half():
    g = need_lib()
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.float16).view(512, 128).clone()
    q, s = g.fp8_block_quantize(x.cuda())
    check_quantized(q, s, x, 1)
    y = x.view(128, 512).t().contiguous().view(512, 128)
    q, s = g.fp8_block_quantize(y.cuda())
    check_quantized(q, s, y, 1)


@pytest.mark.parametrize("off", [0, 1, 8])
@pytest.mark.parametrize("dt", TYPES)
def test_strided_rows_and_what_lies_behind_them(dt, off):
    """Views into larger buffers, aligned and not: same result, and nothing outside them is written."""
    g = need_lib()
    gen = torch.Generator().manual_seed(11)
    m, k = 37, 333
    buf = rnd(gen, m, 401).to(dt).cuda()
    x = buf[:, off:off + k]
    want_q, want_s = g.fp8_block_quantize(x.contiguous())
    qbuf = torch.full((m + 1, 400), 0x55, dtype=torch.uint8, device="cuda")
    sbuf = torch.full((m + 1, 9), -7.0, device="cuda")
    g.fp8_block_quantize(x, out=qbuf[:m, off:off + k].view(F8), out_scale=sbuf[:m, 2:5])
    assert torch.equal(qbuf[:m, off:off + k], want_q.view(torch.uint8)) and torch.equal(sbuf[:m, 2:5], want_s)
    keep = torch.ones_like(qbuf, dtype=torch.bool)
    keep[:m, off:off + k] = False
    assert bool((qbuf[keep] == 0x55).all())
    sbuf[:m, 2:5] = -7.0
    assert bool((sbuf == -7.0).all())
    xbuf = torch.full((m + 1, 400), 3.0, dtype=dt, device="cuda")
    g.fp8_block_dequantize(want_q, want_s, out=xbuf[:m, off:off + k])
    assert torch.equal(xbuf[:m, off:off + k], g.fp8_block_dequantize(want_q, want_s, dtype=dt))
    assert bool((xbuf[keep] == 3.0).all())


# ---- products ------------------------------------------------------------------------------------------------------------
def operands(gen, m, n, k, transposed, any_scales=True):
    g = need_lib()
    a, sa = g.fp8_block_quantize((rnd(gen, m, k) * torch.exp(rnd(gen, m, 1))).cuda())
    w = rnd(gen, k, n) if transposed else rnd(gen, n, k)
    b, sb = g.fp8_block_quantize(w.cuda(), rows=128)
    if any_scales:
        sa = sa * (0.5 + torch.rand(sa.shape, generator=gen).cuda())
        sb = sb * (0.5 + torch.rand(sb.shape, generator=gen).cuda())
    return a, b, sa, sb


def check_gemm(c, a, b, sa, sb, transposed):
    want, mag = block8.gemm(a, sa, b, sb, transposed)
    k = a.shape[1]
    tol = eps(c.dtype) * want.abs() + (128 + k // 128 + 3) * 2.0 ** -23 * mag
    if c.dtype == torch.float16:
        tol = tol + 2.0 ** -25                             # half of the smallest step
    err = (c.double() - want).abs()
    assert bool((err <= tol).all()), f"worst {float((err / tol).max())} of the bound, {int((err > tol).sum())} of {err.numel()} outside"


GEMM_SIZES = [(1, 8, 128), (1, 2048, 512), (3, 130, 127), (7, 1, 1), (64, 384, 1000), (128, 256, 128), (129, 257, 129), (333, 1536, 512), (1000, 72, 2049),
              (300, 129, 100), (20, 4096, 4096), (2500, 520, 640), (600, 1000, 300), (600, 1000, 2300), (5000, 1001, 520), (20000, 520, 384),
              (1, 1000, 4097), (2, 72, 5120), (3, 513, 1000), (4, 1024, 2048), (5, 40, 300), (2, 9, 10240), (1, 16, 12000), (30000, 128, 200), (20001, 130, 700), (12000, 384, 384)]


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m,n,k", GEMM_SIZES)
def test_gemm(m, n, k, dt, transposed):
    g = need_lib()
    a, b, sa, sb = operands(torch.Generator().manual_seed(m + n + k), m, n, k, transposed)
    c = g.gemm_fp8_block(a, b, sa, sb, dtype=dt, b_transposed=transposed)
    assert c.shape == (m, n) and c.dtype == dt
    check_gemm(c, a, b, sa, sb, transposed)
    again = g.gemm_fp8_block(a, b, sa, sb, dtype=dt, b_transposed=transposed)
    assert torch.equal(c, again)
    assert g.device_status()[0] == 0


@pytest.mark.parametrize("transposed", [False, True])
def test_gemm_places_every_element(transposed):
    """One element of each operand at a time: the product lands where it belongs and nowhere else."""
    g = need_lib()
    m, n, k = 150, 300, 200
    for i, j, l in [(0, 0, 0), (149, 299, 199), (17, 130, 127), (128, 255, 128), (31, 64, 96), (127, 256, 33)]:
        a = torch.zeros(m, 208, dtype=torch.uint8, device="cuda").view(F8)[:, :k]
        b = torch.zeros((k, 304) if transposed else (n, 208), dtype=torch.uint8, device="cuda").view(F8)[:, :n if transposed else k]
        a.view(torch.uint8)[i, l] = 0x40                   # 2
        b.view(torch.uint8)[(l, j) if transposed else (j, l)] = 0x44     # 3
        sa = torch.arange(1, m * 2 + 1, device="cuda").float().view(m, 2)
        sb = torch.arange(1, 7, device="cuda").float().view((2, 3) if transposed else (3, 2))
        c = g.gemm_fp8_block(a, b, sa, sb, dtype=torch.float32, b_transposed=transposed)
        want = torch.zeros(m, n, device="cuda")
        want[i, j] = 6 * sa[i, l // 128] * (sb[l // 128, j // 128] if transposed else sb[j // 128, l // 128])
        assert torch.equal(c, want)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("off,ld", [(0, 320), (1, 333), (8, 352)])
def test_gemm_into_a_view(off, ld, dt):
    """Outputs whose rows TMA can and cannot address; nothing outside the view is written."""
    g = need_lib()
    m, n, k = 140, 300, 256
    a, b, sa, sb = operands(torch.Generator().manual_seed(3), m, n, k, False)
    buf = torch.full((m + 2, ld), 5.0, dtype=dt, device="cuda")
    g.gemm_fp8_block(a, b, sa, sb, out=buf[:m, off:off + n])
    assert torch.equal(buf[:m, off:off + n], g.gemm_fp8_block(a, b, sa, sb, dtype=dt))
    keep = torch.ones_like(buf, dtype=torch.bool)
    keep[:m, off:off + n] = False
    assert bool((buf[keep] == 5.0).all())


def test_gemm_nan_stays_in_its_row_and_column():
    g = need_lib()
    m, n, k = 200, 300, 300
    a, b, sa, sb = operands(torch.Generator().manual_seed(4), m, n, k, False)
    ref = g.gemm_fp8_block(a, b, sa, sb, dtype=torch.float32)
    a.view(torch.uint8)[130, 299] = 0x7f
    b.view(torch.uint8)[257, 5] = 0x7f
    c = g.gemm_fp8_block(a, b, sa, sb, dtype=torch.float32)
    nan = c.isnan()
    want = torch.zeros_like(nan)
    want[130, :] = True
    want[:, 257] = True
    assert torch.equal(nan, want) and torch.equal(c[~want], ref[~want])


def test_gemm_what_lies_behind_the_operands_rows_does_not_matter():
    g = need_lib()
    m, n, k = 70, 90, 200
    for transposed in (False, True):
        a, b, sa, sb = operands(torch.Generator().manual_seed(6), m, n, k, transposed)
        ref = g.gemm_fp8_block(a, b, sa, sb, b_transposed=transposed)
        abuf = torch.full((m + 60, 256), 0x7f, dtype=torch.uint8, device="cuda")
        bbuf = torch.full((b.shape[0] + 60, 256), 0x7f, dtype=torch.uint8, device="cuda")
        abuf[:m, :k] = a.view(torch.uint8)
        bbuf[:b.shape[0], :b.shape[1]] = b.view(torch.uint8)
        got = g.gemm_fp8_block(abuf.view(F8)[:m, :k], bbuf.view(F8)[:b.shape[0], :b.shape[1]], sa, sb, b_transposed=transposed)
        assert torch.equal(got, ref)


@pytest.mark.parametrize("limit", [1, 9, 60])
def test_gemm_under_an_sm_limit(limit):
    """Fewer CTAs than tiles: the same bytes."""
    g = need_lib()
    sets = [operands(torch.Generator().manual_seed(5), m, n, k, tr) + (tr,) for m, n, k, tr in ((700, 400, 300, False), (2100, 520, 260, True), (40, 700, 512, False))]
    ref = [g.gemm_fp8_block(a, b, sa, sb, b_transposed=tr) for a, b, sa, sb, tr in sets]
    g.lib().gsb200_set_sm_limit(limit)
    try:
        got = [g.gemm_fp8_block(a, b, sa, sb, b_transposed=tr) for a, b, sa, sb, tr in sets]
        torch.cuda.synchronize()
    finally:
        g.lib().gsb200_set_sm_limit(0)
    assert all(torch.equal(x, y) for x, y in zip(got, ref)) and g.device_status()[0] == 0


@pytest.mark.parametrize("m", [1, 2, 3, 4, 5])
def test_gemm_rows_do_not_depend_on_the_form(m):
    """A row's result is the same whichever kernel the number of rows selects, up to the order of fp32 sums."""
    g = need_lib()
    a, b, sa, sb = operands(torch.Generator().manual_seed(m), 300, 264, 1000, False)
    for dt in TYPES:
        full = g.gemm_fp8_block(a, b, sa, sb, dtype=dt)
        _, mag = block8.gemm(a[:m], sa[:m], b, sb)
        few = g.gemm_fp8_block(a[:m], b, sa[:m], sb, dtype=dt)
        tol = 2 * eps(dt) * full[:m].double().abs() + 2 * (128 + 11) * 2.0 ** -23 * mag + 2.0 ** -24
        assert bool(((few.double() - full[:m].double()).abs() <= tol).all())


# ---- weight gradient -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(1, 8, 128), (1, 1, 1), (63, 130, 127), (64, 256, 256), (65, 129, 257), (300, 1000, 520), (2000, 512, 100), (5000, 264, 512),
                                   (9001, 72, 1001), (33000, 264, 200), (40001, 40, 136)])
def test_wgrad(m, n, k, dt):
    g = need_lib()
    gen = torch.Generator().manual_seed(m + n + k)
    q, s = g.fp8_block_quantize(rnd(gen, m, k).cuda())
    pad = (n + 7) // 8 * 8
    dy = (rnd(gen, m, pad) * 0.1).to(dt).cuda()[:, :n]
    want, mag = block8.wgrad(dy, q, s)
    dw = g.gemm_fp8_block_wgrad(dy, q, s)
    tol = eps(torch.float32) * want.abs() + (m + 160) * 2.0 ** -23 * mag          # (up to 148 parts are added)
    assert bool(((dw.double() - want).abs() <= tol).all())
    assert torch.equal(dw, g.gemm_fp8_block_wgrad(dy, q, s))
    start = rnd(gen, n, k).cuda()
    acc = start.clone()
    g.gemm_fp8_block_wgrad(dy, q, s, out=acc, accumulate=True)
    want = want + start.double()
    tol = tol + 2.0 ** -23 * (want.abs() + mag)
    assert bool(((acc.double() - want).abs() <= tol).all())
    assert g.device_status()[0] == 0


@pytest.mark.parametrize("dt,m", [(torch.float16, 4100), (torch.float16, 8250), (torch.bfloat16, 8250)])
@pytest.mark.parametrize("k,ld", [(1000, 1000), (1000, 1004), (1000, 1001), (1001, 1001)])
def test_wgrad_in_segments_straight_to_dw(k, ld, dt, m):
    """So many tiles that the batch is not cut: its segments are added in dW itself, in boxes or element by element, or (rows
    that are no whole vectors) in the workspace, to what dW holds or not."""
    g = need_lib()
    gen = torch.Generator().manual_seed(m + ld)
    n = 9700
    assert (g.lib().gsb200_gemm_fp8_block_wgrad_workspace_bytes(m, n, k) == 0) == (k % 4 == 0)
    q, s = g.fp8_block_quantize(rnd(gen, m, k).cuda())
    dy = (rnd(gen, m, 9704) * 0.1).to(dt).cuda()[:, :n]
    want, mag = block8.wgrad(dy, q, s)
    tol = eps(torch.float32) * want.abs() + (m + 160) * 2.0 ** -23 * mag
    buf = torch.full((n, ld), math.nan, device="cuda")
    dw = g.gemm_fp8_block_wgrad(dy, q, s, out=buf[:, :k])
    assert bool(((dw.double() - want).abs() <= tol).all()) and bool(buf[:, k:].isnan().all())
    start = dw.double()
    g.gemm_fp8_block_wgrad(dy, q, s, out=dw, accumulate=True)
    want = want + start
    assert bool(((dw.double() - want).abs() <= tol + 3 * 2.0 ** -23 * (want.abs() + mag)).all()) and bool(buf[:, k:].isnan().all())     # (up to three additions to dW)
    assert g.device_status()[0] == 0


def test_wgrad_and_few_rows_know_no_sm_limit():
    g = need_lib()
    gen = torch.Generator().manual_seed(4)
    q, s = g.fp8_block_quantize(rnd(gen, 3000, 520).cuda())
    dy = rnd(gen, 3000, 1000).half().cuda()
    a, b, sa, sb = operands(gen, 2, 700, 512, False)
    ref = [g.gemm_fp8_block_wgrad(dy, q, s), g.gemm_fp8_block(a, b, sa, sb)]
    g.lib().gsb200_set_sm_limit(1)
    try:
        got = [g.gemm_fp8_block_wgrad(dy, q, s), g.gemm_fp8_block(a, b, sa, sb)]
        torch.cuda.synchronize()
    finally:
        g.lib().gsb200_set_sm_limit(0)
    assert all(torch.equal(x, y) for x, y in zip(got, ref)) and g.device_status()[0] == 0


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_wgrad_any_scales(dt):
    """Scales that are no powers of two: the restored element is rounded to dY's type, once."""
    g = need_lib()
    gen = torch.Generator().manual_seed(8)
    m, n, k = 700, 136, 300
    q, s = g.fp8_block_quantize(rnd(gen, m, k).cuda())
    s = s * (0.5 + torch.rand(s.shape, generator=gen).cuda())
    dy = rnd(gen, m, n).to(dt).cuda()
    want, mag = block8.wgrad(dy, q, s)
    tiny = 2.0 ** -25 * dy.double().abs().sum(0)[:, None] if dt == torch.float16 else 0.0
    dw = g.gemm_fp8_block_wgrad(dy, q, s)
    assert bool(((dw.double() - want).abs() <= (eps(dt) + 2.0 ** -23 + (m + 160) * 2.0 ** -23) * mag + tiny).all())


def test_wgrad_places_every_element_and_leaves_the_rest():
    g = need_lib()
    m, n, k = 200, 300, 400
    for i, j, l in [(0, 0, 0), (199, 299, 399), (63, 127, 255), (64, 128, 256), (130, 257, 130), (77, 63, 64), (10, 200, 17)]:
        dy = torch.zeros(m, 304, dtype=torch.bfloat16, device="cuda")[:, :n]
        q = torch.zeros(m, k, dtype=torch.uint8, device="cuda")
        dy[i, j] = 3.0
        q[i, l] = 0x40
        s = torch.exp2((torch.arange(m * 4, device="cuda") % 9 - 4).float()).view(m, 4)
        buf = torch.full((n + 1, 413), 9.0, device="cuda")
        out = g.gemm_fp8_block_wgrad(dy, q.view(F8), s, out=buf[:n, 5:5 + k])
        want = torch.full_like(buf, 9.0)
        want[:n, 5:5 + k] = 0
        want[j, 5 + l] = 6 * s[i, l // 128]
        assert torch.equal(buf, want) and out.data_ptr() == buf[:n, 5:].data_ptr()


def test_wgrad_nan_and_rows_behind_the_batch():
    g = need_lib()
    gen = torch.Generator().manual_seed(9)
    m, n, k = 90, 136, 200
    q, s = g.fp8_block_quantize(rnd(gen, m, k).cuda())
    dy = rnd(gen, m, n).half().cuda()
    ref = g.gemm_fp8_block_wgrad(dy, q, s)
    dbuf = torch.full((m + 70, 160), math.nan, dtype=torch.float16, device="cuda")
    qbuf = torch.full((m + 70, 256), 0x7f, dtype=torch.uint8, device="cuda")
    sbuf = torch.full((m + 70, 8), math.nan, device="cuda")
    dbuf[:m, :n], qbuf[:m, :k], sbuf[:m, :2] = dy, q.view(torch.uint8), s
    assert torch.equal(g.gemm_fp8_block_wgrad(dbuf[:m, :n], qbuf.view(F8)[:m, :k], sbuf[:m, :2]), ref)
    dy[89, 130] = math.inf
    q.view(torch.uint8)[5, 199] = 0x7f
    nan = ~torch.isfinite(g.gemm_fp8_block_wgrad(dy, q, s))
    want = torch.zeros_like(nan)
    want[130, :] = True
    want[:, 199] = True
    assert torch.equal(nan, want)


def test_wgrad_of_no_rows():
    g = need_lib()
    e = lambda *sh, dtype: torch.empty(*sh, dtype=dtype, device="cuda")
    args = e(0, 24, dtype=torch.float16), e(0, 40, dtype=F8), e(0, 1, dtype=torch.float32)
    assert bool((g.gemm_fp8_block_wgrad(*args) == 0).all())
    out = torch.ones(24, 40, device="cuda")
    g.gemm_fp8_block_wgrad(*args, out=out, accumulate=True)
    assert bool((out == 1).all())
    g.gemm_fp8_block_wgrad(*args, out=out)
    assert bool((out == 0).all())


# ---- SwiGLU ------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m,f", SIZES)
def test_swiglu_and_its_gradient(m, f, dt):
    g = need_lib()
    gen = torch.Generator().manual_seed(m * 7 + f)
    gate, up, dh = ((rnd(gen, m, f) * c).to(dt).cuda() for c in (3.0, 1.0, 0.1))
    (hq, hs), (gq, gs), (uq, us) = g.swiglu_fp8_block(gate, up)
    for (q, s), x in (((gq, gs), gate), ((uq, us), up)):
        want_q, want_s = g.fp8_block_quantize(x)
        assert torch.equal(q.view(torch.uint8), want_q.view(torch.uint8)) and torch.equal(s, want_s)
    # h: within an E4M3 rounding (2^-4, or half the least step 2^-9 of the scale) of the exact value; fp32's own error is far below
    h, want = block8.values(hq, hs), block8.swiglu(gate.double(), up.double())
    sp = block8.spread(hs, 1, m, f)
    assert bool(((h - want).abs() <= (2.0 ** -4 * want.abs()).maximum(2.0 ** -10 * sp) * (1 + 2.0 ** -15)).all())
    top = torch.nn.functional.pad(want.abs(), (0, -f % 128)).view(m, -1, 128).amax(2)
    slack = 1 + 2.0 ** -19
    assert bool((top <= 448 * hs.double() * slack).all())
    assert bool(((top * slack > 224 * hs.double()) | (hs == 2.0 ** -126) | (top == 0)).all())
    # gradient, from the values that the checkpoints stand for
    gv, uv = block8.values(gq, gs), block8.values(uq, us)
    wg, wu = block8.swiglu_bwd(dh.double(), gv, uv)
    dg, du, dgq, duq = g.swiglu_fp8_block_bwd(dh, gq, gs, uq, us, quantize=True)
    sig = torch.sigmoid(gv)
    mag = (dh.double() * uv * sig).abs() * (1 + (gv * (1 - sig)).abs())
    tiny = 2.0 ** -25 if dt == torch.float16 else 2.0 ** -133
    # sigmoid: exponential 2 ulp, sum, quotient 2 ulp; four more roundings of products and sums: within 16 2^-23 in all
    assert bool(((dg.double() - wg).abs() <= eps(dt) * wg.abs() + 2.0 ** -19 * mag + tiny).all())
    assert bool(((du.double() - wu).abs() <= (eps(dt) + 2.0 ** -19) * wu.abs() + tiny).all())
    for (q, s), x in ((dgq, dg), (duq, du)):
        want_q, want_s = g.fp8_block_quantize(x)
        assert torch.equal(q.view(torch.uint8), want_q.view(torch.uint8)) and torch.equal(s, want_s)
    two = g.swiglu_fp8_block_bwd(dh, gq, gs, uq, us)
    assert torch.equal(two[0], dg) and torch.equal(two[1], du)


def test_swiglu_gradient_is_the_difference_quotient():
    """The 64-bit formula that the kernel is held to, against central differences (step 2^-12: error of the quotient below
    2^-24 times the third derivative, which is below 1, and rounding below 2^-40)."""
    gen = torch.Generator().manual_seed(2)
    gate, up, dh = (torch.randn(50, 60, generator=gen, dtype=torch.float64) * c for c in (4.0, 1.0, 1.0))
    dg, du = block8.swiglu_bwd(dh, gate, up)
    t = 2.0 ** -12
    qg = dh * (block8.swiglu(gate + t, up) - block8.swiglu(gate - t, up)) / (2 * t)
    qu = dh * (block8.swiglu(gate, up + t) - block8.swiglu(gate, up - t)) / (2 * t)
    assert bool(((dg - qg).abs() <= 2.0 ** -24 * (dh * up).abs() + 2.0 ** -36).all()) and bool(((du - qu).abs() <= 2.0 ** -36).all())


def test_swiglu_far_gates_and_nan():
    g = need_lib()
    gate = torch.tensor([[-1e4, -100.0, -88.0, -20.0, 20.0, 88.0, 100.0, 1e4, math.nan, 1.0, 0.0, -0.0]], device="cuda").repeat(3, 1)
    up = torch.ones_like(gate)
    (hq, hs), (gq, gs), (uq, us) = g.swiglu_fp8_block(gate, up)
    h = g.fp8_block_dequantize(hq, hs, dtype=torch.float32)
    assert bool(h[:, 8].isnan().all()) and bool(torch.isfinite(h[:, [i for i in range(12) if i != 8]]).all())
    dg, du = g.swiglu_fp8_block_bwd(torch.ones_like(gate), gq, gs, uq, us)
    assert bool(dg[:, 8].isnan().all()) and bool(torch.isfinite(dg[:, [i for i in range(12) if i != 8]]).all())
    assert bool((dg[:, 0] == 0).all()) and bool((dg[:, 7] == 1).all())


@pytest.mark.parametrize("dt", TYPES)
def test_swiglu_gates_where_the_sigmoid_leaves_fp32(dt):
    """e^-g passes fp32's range at g = -88.7, and 1 / e^-g its normal numbers at -87.3: from there on the sigmoid may be 0 instead of its value, which is below
    2^-125 (1.00001 of it).  Before that its exponent is rounded at |g| log2 e < 128: 2^-18 relative, and as much for the rest."""
    g = need_lib()
    gate = torch.linspace(-92, -80, 256).to(dt).repeat(2, 1).cuda()
    up = torch.stack([torch.ones(256), torch.full((256,), 3e4)]).to(dt).cuda()
    (hq, hs), (gq, gs), (uq, us) = g.swiglu_fp8_block(gate, up)
    h, want = block8.values(hq, hs), block8.swiglu(gate.double(), up.double())
    lost = (gate.double() * up.double()).abs() * 2.0 ** -125
    assert bool(((h - want).abs() <= (2.0 ** -4 * want.abs()).maximum(2.0 ** -10 * block8.spread(hs, 1, 2, 256)) * (1 + 2.0 ** -15) + lost).all())
    dh = torch.ones_like(gate)
    wg, wu = block8.swiglu_bwd(dh.double(), block8.values(gq, gs), block8.values(uq, us))
    dg, du = g.swiglu_fp8_block_bwd(dh, gq, gs, uq, us)
    tiny = 2.0 ** -25 if dt == torch.float16 else 2.0 ** -133
    gv, uv = block8.values(gq, gs), block8.values(uq, us)
    for got, w, lost in ((dg, wg, (uv * (1 + gv.abs())).abs() * 2.0 ** -125), (du, wu, gv.abs() * 2.0 ** -125)):
        assert bool(((got.double() - w).abs() <= (eps(dt) + 2.0 ** -16) * w.abs() + lost + tiny).all())


def test_swiglu_views():
    """gate and up as the halves of one product's output, rows that are not on 16-byte boundaries."""
    g = need_lib()
    gen = torch.Generator().manual_seed(12)
    for f in (256, 333):
        both = rnd(gen, 41, 2 * f).bfloat16().cuda()
        got = g.swiglu_fp8_block(both[:, :f], both[:, f:])
        want = g.swiglu_fp8_block(both[:, :f].contiguous(), both[:, f:].contiguous())
        for (q, s), (wq, ws) in zip(got, want):
            assert torch.equal(q.view(torch.uint8), wq.view(torch.uint8)) and torch.equal(s, ws)


# ---- together ----------------------------------------------------------------------------------------------------------------------
def _mlp_step(g, x, w1g, w1u, w2, dy):
    """Forward and backward of a gated feed-forward with 8-bit checkpoints, as a training step calls it."""
    c, (wg, wu, wd) = x.dtype, (g.fp8_block_quantize(w, rows=128) for w in (w1g, w1u, w2))
    xq, xs = g.fp8_block_quantize(x)
    gate = g.gemm_fp8_block(xq, wg[0], xs, wg[1], dtype=c)
    up = g.gemm_fp8_block(xq, wu[0], xs, wu[1], dtype=c)
    (hq, hs), gc, uc = g.swiglu_fp8_block(gate, up)
    y = g.gemm_fp8_block(hq, wd[0], hs, wd[1], dtype=c)
    dq, ds = g.fp8_block_quantize(dy)
    dh = g.gemm_fp8_block(dq, wd[0], ds, wd[1], dtype=c, b_transposed=True)
    dw2 = g.gemm_fp8_block_wgrad(dy, hq, hs)
    dg, du, dgq, duq = g.swiglu_fp8_block_bwd(dh, *gc, *uc, quantize=True)
    dx = g.gemm_fp8_block(dgq[0], wg[0], dgq[1], wg[1], dtype=torch.float32, b_transposed=True)
    dx += g.gemm_fp8_block(duq[0], wu[0], duq[1], wu[1], dtype=torch.float32, b_transposed=True)
    return y, dx, g.gemm_fp8_block_wgrad(dg, xq, xs), g.gemm_fp8_block_wgrad(du, xq, xs), dw2


def _mlp_data(m, d, f, dt, seed=1):
    gen = torch.Generator().manual_seed(seed)
    return [rnd(gen, m, d).to(dt).cuda(), (rnd(gen, f, d) * d ** -0.5).cuda(), (rnd(gen, f, d) * d ** -0.5).cuda(), (rnd(gen, d, f) * f ** -0.5).cuda(),
            (rnd(gen, m, d) * 0.01).to(dt).cuda()]


@pytest.mark.parametrize("m,d,f,dt", [(200, 256, 512, torch.bfloat16), (333, 136, 264, torch.float16), (1, 128, 128, torch.bfloat16)])
def test_training_step_gradients(m, d, f, dt):
    """Outputs and gradients of a whole feed-forward against autograd in 64 bits.  Each quantisation is off by up to 2^-4 of an element and
    2^-5 on the average; the errors of a sum's terms are independent, so a result is off by about the root of the number of quantised factors on
    its path (at most six) times 2^-5.3 (uniform in +-2^-4 relative at worst) in the 2-norm: 0.062, with 30 % on top."""
    g = need_lib()
    x, wg, wu, wd, dy = _mlp_data(m, d, f, dt)
    got = _mlp_step(g, x, wg, wu, wd, dy)
    leaves = [t.double().requires_grad_() for t in (x, wg, wu, wd)]
    X, G, U, D = leaves
    y = (torch.nn.functional.silu(X @ G.t()) * (X @ U.t())) @ D.t()
    y.backward(dy.double())
    for name, a, b in zip(("y", "dx", "dwg", "dwu", "dwd"), got, (y.detach(), X.grad, G.grad, U.grad, D.grad)):
        rel = float((a.double() - b).norm() / b.norm())
        assert rel <= 0.08, (name, rel)
    assert g.device_status()[0] == 0


def test_training_step_streams_and_graphs():
    """The same bytes on a second stream, from a graph replayed over changing inputs, and with two graphs one after the other."""
    g = need_lib()
    sets = [_mlp_data(300, 256, 384, torch.bfloat16, seed=s) for s in (1, 2)]
    want = [[t.clone() for t in _mlp_step(g, *v)] for v in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [_mlp_step(g, *v) for v in sets]
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    ins = [t.clone() for t in sets[0]]
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _mlp_step(g, *ins)
        graphs.append((graph, out))
    for v, ref in list(zip(sets, want)) * 2:
        for t, x in zip(ins, v):
            t.copy_(x)
        for graph, out in graphs:
            graph.replay()
            assert all(torch.equal(x, y) for x, y in zip(out, ref))


def test_offsets_beyond_32_bits():
    """The last rows of a checkpoint of more than 2^31 elements."""
    g = need_lib()
    rows, k = 140000, 16384                                # 2.3e9 elements
    q = torch.zeros(rows, k, dtype=torch.uint8, device="cuda")
    s = torch.ones(rows, k // 128, device="cuda")
    gen = torch.Generator().manual_seed(1)
    x = rnd(gen, 128, k).cuda()
    g.fp8_block_quantize(x, out=q[-128:].view(F8), out_scale=s[-128:])
    tail = g.fp8_block_dequantize(q.view(F8), s, dtype=torch.float16)[-128:]
    assert torch.equal(tail, g.fp8_block_dequantize(q[-128:].view(F8), s[-128:], dtype=torch.float16))
    assert float((tail.double() - x.double()).norm() / x.double().norm()) < 0.05
    dy = torch.zeros(rows, 8, dtype=torch.bfloat16, device="cuda")
    dy[-128:] = 1.0
    dw = g.gemm_fp8_block_wgrad(dy, q.view(F8), s)
    ref = g.gemm_fp8_block_wgrad(dy[-128:], q[-128:].view(F8), s[-128:])
    assert float((dw - ref).abs().max()) <= 128 * 2.0 ** -23 * float(x.abs().sum(0).max())
    b, sb = g.fp8_block_quantize(rnd(gen, 16, k).cuda(), rows=128)
    c = g.gemm_fp8_block(q.view(F8), b, s, sb)
    assert torch.equal(c[-128:], g.gemm_fp8_block(q[-128:].view(F8), b, s[-128:], sb)) and bool((c[:-128] == 0).all())


# ---- the native call path ----------------------------------------------------------------------------------------------------------
def test_native_path_gives_the_bytes_of_the_checked_path():
    """Every operator through csrc/binding.cpp and through its checked Python function, aligned and ragged widths, given outputs."""
    g = need_lib()
    from gigaslop_b200 import _lib, ops
    n = _lib.native
    assert n is not None
    same = lambda a, b: a.shape == b.shape and a.stride() == b.stride() and a.dtype == b.dtype and torch.equal(a.view(torch.uint8) if a.dtype == F8 else a, b.view(torch.uint8) if b.dtype == F8 else b)
    gen = torch.Generator().manual_seed(21)
    for m, f, o in ((70, 256, 384), (33, 200, 72), (1, 128, 8), (5, 333, 130)):
        x = rnd(gen, m, f).half().cuda()
        for rows in (1, 128):
            a, b = n.block_quantize(x, rows, None, None), ops._checked_fp8_block_quantize(x, rows, None, None)
            assert same(a[0], b[0]) and same(a[1], b[1])
            assert same(n.block_dequantize(*a, rows, _lib.BF16, None), ops._checked_fp8_block_dequantize(*b, rows, torch.bfloat16, None))
        q, s = g.fp8_block_quantize(x)
        for tr in (False, True):
            w, sw = g.fp8_block_quantize(rnd(gen, *((f, o) if tr else (o, f))).cuda(), rows=128)
            for code, dt in ((_lib.F16, torch.float16), (_lib.BF16, torch.bfloat16), (_lib.F32, torch.float32)):
                assert same(n.block_gemm(q, w, s, sw, None, code, tr), ops._checked_gemm_fp8_block(q, w, s, sw, None, dt, tr))
                out = torch.empty(m, o, dtype=dt, device="cuda")
                assert n.block_gemm(q, w, s, sw, out, code, tr) is out and same(out, ops._checked_gemm_fp8_block(q, w, s, sw, torch.empty_like(out), dt, tr))
        dy = rnd(gen, m, (o + 7) // 8 * 8).half().cuda()[:, :o]
        assert same(n.block_wgrad(dy, q, s, None, False), ops._checked_gemm_fp8_block_wgrad(dy, q, s, None, False))
        acc, acc2 = (torch.ones(o, f, device="cuda") for _ in range(2))
        assert n.block_wgrad(dy, q, s, acc, True) is acc and same(acc, ops._checked_gemm_fp8_block_wgrad(dy, q, s, acc2, True))
        a, b = n.block_swiglu(x, x), ops._checked_swiglu_fp8_block(x, x)
        assert all(same(u, v) for p, r in zip(a, b) for u, v in zip(p, r))
        a, b = n.block_swiglu_bwd(x, q, s, q, s), ops._checked_swiglu_fp8_block_bwd(x, q, s, q, s, False)
        assert same(a[0], b[0]) and same(a[1], b[1])


def test_native_path_leaves_the_rest_to_the_checked_path():
    g = need_lib()
    from gigaslop_b200 import _lib
    n = _lib.native
    z = lambda *sh, dt=torch.float16: torch.zeros(*sh, dtype=dt, device="cuda")
    x, q, s, w, sw, dy = z(40, 256), z(40, 256, dt=torch.uint8), z(40, 2, dt=torch.float32), z(64, 256, dt=torch.uint8), z(1, 2, dt=torch.float32), z(40, 64)
    for i, r in enumerate((n.block_quantize(x.t(), 1, None, None), n.block_quantize(x, 2, None, None), n.block_quantize(x[:0], 1, None, None), n.block_quantize(x.int(), 1, None, None),
              n.block_quantize(x, 1, q[:, :8], None), n.block_quantize(x, 1, None, s[:, :1]),
              n.block_dequantize(q, s[:, :1], 1, 0, None), n.block_dequantize(q, s, 128, 0, None), n.block_dequantize(q, s, 1, -1, None), n.block_dequantize(x, s, 1, 0, None),
              n.block_gemm(q, w[:, :240], s, sw, None, 0, False), n.block_gemm(q, w, s, sw, None, 0, True), n.block_gemm(q, w, s, sw, None, -1, False), n.block_gemm(q, w, s, s, None, 0, False),
              n.block_gemm(q, w, s, sw, x, 0, False), n.block_gemm(q, w, s, sw, None, 0, 0),
              n.block_wgrad(dy.float(), q, s, None, False), n.block_wgrad(dy, q, s, None, True), n.block_wgrad(dy[:39], q, s, None, False), n.block_wgrad(dy, q, s, x, False),
              n.block_swiglu(x, x[:, :128]), n.block_swiglu(x, x.float()), n.block_swiglu(x.cpu(), x), n.block_swiglu_bwd(x, q, s, q[:39], s), n.block_swiglu_bwd(x, q, s, q, s[:, :1]))):
        assert r is None, i
