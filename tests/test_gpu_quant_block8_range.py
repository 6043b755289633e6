"""Weight gradient from checkpoints whose scales are far from 1, against float64.  A restored element is exact whatever its (power-of-two) scale,
so the bounds are those of fp32 sums alone: n additions, each off by at most 2^-23 of the magnitudes summed so far, and one of each pass over the batch and
of each part."""
import pytest
import torch

from oracle import block8
from util import need_lib

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def codes(gen, m, k):
    """Every finite E4M3 code, subnormals among them; rows on 16-byte boundaries."""
    v = torch.randint(0, 256, (m, (k + 15) // 16 * 16), generator=gen, device="cuda", dtype=torch.uint8)
    v[(v & 0x7f) == 0x7f] = 0
    return v.view(F8)[:, :k]


def gradient(gen, m, n, dt):
    return (0.1 * torch.randn(m, (n + 7) // 8 * 8, generator=gen, device="cuda")).to(dt)[:, :n]


def bound(want, mag, additions):
    return 2.0 ** -24 * want.abs() + additions * 2.0 ** -23 * mag


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("t", [-100, -60, -36, -30, -24, -20, -15, 0, 8, 20, 100])
def test_wgrad_of_any_scale(t, dt):
    g = need_lib()
    gen = torch.Generator(device="cuda").manual_seed(t + 200)
    for m, n, k in ((700, 136, 300), (1000, 520, 257)):
        q, dy = codes(gen, m, k), gradient(gen, m, n, dt)
        s = torch.exp2(t + torch.randint(-3, 4, (m, (k + 127) // 128), generator=gen, device="cuda").float())
        want, mag = block8.wgrad(dy, q, s)
        dw = g.gemm_fp8_block_wgrad(dy, q, s)
        assert bool(((dw.double() - want).abs() <= bound(want, mag, m + 160)).all())
        assert torch.equal(dw, g.gemm_fp8_block_wgrad(dy, q, s))
    assert g.device_status()[0] == 0


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k,ld", [(700, 136, 300, 300), (3000, 600, 520, 520), (9001, 1000, 520, 523), (33000, 264, 200, 200), (8250, 9704, 1000, 1000),
                                      (4200, 9704, 1000, 1001), (4200, 9704, 1001, 1001), (64, 8, 128, 128), (1, 16, 40, 40)])
def test_wgrad_of_scales_far_apart(m, n, k, ld, dt):
    """Rows in four groups whose scales are 2^33 and more apart, and one of zeros (whose scale is 1), as padding leaves them.  Column j of dY belongs to
    group j % 6 (5: to all of them), so a dW row shows each group's terms by themselves."""
    g = need_lib()
    gen = torch.Generator(device="cuda").manual_seed(m + n + k)
    q, dy = codes(gen, m, k), gradient(gen, m, n, dt)
    group = torch.arange(m, device="cuda") // 16 % 5
    t = torch.tensor([3.0, -30.0, -70.0, -95.0, 0.0], device="cuda")[group]
    s = torch.exp2(t[:, None] - 5 * torch.arange((k + 127) // 128, device="cuda") % 4)
    zeros = (group == 4).nonzero()[:, 0]
    q.view(torch.uint8)[zeros] = 0
    s[zeros] = 1.0
    of = torch.arange(n, device="cuda") % 6
    dy = dy * ((of[None, :] == 5) | (of[None, :] == group[:, None]))
    pad = torch.zeros(m, (n + 7) // 8 * 8, dtype=dt, device="cuda")
    pad[:, :n] = dy
    dy = pad[:, :n]
    want, mag = block8.wgrad(dy, q, s)
    buf = torch.full((n, ld), float("nan"), device="cuda")
    dw = g.gemm_fp8_block_wgrad(dy, q, s, out=buf[:, :k])
    tol = bound(want, mag, m + 160 + 12)
    assert bool(((dw.double() - want).abs() <= tol).all()) and bool(buf[:, k:].isnan().all())
    again = g.gemm_fp8_block_wgrad(dy, q, s)
    assert torch.equal(again, dw)
    start = dw.double()
    g.gemm_fp8_block_wgrad(dy, q, s, out=dw, accumulate=True)      # (up to 12 passes of up to three segments are added to dW)
    assert bool(((dw.double() - want - start).abs() <= tol + 36 * 2.0 ** -23 * ((want + start).abs() + mag)).all()) and bool(buf[:, k:].isnan().all())
    assert g.device_status()[0] == 0


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(1000, 136, 300), (5000, 9704, 520), (9001, 1000, 520), (40000, 264, 200)])
@pytest.mark.parametrize("ts", [(-20, 10), (10, -20), (-60, -20, 20, 60, 100), (100, 60, 20, -20, -60), (None, -40), (-40, None), (0, 118), (118, -115), (None, None)])
def test_wgrad_of_scales_that_change_along_the_batch(ts, m, n, k, dt):
    """The first rows say nothing of the others: scales that grow, shrink, start or end with rows of zeros, up to the largest and the smallest.  Column
    j of dY belongs to one stretch of the batch."""
    g = need_lib()
    gen = torch.Generator(device="cuda").manual_seed(m + len(ts))
    q, dy = codes(gen, m, k), gradient(gen, m, n, dt)
    of_row = torch.arange(m, device="cuda") * len(ts) // m
    s = torch.exp2(torch.tensor([0.0 if t is None else float(t) for t in ts], device="cuda")[of_row][:, None] + torch.randint(-2, 3, (m, (k + 127) // 128), generator=gen, device="cuda"))
    for i, t in enumerate(ts):
        if t is None:
            q.view(torch.uint8)[of_row == i] = 0
            s[of_row == i] = 1.0
    dy = dy * (torch.arange(n, device="cuda")[None, :] % len(ts) == of_row[:, None])
    pad = torch.zeros(m, (n + 7) // 8 * 8, dtype=dt, device="cuda")
    pad[:, :n] = dy
    dy = pad[:, :n]
    want, mag = block8.wgrad(dy, q, s)
    dw = g.gemm_fp8_block_wgrad(dy, q, s)
    # (Every partial sum is within mag: below 2^127 none leaves fp32.  Above, the sum itself may: 448 2^120 alone does.  And an element beyond
    # bf16's largest number, 255 2^120, is infinite there, which makes every dW of its column one or, times 0, NaN.)
    none = (mag >= 2.0 ** 127) | (block8.values(q, s).abs() > torch.finfo(dt).max).any(0)[None, :] & (dt == torch.bfloat16)
    assert bool((((dw.double() - want).abs() <= bound(want, mag, m + 172)) | none).all())
    assert torch.equal(dw.view(torch.int32), g.gemm_fp8_block_wgrad(dy, q, s).view(torch.int32))
    assert g.device_status()[0] == 0


def test_wgrad_passes_from_a_graph_and_on_two_streams():
    """How many passes a call takes is for the device to find out: a captured call replayed over scales that need one, two and six, and calls that
    need different numbers side by side, give the bytes of calls by themselves."""
    g = need_lib()
    gen = torch.Generator(device="cuda").manual_seed(9)
    m, n, k = 5000, 520, 300
    q, dy = codes(gen, m, k), gradient(gen, m, n, torch.float16)
    row = torch.arange(m, device="cuda")[:, None] * torch.ones(1, 3, device="cuda")
    sets = [torch.exp2((row % 5) - 9), torch.exp2(30 * (row // 64 % 2) - 20), torch.exp2(100 - 25 * (row // 700))]
    want = [g.gemm_fp8_block_wgrad(dy, q, s) for s in sets]
    s = sets[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = g.gemm_fp8_block_wgrad(dy, q, s)
    for i in (0, 1, 2, 0, 2):
        s.copy_(sets[i])
        graph.replay()
        assert torch.equal(out, want[i])
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for st, x in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(g.gemm_fp8_block_wgrad(dy, q, x))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want[i % 3]) for i, a in enumerate(got))
    assert g.device_status()[0] == 0


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_wgrad_of_a_scale_that_is_no_number(dt):
    """An infinite or NaN scale, and a NaN element in a row of another pass, reach their own columns and no other; a scale of zero adds nothing."""
    g = need_lib()
    gen = torch.Generator(device="cuda").manual_seed(1)
    m, n, k = 300, 136, 384
    q, dy = codes(gen, m, k), gradient(gen, m, n, dt)
    q.view(torch.uint8)[q.view(torch.uint8) & 0x7f == 0] = 0x38              # (no zeros: infinity times zero is NaN too, but let it be one case)
    s = torch.exp2(torch.randint(-40, 1, (m, 3), generator=gen, device="cuda").float())
    s[5, 0], s[7, 1] = float("inf"), float("nan")
    q.view(torch.uint8)[9, 300] = 0x7f
    s[9, 2] = 2.0 ** -60
    s[11, 2] = 0.0
    q.view(torch.uint8)[7] = 0                             # (NaN all the same)
    dw = g.gemm_fp8_block_wgrad(dy, q, s)
    bad = torch.zeros(k, dtype=torch.bool, device="cuda")
    bad[:256] = True
    bad[300] = True
    assert bool((~torch.isfinite(dw) == bad[None, :]).all())
    want, mag = block8.wgrad(dy, q, torch.where(torch.isfinite(s), s, 0.0))
    err = (dw.double() - want).abs()
    assert bool((err <= bound(want, mag, m + 170))[:, ~bad].all())


def test_swiglu_gradient_in_fp32_down_to_the_last_exponential():
    """Gates to -88.7, where e^-g leaves fp32.  dup = dh g sigmoid(g): the exponential within 2 ulp (2^-22), the reciprocal within one (2^-23), and a sum and
    three products off by 2^-24 each, are 2^-22 (1 + 1/2 + 4/4) = 1.25 2^-21 in all; dgate has a difference, a multiply-add and a product more, and as much of its terms'
    magnitudes each at most."""
    g = need_lib()
    gate = torch.cat([torch.linspace(-88.7, -87.0, 200), torch.linspace(-87, 60, 312)]).cuda().view(4, 128)
    gen = torch.Generator(device="cuda").manual_seed(5)
    # (a gate per block of its own scale is not needed: a scale of g / 256 and the code of 256 give any fp32 gate, in blocks of one value)
    codes_, ones = torch.full((512, 128), 0x78, dtype=torch.uint8, device="cuda").view(F8), torch.full((512, 128), 0x38, dtype=torch.uint8, device="cuda").view(F8)
    gs = (gate.view(-1, 1) / 256).contiguous()
    us = torch.rand(512, 1, generator=gen, device="cuda") + 0.5
    dh = torch.randn(512, 128, generator=gen, device="cuda")
    dg, du = g.swiglu_fp8_block_bwd(dh, codes_, gs, ones, us)
    gv, uv = block8.values(codes_, gs), block8.values(ones, us)
    wg, wu = block8.swiglu_bwd(dh.double(), gv, uv)
    tiny = 2.0 ** -140                                     # (half of fp32's least step, 2^-149, times |g|, dh and u)
    assert bool(((du.double() - wu).abs() <= 1.25 * 2.0 ** -21 * wu.abs() + tiny).all())
    sig = torch.sigmoid(gv)
    mag = (dh.double() * uv * sig).abs() * (1 + (gv * (1 - sig)).abs())
    assert bool(((dg.double() - wg).abs() <= 4 * 1.25 * 2.0 ** -21 * mag + tiny).all())


def test_down_projection_gradient_of_small_activations():
    """SwiGLU of values about 1e-4: h is about 5e-9, its checkpoint's scales about 2^-34, far below what fp16 itself holds."""
    g = need_lib()
    gen = torch.Generator(device="cuda").manual_seed(3)
    m, f, n = 500, 384, 256
    gate, up = ((1e-4 * torch.randn(m, f, generator=gen, device="cuda")).half() for _ in range(2))
    (h, hs), _, _ = g.swiglu_fp8_block(gate, up)
    dy = gradient(gen, m, n, torch.float16)
    want, mag = block8.wgrad(dy, h, hs)
    dw = g.gemm_fp8_block_wgrad(dy, h, hs)
    assert float(mag.min()) > 0 and bool(((dw.double() - want).abs() <= bound(want, mag, m + 160)).all())
    exact = dy.double().t() @ block8.swiglu(gate.double(), up.double())
    assert float((dw.double() - exact).norm() / exact.norm()) <= 2.0 ** -4      # (each element of h is off by 2^-4 at most)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(65536, 2048, 512), (65536, 512, 512), (65536, 1536, 2048), (65536, 200, 1024), (8192, 4096, 4096), (9000, 256, 9472), (3000, 512, 512)])
def test_wgrad_truncation_stays_small(m, n, k, dt):
    """The header's bound on the sums: 2^-19 of the 2-norm.  (The tensor core's own sums of 7300 rows are 1.7 times as far off, with every shortened sum
    nearer to zero.)"""
    g = need_lib()
    gen = torch.Generator(device="cuda").manual_seed(m + n)
    q, s = g.fp8_block_quantize(torch.randn(m, k, generator=gen, device="cuda").to(dt))
    dy = gradient(gen, m, n, dt)
    want = dy.double().t() @ block8.values(q, s)
    dw = g.gemm_fp8_block_wgrad(dy, q, s)
    assert float((dw.double() - want).norm() / want.norm()) <= 2.0 ** -19
    assert g.device_status()[0] == 0
