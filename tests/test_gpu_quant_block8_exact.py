"""Block-scaled products and weight gradients whose every sum is exact: elements that are small integers, scales that are powers of two, and
sums of magnitudes below 2^24 units, so that no order of fp32 additions rounds and one lost, repeated or misplaced term shows."""
import pytest
import torch

from util import need_lib

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def whole(gen, m, n, most=1):
    """[m, n] integers in -most .. most as E4M3 whose rows are on 16-byte boundaries."""
    v = torch.randint(-most, most + 1, (m, n), generator=gen, device="cuda", dtype=torch.int8)
    out = torch.zeros(m, (n + 15) // 16 * 16, dtype=torch.uint8, device="cuda").view(F8)[:, :n]
    out.copy_(v.to(torch.float32))
    return out


def powers(gen, m, n, lo, hi):
    return torch.exp2(torch.randint(lo, hi + 1, (m, n), generator=gen, device="cuda").float())


def spread(s, rows, m, k):
    return s.double().repeat_interleave(rows, 0)[:m].repeat_interleave(128, 1)[:, :k]


def gemm_case(seed, m, n, k, transposed):
    """(A, B, scale_a, scale_b, the product in float64): every K block has scales of its own, so one that is used for another's block shows."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    nb = lambda v: (v + 127) // 128
    a, sa = whole(gen, m, k), powers(gen, m, nb(k), 0, 3)
    shape = (k, n) if transposed else (n, k)
    b, sb = whole(gen, *shape), powers(gen, nb(shape[0]), nb(shape[1]), -2, 1)
    av, bv = a.double() * spread(sa, 1, m, k), b.double() * spread(sb, 128, *shape)
    assert k * 8 * 2 * 4 < 2 ** 24                         # (in units of 2^-2)
    return a, b, sa, sb, av @ (bv if transposed else bv.t())


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("m,n,k", [(5121, 1030, 2049), (20000, 390, 1300), (1500, 4097, 900), (12000, 384, 384)])
def test_gemm_takes_each_block_with_its_own_scales(m, n, k, transposed):
    """Many K blocks on CTA pairs of both widths: the scales' places in shared memory are used over and over."""
    g = need_lib()
    a, b, sa, sb, want = gemm_case(m + n + k, m, n, k, transposed)
    for _ in range(3):
        assert torch.equal(g.gemm_fp8_block(a, b, sa, sb, dtype=torch.float32, b_transposed=transposed).double(), want)
    assert g.device_status()[0] == 0


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k", [(5121, 1030, 520), (5000, 2048, 300), (20000, 390, 260), (12000, 384, 384), (65, 19000, 130)])
@pytest.mark.parametrize("off,pad", [(0, 0), (1, 2), (3, 8), (8, 9)])
def test_gemm_on_pairs_into_rows_of_no_alignment(off, pad, m, n, k, dt, transposed):
    """So many tiles that CTA pairs take them, into views whose base or stride TMA cannot address: every element, rounded once, and nothing beside them."""
    g = need_lib()
    a, b, sa, sb, want = gemm_case(n + k, m, n, k, transposed)
    ld = n + off + pad
    buf = torch.full((m + 1, ld), 5.0, dtype=dt, device="cuda")
    out = buf[:m, off:off + n]
    assert g.gemm_fp8_block(a, b, sa, sb, out=out, b_transposed=transposed) is out
    assert torch.equal(out, want.to(dt))
    buf[:m, off:off + n] = 5.0
    assert bool((buf == 5.0).all())
    assert g.device_status()[0] == 0


# parts of the batch (with how many segments, at 64 rows a step); one or two accumulators
WGRAD = [(40001, 40, 136), (33000, 264, 200),              # 74 and 37 parts
         (65536, 2048, 512), (65536, 1536, 2048),          # 9 parts of 114 steps, 3 of 341
         (9000, 200, 9500), (9000, 256, 9501),             # one part of 141 steps on one accumulator, straight to dW and through the workspace
         (30000, 250, 2600), (12345, 9704, 1000)]          # 6 parts of 78 steps on one accumulator; one part of 193 on two


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", WGRAD)
def test_wgrad_adds_every_term_once(m, n, k, dt):
    g = need_lib()
    gen = torch.Generator(device="cuda").manual_seed(m + n + k)
    q, s = whole(gen, m, k), powers(gen, m, (k + 127) // 128, 0, 3)
    dy = torch.zeros(m, (n + 7) // 8 * 8, dtype=dt, device="cuda")[:, :n]
    dy.copy_(torch.randint(-1, 2, (m, n), generator=gen, device="cuda", dtype=torch.int8))
    assert m * 8 + 1000 < 2 ** 24
    want = dy.double().t() @ (q.double() * spread(s, 1, m, k))
    dw = g.gemm_fp8_block_wgrad(dy, q, s)
    assert torch.equal(dw.double(), want)
    start = torch.randint(-1000, 1001, (n, k), generator=gen, device="cuda").float()
    acc = start.clone()
    g.gemm_fp8_block_wgrad(dy, q, s, out=acc, accumulate=True)
    assert torch.equal(acc.double(), want + start.double())
    assert g.device_status()[0] == 0
