"""Block-scaled products and weight gradients whose every sum is exact: elements that are small integers, scales that are powers of two, and
sums of magnitudes below 2^24 units, so that no order of fp32 additions rounds and one lost, repeated or misplaced term shows."""
import math

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
