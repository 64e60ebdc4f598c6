"""The 8-bit product (ivf_sq_matmul) on the tensor cores: every tile of tokens
and every way of splitting k that the library chooses on 148 SMs, against the
product in 64 bits (tolerances derived in test_gpu_sq.py).

A product takes a tile of 16, 32, 64, 128 or 256 tokens by 128 channels; the
sizes below are ones for which the choice falls on the tile they are listed
under.  Each tile is met with fewer tokens than it has, with all of them, with
one more (two token tiles, the second nearly empty) and with more than eight
token tiles (bands); with fewer tiles than the GPU holds at once and with more
than twice as many (both accumulators of a block used again); with k up to 256
and above (two ways of converting the sums)."""
import pytest
import torch

import insitu_b200 as ib
from test_gpu_sq import TYPES, check_product, codes_of, scales_of

pytestmark = pytest.mark.gpu

WHOLE = {
    16: [(9, 129, 129), (16, 129, 257), (17, 129, 64), (15, 80001, 255), (16, 80001, 257), (1000, 129, 257)],
    32: [(17, 12001, 129), (31, 12001, 257), (32, 12001, 64), (33, 7777, 200), (32, 80001, 257), (65, 30001, 129),
         (5000, 129, 64), (2500, 129, 257)],
    64: [(33, 12001, 129), (63, 12001, 257), (64, 12001, 64), (65, 7777, 257), (64, 80001, 200), (129, 30001, 257),
         (4444, 513, 64), (9000, 129, 257)],
    128: [(65, 15001, 129), (127, 12001, 257), (128, 12001, 64), (129, 7777, 255), (128, 80001, 129),
          (257, 30001, 257), (4444, 1300, 64), (4444, 777, 257)],
    256: [(129, 15001, 1031), (255, 12001, 1031), (257, 7777, 1031), (256, 100003, 129), (512, 30001, 64),
          (513, 20011, 1031), (2049, 7777, 64), (2049, 7777, 257)],
}
# (m, n, k) that are computed in 2, 4, 6, 7 and 8 parts of k (as far as a tile has them)
SPLIT = {
    16: [(9, 6000, 2048), (17, 129, 1300), (16, 129, 2100), (35, 129, 2500), (145, 129, 5000)],
    32: [(17, 7777, 3500), (33, 2001, 1300), (32, 1300, 2100), (289, 129, 2600), (33, 777, 2048)],
    64: [(65, 7777, 2500), (577, 513, 2100), (131, 513, 2600), (64, 1300, 2048)],
    128: [(129, 9001, 3500), (128, 5000, 2500), (259, 1300, 4224), (1153, 257, 8400)],
    256: [(257, 4000, 5000), (515, 1300, 5000), (256, 1300, 16384)],
}


def check(m, n, k, ld, offset=0):
    a, b = codes_of(m, k, m + k, ld, offset), codes_of(n, k, n + k + 1, ld, offset)
    sa, sb = scales_of(m, 1), scales_of(n, 2)
    bias = torch.randn(n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    for t in TYPES:
        check_product(ib.sq_matmul(a, sa, b, sb, bias=bias, dtype=t), a, sa, b, sb, bias, t)
        # rows of the output at an odd distance, and at an even one: what is beside them stays
        for lo, width in ((1, n + n % 2 + 3), (2, n + n % 2 + 2)):
            wide = torch.full((m, width), 5.0, dtype=t, device="cuda")
            ib.sq_matmul(a, sa, b, sb, out=wide[:, lo:lo + n])
            check_product(wide[:, lo:lo + n], a, sa, b, sb, None, t)
            assert (wide[:, :lo] == 5).all() and (wide[:, lo + n:] == 5).all()


def cases(table):
    return [pytest.param(*s, id=f"{nt}-{s[0]}x{s[1]}x{s[2]}") for nt, sizes in table.items() for s in sizes]


@pytest.mark.parametrize("m,n,k", cases(WHOLE))
def test_tiles(cuda_ok, m, n, k):
    check(m, n, k, (k + 15) // 16 * 16)


@pytest.mark.parametrize("m,n,k", cases(SPLIT))
def test_split(cuda_ok, m, n, k):
    check(m, n, k, (k + 15) // 16 * 16)


@pytest.mark.parametrize("m,n,k", cases({nt: WHOLE[nt][1:2] + SPLIT[nt][-1:] for nt in WHOLE}))
def test_unaligned_rows(cuda_ok, m, n, k):
    """the same through the copy of rows that are not 16-byte aligned"""
    check(m, n, k, k + (k + 1) % 2, 3)
