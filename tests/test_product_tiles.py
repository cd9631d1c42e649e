"""matmul_fp8 by every one of its tiles, in every type, from one step of K to many.

Which tiles a call takes goes by its sizes (csrc/product.hip); dsa_product_tile says it
without a device, so that the sizes below are known to reach each of them.
"""
import pytest
import torch

import dsa_amd
from dsa_amd import _lib
from dsa_amd.rotary import DTYPES
from test_gpu_product import E4M3, check

BF, HALF, FULL = torch.bfloat16, torch.float16, torch.float32
CUS = 256  # of an MI355X
# One block of K, an even and an odd number of them, as many as a step of four has and one
# more, more than the scales that come at once, and many; 16, 272, .. end inside a block.
KS = (16, 128, 256, 272, 400, 528, 1040, 1552, 7184)

# M and N by the number of the tiles; odd, so that rows and columns end inside a tile.
SHORT = (16, 128, 256)
SIZES = {
    0: {k: (37, 141) for k in KS},                                                            # 16 by 16, five stages
    1: {k: (99, 1157) for k in KS if k not in SHORT},                                         # 16 by 16, two to a CU
    2: {k: (4118, 15) for k in KS if k not in (16, 128)},                                     # 16 columns by 32 rows
    3: {k: (13, 4109) for k in KS if k not in SHORT},                                         # 32 by 16, four stages
    4: {k: (13, 8203) for k in KS if k not in SHORT},                                         # 32 by 16, two to a CU
    5: {k: (17, 4133) for k in KS if k not in SHORT},                                         # 32 by 32
    6: {256: (9, 4101), **{k: (4139, 33) for k in KS if k not in SHORT + (272,)}},            # 64 by 32
    7: {k: (33, 8303) for k in KS if k not in (16, 128, 272)} | {k: (9, 4111) for k in (16, 128)} | {272: (4201, 33)},  # 64 by 64
    8: {k: (29, 16421) for k in KS},                                                          # 128 by 32
    9: {k: (33, 16457) for k in KS},                                                          # 128 by 64
    10: {k: (67, 16627) for k in KS},                                                         # 128 by 96
    11: {k: (98, 17049) for k in KS},                                                         # 128 by 128
    12: {k: (131, 16929) for k in KS if k != 7184} | {7184: (132, 16621)},                    # 128 by 160
    13: {k: (163, 16607) for k in KS if k != 7184} | {7184: (193, 21774)},                    # 128 by 256
    14: {k: (515, 22179) for k in SHORT} | {k: (515, 24633) for k in (272, 400)}              # 256 by 256, the rest in halves
        | {k: (782, 16138) for k in (528, 1040)} | {1552: (515, 26169), 7184: (1283, 14649)},  # 528, 1040: no rest
}


def cases(wide):
    have = _lib.load().dsa_product_tiles(DTYPES[FULL if wide else BF])
    for tile, sizes in SIZES.items():
        for k, (m, n) in sizes.items():
            if have >> tile & 1:
                yield tile, m, n, k


ALL = [(dtype, *case) for dtype in (BF, HALF, FULL) for case in cases(dtype == FULL)]


@pytest.mark.parametrize("dtype", (BF, HALF, FULL))
def test_every_tile_has_its_sizes(dtype):
    lib, name = _lib.load(), DTYPES[dtype]
    reached = {}
    for of, tile, m, n, k in ALL:
        if of is dtype:
            assert lib.dsa_product_tile(m, n, k, name, CUS) == tile, (tile, m, n, k)
            reached.setdefault(tile, set()).add(k)
    assert sum(1 << tile for tile in reached) == lib.dsa_product_tiles(name)
    for tile, ks in reached.items():  # an odd and an even number of steps of a block, and many
        assert max(ks) == 7184 and {-(-k // 128) % 2 for k in ks} == {0, 1} and any(k % 128 for k in ks), tile


def test_the_choice_refuses_what_the_call_refuses():
    lib = _lib.load()
    for args in [(0, 8, 16, 0, 256), (8, 0, 16, 0, 256), (8, 8, 8, 0, 256), (8, 8, 1 << 20, 0, 256), (8, 8, 16, 3, 256),
                 (8, 8, 16, 0, 0), ((1 << 24) + 1, 8, 16, 0, 256), (1 << 19, (1 << 18) + 1, 16, 0, 256)]:
        assert lib.dsa_product_tile(*args) < 0 and lib.dsa_last_error()
    assert lib.dsa_product_tiles(3) == 0 and lib.dsa_product_tiles(-1) == 0
    for dtype in (0, 1, 2):  # the largest calls have tiles
        for m, n in ((1 << 24, 1 << 13), (1 << 13, 1 << 24), (1 << 24, 1), (1, 1 << 24)):
            assert lib.dsa_product_tiles(dtype) >> lib.dsa_product_tile(m, n, (1 << 20) - 16, dtype, CUS) & 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, tile, M, N, K", ALL)
def test_against_64_bits(dtype, tile, M, N, K):
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    assert _lib.load().dsa_product_tile(M, N, K, DTYPES[dtype], cus) == tile
    g = torch.Generator(device="cuda").manual_seed(K)
    codes = [(torch.randn(rows, K, generator=g, device="cuda") * 100).clamp(-448, 448).to(E4M3) for rows in (M, N)]
    scales = [torch.exp(torch.randn(rows, -(-K // 128), generator=g, device="cuda")) for rows in (M, -(-N // 128))]
    args = codes[0], scales[0], codes[1], scales[1] / 1024
    check(dsa_amd.matmul_fp8(*args, dtype=dtype), *args, cut=True)
