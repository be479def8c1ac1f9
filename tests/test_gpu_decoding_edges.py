"""GPU tests of the decoding operators where their statements (include/faiss_amd_c.h) are easiest to break: codes and scales that
are no numbers, sums over scores and scales far apart, lengths past the table, sizes past a launch, blocks that come back.

The attention is compared with the 64-bit form of test_gpu_decoding.py under the tolerances that are derived there."""
import math

import pytest
import torch

from faiss_amd import decoding
from test_gpu_decoding import I32, check, filled, ints, paged, reference

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ codes that are no numbers
@pytest.mark.parametrize("d, hq, length, nq, at", [
    (64, 1, 300, 200, 110),    # whole tiles of the later wavefronts, masked by the first one's rows
    (64, 1, 300, 200, 70), (128, 1, 300, 200, 128), (192, 1, 300, 200, 110), (256, 2, 300, 100, 210), (96, 1, 140, 100, 60),
    (128, 3, 1500, 170, 1400), (64, 1, 5000, 200, 4830),  # the last one in a split context
    (64, 2, 300, 5, 296), (128, 16, 90, 2, 88)])         # few rows: straight from memory
def test_attend_nan_value_codes_anywhere(res, d, hq, length, nq, at):
    """a value of code NaN reaches every row that sees it and no other, whichever tiles of the row's workgroup mask it"""
    c, table = paged(res, [length], 16, 1, d, "e4m3", 3)
    g = torch.Generator(device="cuda")
    g.manual_seed(at)
    q = torch.randn((nq, hq, d), generator=g, device="cuda").bfloat16()
    offs = ints([0, nq])
    want, wl, tol = reference(c, q, table, [length], [0, nq], 1 / math.sqrt(d), True)
    sees = torch.arange(nq) + length - nq + 1 > at
    raw = c.v_codes.view(torch.uint8)
    for code in (0x7f, 0xff):
        raw[int(table[0, at // 16]), 0, 50, at % 16] = code
        got, lse = c.attend(q, table, ints([length]), query_offsets=offs, return_lse=True)
        assert bool(got[sees][:, :, 50].isnan().all())
        check(got[~sees], lse[~sees], want[~sees], wl[~sees], tol[~sees])
