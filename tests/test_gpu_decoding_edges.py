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


@pytest.mark.parametrize("d, hq, length, nq", [(64, 2, 300, 1), (64, 1, 300, 200), (128, 4, 2000, 3), (192, 1, 700, 90), (96, 2, 3000, 150)])
def test_attend_nan_codes_make_the_whole_row_nan(res, d, hq, length, nq):
    """every dimension and the log-sum, for keys and values, whether some rows mask the code's tile or all see it"""
    c, table = paged(res, [length], 16, 1, d, "e4m3", 3)
    q = torch.randn((nq, hq, d), device="cuda").bfloat16()
    want, wl, tol = reference(c, q, table, [length], [0, nq], 1 / math.sqrt(d), True)
    for at in (0, 63, length // 2, length - nq - 1, length - nq, length - nq // 2 - 1, length - 1):
        if at < 0:
            continue
        sees = torch.arange(nq) + length - nq + 1 > at
        for codes, where in ((c.k_codes, (0, at % 16, 7)), (c.v_codes, (0, d - 1, at % 16))):
            raw = codes.view(torch.uint8)[int(table[0, at // 16])]
            old = int(raw[where])
            raw[where] = 0xff
            got, lse = c.attend(q, table, ints([length]), query_offsets=ints([0, nq]), return_lse=True)
            raw[where] = old
            assert bool(got[sees].isnan().all()) and bool(lse[sees].isnan().all()), (at, where)
            check(got[~sees], lse[~sees], want[~sees], wl[~sees], tol[~sees], at)


@pytest.mark.parametrize("nq", [1, 7, 20, 150])
def test_attend_nan_codes_of_values_that_are_zero(res, nq):
    """values of a zero scale are zero whatever their codes, wherever the rows' limits are"""
    length = 200
    c, table = paged(res, [length], 16, 1, 64, "e4m3", 3)
    q = torch.randn((nq, 2, 64), device="cuda").bfloat16()
    for col in (0, 5, 10, 12):
        page = int(table[0, col])
        old = c.v_scales[page].clone()
        c.v_scales[page] = 0.0
        want, wl, tol = reference(c, q, table, [length], [0, nq], 1 / 8, True)
        raw = c.v_codes.view(torch.uint8)[page]
        was = raw.clone()
        raw[:, ::3] = 0x7f
        got, lse = c.attend(q, table, ints([length]), query_offsets=ints([0, nq]), return_lse=True)
        raw.copy_(was)
        c.v_scales[page] = old
        check(got, lse, want, wl, tol, col)


# ------------------------------------------------------------------------------------------------ scores and scales far apart
def stepped(res, code, tiles, seed=0, extra=2, sign=False):
    """a context of 64 tokens per entry (score in units of log 2 of a query whose first element is 1, scale of the values)"""
    n, bs, d = 64 * len(tiles), 16, 64
    c, table = paged(res, [n], bs, 1, d, code, seed)
    wide = torch.full((1, table.shape[1] + extra), -1, dtype=I32, device="cuda")
    wide[:, :table.shape[1]] = table
    c.k_codes.zero_()
    c.k_scales.fill_(1.0)
    if sign:  # values that add up
        c.v_codes.copy_(c.v_codes.float().abs().to(c.v_codes.dtype))
    for t, (score, scale) in enumerate(tiles):
        pages = table[0, 4 * t:4 * t + 4].long()
        c.k_codes[pages, 0, :, 0] = torch.tensor(float(score), device="cuda").to(c.k_codes.dtype)
        c.v_scales[pages] = scale
    return c, wide, n


STEPS = {
    # tiles of zero values with large scores, then small scores, then what nearly all of the probability goes to
    "zero first": [(96, 0.0)] * 4 + [(-32, 0.125)] * 4 + [(120, 0.125)] * 4,
    "zero first, small": [(96, 0.0)] * 4 + [(-32, 2.0 ** -125)] * 4 + [(120, 2.0 ** -120)] * 4,
    "zero first, nothing more": [(96, 0.0)] * 4 + [(-120, 0.125)] * 8,
    "zero last": [(-32, 0.125)] * 4 + [(112, 0.0)] * 8,
    # scales that grow by far more than the scores fall
    "small first": [(80, 2.0 ** -85)] * 4 + [(-80, 2.0 ** 90)] * 4,
    "small first, then between": [(64, 2.0 ** -60)] * 4 + [(-64, 2.0 ** 70)] * 4 + [(0, 1.0)] * 4,
    "growing": [(120 - 30 * (i // 4), 2.0 ** (-100 + 50 * (i // 4))) for i in range(16)],
    "large first": [(-80, 2.0 ** 90)] * 4 + [(80, 1.0)] * 4,
    "up and down": [(96, 2.0 ** -40)] * 4 + [(-96, 2.0 ** 40)] * 4 + [(104, 2.0 ** -40)] * 4 + [(-24, 2.0 ** 40)] * 4,
}


@pytest.mark.parametrize("name", list(STEPS))
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_attend_scores_and_scales_far_apart(res, name, code):
    """what a value's scale is has no say in the sum of the probabilities, in whichever order the scales come; both kernels, whole
    and split contexts (a wider table), several requests' worth of rows"""
    for nq in (1, 2, 40, 150):
        for extra in (2, 90):
            c, table, n = stepped(res, code, STEPS[name], extra=extra)
            q = torch.randn((nq, 2, 64), device="cuda").bfloat16()
            q[:, :, 0] = 1.0
            q[:, 1, 0] = 0.75
            got, lse = c.attend(q, table, ints([n]), query_offsets=ints([0, nq]), scale=math.log(2), causal=False, return_lse=True)
            want, wl, tol = reference(c, q, table, [n], [0, nq], math.log(2), False)
            check(got, lse, want, wl, tol, (name, code, nq, extra))


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_attend_large_values(res, code):
    """values near the top of the type's range: what is joined are results, which fit it"""
    for nq in (1, 40):
        for extra, tiles in ((2, 12), (90, 12), (2, 700)):
            c, table, n = stepped(res, code, [(3, 2.0 ** 118)] * tiles, extra=extra, sign=True)
            q = torch.ones((nq, 2, 64), device="cuda").bfloat16()
            got, lse = c.attend(q, table, ints([n]), query_offsets=ints([0, nq]), scale=math.log(2), return_lse=True)
            want, wl, tol = reference(c, q, table, [n], [0, nq], math.log(2), True)
            assert bool(torch.isfinite(got).all())
            check(got, lse, want, wl, tol, (code, nq, extra, tiles))


@pytest.mark.parametrize("extra", [2, 60])
@pytest.mark.parametrize("nq", [1, 40])
def test_attend_nan_codes_of_no_weight(res, nq, extra):
    """tokens whose probability is zero in fp32 are seen all the same"""
    c, table, n = stepped(res, "e4m3", [(120, 0.1)] * 12 + [(-120, 0.1)] * 12, extra=extra)
    c.v_codes.view(torch.uint8)[int(table[0, 20 * 4]), 0, 5, 3] = 0x7f
    q = torch.ones((nq, 2, 64), device="cuda").bfloat16()
    got, lse = c.attend(q, table, ints([n]), query_offsets=ints([0, nq]), scale=math.log(2), causal=False, return_lse=True)
    assert bool(got.isnan().all()) and bool(lse.isnan().all())


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_attend_subnormal_scales(res, code):
    """value scales below fp32's normal numbers, alone and beside larger ones; key scales too (their scores vanish)"""
    for nq in (1, 40):
        for extra in (2, 60):
            for tiles in ([(3, 2.0 ** -130)] * 12, [(60, 2.0 ** -128)] * 4 + [(0, 2.0 ** -60)] * 8, [(3, 2.0 ** -149)] * 4 + [(3, 2.0 ** -127)] * 4):
                c, table, n = stepped(res, code, tiles, extra=extra, sign=True)
                q = torch.ones((nq, 2, 64), device="cuda").bfloat16()
                got, lse = c.attend(q, table, ints([n]), query_offsets=ints([0, nq]), scale=math.log(2), causal=False, return_lse=True)
                want, wl, tol = reference(c, q, table, [n], [0, nq], math.log(2), False)
                check(got, lse, want, wl, tol, (code, nq, extra, tiles[0]))
                c.k_scales[table[0, 1].long()] = 2.0 ** -135
                got, lse = c.attend(q, table, ints([n]), query_offsets=ints([0, nq]), scale=math.log(2), causal=False, return_lse=True)
                want, wl, tol = reference(c, q, table, [n], [0, nq], math.log(2), False)
                check(got, lse, want, wl, tol, (code, nq, extra, tiles[0]))


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("dim, bs", [(64, 16), (128, 32)])
def test_attend_zero_values_with_most_of_the_probability(res, code, dim, bs):
    """tokens whose values have the scale zero take up to all but 2^-40 of the probability; the others' products keep their digits"""
    for nq in (1, 8, 60, 150):
        for length, cols in ((131, 0), (700, 0), (5000, 400)):
            c, table = paged(res, [length], bs, 1, dim, code, 3)
            table = torch.cat([table, torch.full((1, cols), -1, dtype=I32, device="cuda")], 1)
            some = table[0, 1:length // bs:3].long()
            g = torch.Generator(device="cuda")
            g.manual_seed(length + nq)
            q = torch.randn((nq, 2, dim), generator=g, device="cuda").bfloat16()
            for log2 in (4, 12, 20, 30, 40):
                # an element of the queries that the zero-valued blocks' keys meet, and no others
                c.k_codes.view(torch.uint8)[..., 0] = 0
                c.k_codes[some, 0, :, 0] = torch.tensor(8.0, device="cuda").to(c.k_codes.dtype)
                c.k_scales[some] = 2.0 ** -4
                c.v_scales[some] = 0.0
                q[:, :, 0] = log2 * math.log(2) / 0.5 * math.sqrt(dim)
                for causal in (True, False):
                    got, lse = c.attend(q, table, ints([length]), query_offsets=ints([0, nq]), causal=causal, return_lse=True)
                    want, wl, tol = reference(c, q, table, [length], [0, nq], 1 / math.sqrt(dim), causal)
                    check(got, lse, want, wl, tol, (nq, length, log2, causal))


LARGE = {
    "ties": [(5, 0.01), (3, 0.01), (5, 0.01), (-7, 0.01)],
    "ties of other scales": [(5, 2.0 ** -9), (5, 2.0 ** 3), (-7, 2.0 ** 20), (5, 2.0 ** -12)] * 3,
    "growing": [(-100 + 10 * i, 0.01 + 0.002 * i) for i in range(20)],
    "falling": [(100 - 10 * i, 0.01 + 0.002 * i) for i in range(20)],
    "all far below": [(-96, 0.01), (-112, 0.5), (-96, 0.25), (-120, 1.0)] * 2,
    "zero values first": [(-64, 0.0)] * 4 + [(64, 0.5)] * 4 + [(-3, 2.0 ** 30)] * 4,
    "zero values are largest": [(3, 0.5)] * 4 + [(64, 0.0)] * 8,
}


@pytest.mark.parametrize("name", list(LARGE))
@pytest.mark.parametrize("k", [0, 4, 8, 11, 12, 13, 16, 20, 24, 27, 30, 48, 90])
def test_attend_large_scores(res, name, k):
    """Scores far from zero, up to 2^97: their differences count, not their size.  The scores are small integers times 2^k (times ln 2
    log2 e, which rounds them all by the same factor): from k = 8 on equal ones share the probability, all others have none"""
    for nq in (1, 40):
        for extra in (2, 60):
            c, table, n = stepped(res, "int8", LARGE[name], extra=extra)
            q = torch.zeros((nq, 2, 64), device="cuda").bfloat16()
            q[:, 0, 0] = 2.0 ** k
            q[:, 1, 0] = -(2.0 ** k)
            got, lse = c.attend(q, table, ints([n]), query_offsets=ints([0, nq]), scale=math.log(2), causal=False, return_lse=True)
            pages = table[0, :n // 16].long()
            v = (c.v_codes.double() * c.v_scales.double()[:, :, None, None]).transpose(2, 3)[pages, 0].reshape(-1, 64)
            each = c.v_scales.double()[pages, 0].repeat_interleave(16)
            for head, sign in ((0, 1), (1, -1)):
                z = c.k_codes.double()[pages, 0, :, 0].reshape(-1) * 2.0 ** k * sign
                m = z.max()
                p = torch.exp2(z - m)
                # fp16 probabilities (and those that vanish), sums in fp32, the result's rounding; the factor that all scores are
                # rounded by (two roundings, the guard of the reference) where they are not equal
                gap = (m - z)[(z < m) & (z > m - 200)]
                f = 2 ** -11 + (n / 16 + 300) * 2 ** -24 + 2 * (float(gap.max()) if gap.numel() else 0.0) * 2 ** -22
                big, low = p @ v.abs() / p.sum(), 2 ** -31 * (p * each).max() * 127 * n / p.sum()
                want = p @ v / p.sum()
                tol = (f * big + low) * 1.01 + 2 ** -8 * want.abs() + 2 ** -120
                bad = ~((got[:, head].double() - want).abs() <= tol)
                assert not bad.any(), (nq, extra, head, float((got[:, head].double() - want).abs().max()))
                wl = float((m + p.sum().log2()) * math.log(2))
                assert float((lse[:, head].double() - wl).abs().max()) <= 2 ** -11 + abs(wl) * 2 ** -21


@pytest.mark.parametrize("dt, power", [(torch.bfloat16, 8), (torch.bfloat16, 16), (torch.bfloat16, 23), (torch.bfloat16, 30), (torch.bfloat16, 60),
                                       (torch.bfloat16, 100), (torch.float16, 8), (torch.float16, 13)])
@pytest.mark.parametrize("code, lengths, nq", [("e4m3", [90, 700], 1), ("int8", [200, 90], 40), ("e4m3", [9000, 33], 1), ("int8", [20000, 9], 70)])
def test_attend_large_queries(res, code, lengths, nq, dt, power):
    """queries of any numbers times 2^power: a row takes its values from the token with the largest score wherever the next one's is
    further below than the products' and sums' error, (d + 8) 2^-24 sum |q_d k_d|, and 40 units of log 2 tell"""
    c, table = paged(res, lengths, 16, 1, 64, code, 5)
    if code == "int8" and dt == torch.float16:
        c.k_scales.mul_(2.0 ** 10)
    g = torch.Generator(device="cuda")
    g.manual_seed(power)
    q = (torch.randn((2 * nq, 2, 64), generator=g, device="cuda") * 2.0 ** power).to(dt)
    got, lse = c.attend(q, table, ints(lengths), query_offsets=ints([0, nq, 2 * nq]), causal=False, return_lse=True)
    assert bool(torch.isfinite(got).all()) and bool(torch.isfinite(lse).all())
    alone = 0
    for b, n in enumerate(lengths):
        pages = table[b, :-(-n // 16)].long()
        k = (c.k_codes.double() * c.k_scales.double()[:, :, None, None])[pages, 0].reshape(-1, 64)[:n]
        v = (c.v_codes.double() * c.v_scales.double()[:, :, None, None]).transpose(2, 3)[pages, 0].reshape(-1, 64)[:n]
        x = q[b * nq:(b + 1) * nq].double().reshape(-1, 64)
        z = x @ k.T / 8
        error = (x.abs() @ k.abs().T / 8).amax(-1) * 72 * 2 ** -24
        two, at = z.topk(2, -1)
        clear = two[:, 0] - two[:, 1] > 2 * error + 40 * math.log(2)
        alone += int(clear.sum())
        want = v[at[:, 0]][clear]
        out = got[b * nq:(b + 1) * nq].reshape(-1, 64).double()[clear]
        # one probability of one (2^-40 of others), a value, the rounding of its fp16 product and of the result
        assert bool(((out - want).abs() <= (2 ** -11 + 2 ** -20 + torch.finfo(dt).eps / 2) * want.abs() + 2 ** -20).all())
        wl = lse[b * nq:(b + 1) * nq].reshape(-1).double()
        assert bool(((wl - two[:, 0]).abs() <= error + math.log(n) + two[:, 0].abs() * 2 ** -22 + 2 ** -10).all())
    if power >= 16:
        assert alone > nq


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("nq, cols", [(3, None), (3, 200), (3, 2000), (50, None), (50, 200)])
def test_attend_infinite_queries(res, dt, nq, cols):
    """the softmax of scores that are all -inf, or of which one is +inf, is no number; rows that see nothing are zero"""
    length = 2 if cols is None else 1500 if cols == 200 else 30000
    c, table = paged(res, [length], 16, 1, 64, "int8", 1)
    if cols:
        wide = torch.full((1, cols), -1, dtype=I32, device="cuda")
        wide[:, :table.shape[1]] = table
        table = wide
    c.k_codes[..., 0] = 5
    c.k_codes[int(table[0, 0]), 0, 1, 1] = -3
    c.k_codes[int(table[0, 0]), 0, 0, 1] = 3
    for value, at in ((-math.inf, 0), (math.inf, 0), (-math.inf, 1)):
        q = torch.randn((nq, 2, 64), device="cuda").to(dt)
        clean = q.clone()
        q[:, 1, at] = value
        got, lse = c.attend(q, table, ints([length]), query_offsets=ints([0, nq]), return_lse=True)
        want, wl, tol = reference(c, clean, table, [length], [0, nq], 1 / 8, True)
        sees = torch.arange(nq) + length - nq + 1 > 0
        assert bool(got[sees][:, 1].isnan().all()) and bool(lse[sees][:, 1].isnan().all())
        assert bool((got[~sees] == 0).all()) and bool((lse[~sees] == -math.inf).all())
        check(got[:, 0], lse[:, 0], want[:, 0], wl[:, 0], tol[:, 0])


# ------------------------------------------------------------------------------------------------ lengths and batches
@pytest.mark.parametrize("code, bs, hq, length, nq, cols", [
    ("e4m3", 16, 2, 1000, 10, 62), ("int8", 16, 2, 1000, 300, 53), ("e4m3", 16, 1, 1000, 300, 52), ("int8", 64, 2, 5000, 200, 77),
    ("e4m3", 64, 4, 5000, 6, 78), ("int8", 128, 1, 700, 700, 3), ("e4m3", 16, 2, 100, 90, 0), ("e4m3", 256, 2, 300, 20, 1)])
def test_attend_lengths_past_the_table(res, code, bs, hq, length, nq, cols):
    """rows that see tokens behind the table's last column are NaN; those that do not are what they are with a wider table"""
    c, table = paged(res, [length, 50], bs, 1, 64, code, 3)
    q = torch.randn((nq + 3, hq, 64), device="cuda").half()
    offs = [0, nq, nq + 3]
    want, wl, tol = reference(c, q, table, [length, 50], offs, 1 / 8, True)
    narrow = table[:, :cols].contiguous()
    got, lse = c.attend(q, narrow, ints([length, 50]), query_offsets=ints(offs), return_lse=True)
    fine = torch.cat([length - nq + 1 + torch.arange(nq), 50 - 3 + 1 + torch.arange(3)]) <= cols * bs
    check(got[fine], lse[fine], want[fine], wl[fine], tol[fine])
    assert bool(got[~fine].isnan().all()) and bool(lse[~fine].isnan().all())
    got = c.attend(q, narrow, ints([length, 50]), query_offsets=ints(offs), causal=False)
    assert bool(got[:nq].isnan().all())
    # the largest length there is, and the rows that mask all of what is not there
    most = 2 ** 31 - 1
    got, lse = c.attend(q, narrow, ints([most, 50]), query_offsets=ints(offs), return_lse=True)
    assert bool(got[:nq].isnan().all()) and bool(lse[:nq].isnan().all())


@pytest.mark.parametrize("queries", [None, 2, 40])
@pytest.mark.parametrize("split", [False, True])
def test_attend_many_requests(res, queries, split):
    """more requests than a wavefront has lanes, three groups of 64 and a rest; short ones, and contexts that are split"""
    n = 130 if queries != 40 else 67
    g = torch.Generator()
    g.manual_seed(n)
    lens = torch.randint(0, 150, (n,), generator=g).tolist()
    if split:
        for i in (0, 5, 63, 64, 66, n - 1):
            lens[i] = 2000 + 900 * (i % 4)
    nq = None if queries is None else torch.randint(0, queries + 1, (n,), generator=g).tolist()
    offs = None if nq is None else [0] + torch.tensor(nq).cumsum(0).tolist()
    c, table = paged(res, lens, 16, 2, 64, "e4m3", 7)
    q = torch.randn((n if nq is None else offs[-1], 4, 64), device="cuda").bfloat16()
    got, lse = c.attend(q, table, ints(lens), query_offsets=None if offs is None else ints(offs), return_lse=True)
    want, wl, tol = reference(c, q, table, lens, offs, 1 / 8, True)
    check(got, lse, want, wl, tol)


@pytest.mark.parametrize("length, most", [(300, None), (40000, None), (40000, 1)])
def test_attend_offsets_that_decrease(res, length, most):
    """requests that claim each other's rows, many times the work and the partial results that the call has room for: what lies
    around the call's own memory is left alone, and rows of no request too"""
    n, t = 70, 64
    c, table = paged(res, [length], 16, 1, 64, "int8", 3)
    table = table.repeat(n, 1)
    q = torch.randn((t + 2, 2, 64), device="cuda").half()
    out = torch.full((t + 4, 2, 64), 3.0, device="cuda").half()
    offs = [0, t] * (n // 2) + [0]
    c.attend(q[:t], table, ints([length] * n), query_offsets=ints(offs), max_queries=most, out=out[2:t + 2])
    torch.cuda.synchronize()
    assert bool((out[:2] == 3).all()) and bool((out[t + 2:] == 3).all())
    want, _, tol = reference(c, q[:1], table[:1], [length], [0, 1], 1 / 8, True)
    check(c.attend(q[:1], table[:1], ints([length])), None, want, None, tol)


# ------------------------------------------------------------------------------------------------ long rows, other layouts
def test_reorder_long_rows(res):
    """rows, and states together, of more than 65535 pieces of 16384 bytes (a launch's), between short ones; more than 64 states"""
    edge = 65535 * 16384
    p = ints([[1, 0]])
    for sizes in ([edge + 16384 + 7], [100, edge // 2, 5, edge // 2 + 3, 40000], [3] * 63 + [edge - 200, 16385, 9]):
        states = [torch.randint(0, 255, (1, 2, (n + 7) // 8), device="cuda").view(torch.uint8)[:, :, :n] if n > 1000 else
                  torch.randint(0, 255, (1, 2, n), device="cuda", dtype=torch.uint8) for n in sizes]
        got = decoding.reorder_beams(res, states, p)
        for x, y in zip(got, states):
            assert torch.equal(x[0, 0], y[0, 1]) and torch.equal(x[0, 1], y[0, 0]), y.shape
        del states, got


# ------------------------------------------------------------------------------------------------ blocks that come back
@pytest.mark.parametrize("n, w, bs, prompt, steps", [(2, 3, 16, 21, 30), (3, 4, 32, 64, 40), (1, 2, 16, 0, 20)])
def test_fork_and_plan_keep_every_block_once(res, n, w, bs, prompt, steps):
    """three rounds of requests over the same rows, without giving anything by hand: plan, add, fork, whole blocks taken back,
    release.  Every block is in one of the owned table, the spare ones and the free ones at all times, and each beam's context
    is what its history says"""
    import random
    rng = random.Random(n * w)
    h, d, cols = 1, 64, 6
    rows = n * w
    emb = torch.randn((50, 2, h, d), device="cuda").bfloat16()
    total = rows * (cols + 1)
    c = decoding.PagedCache(res, total, bs, h, d, "e4m3")
    pages = torch.randperm(total, generator=torch.Generator().manual_seed(n)).to(I32).cuda()
    spare, ring = pages[:rows].clone(), torch.cat([pages[rows:], torch.full((rows,), -1, dtype=I32, device="cuda")])
    state = torch.tensor([0, total - rows], dtype=torch.int64, device="cuda")
    view = torch.full((rows, cols), -1, dtype=I32, device="cuda")
    owned, lengths = view.clone(), torch.zeros(rows, dtype=I32, device="cuda")

    def plan(want, room):
        p = decoding.plan_blocks(res, view, lengths, ints(want), ring, state, bs, room, owned_table=owned, free_state_out=state)
        assert p.granted.tolist() == [1] * rows
        return p

    def once():
        free = [int(ring[(int(state[0]) + i) % total]) for i in range(int(state[1]))]
        held = [x for r in range(rows) for x in owned[r, :-(-int(lengths[r]) // bs)].tolist()]
        assert sorted(free + held + spare.tolist()) == list(range(total))
        # no two beams write to the same block, and none into a spare or free one
        tails = [int(view[r, int(lengths[r]) // bs]) for r in range(rows) if int(lengths[r]) % bs]
        assert len(set(tails)) == len(tails) and not set(tails) & set(spare.tolist() + free)

    for trial in range(3):
        history = [[rng.randrange(50) for _ in range(prompt + trial)] for _ in range(n) for _ in range(w)]
        history = [list(history[(r // w) * w]) for r in range(rows)]
        new = [list(x) for x in history]
        for step in range(steps):
            p = plan([len(x) for x in history], sum(map(len, new)) + 1)
            lengths = p.lengths
            tok = torch.tensor([t for x in new for t in x] + [0], device="cuda")
            c.add(emb[tok, 0], emb[tok, 1], p.slots)
            once()
            for r in range(rows):
                m = len(history[r])
                if m == 0:
                    continue
                for got, i in zip(c.reconstruct(view[r, :-(-m // bs)]), (0, 1)):
                    e = emb[torch.tensor(history[r], device="cuda"), i].float()
                    got = got.transpose(1, 2).reshape(-1, h, d)[:m]
                    # a code is off by half a step, 2^-4 of the value; a block's scale that grows may round it again: twice that
                    assert bool(((got - e).abs() <= 2 ** -3 * e.abs() + 0.02).all()), (trial, step, r)
            parents = [[rng.randrange(w) for _ in range(w)] for _ in range(n)]
            view, lengths, spare = decoding.fork_blocks(res, [c], view, lengths, spare, ints(parents), owned_table=owned)
            once()
            history = [list(history[(r // w) * w + parents[r // w][r % w]]) for r in range(rows)]
            if step == steps // 2:  # back by whole blocks, all beams together
                keep = [len(x) // bs * bs - bs if len(x) >= bs else 0 for x in history]
                lengths = plan(keep, 1).lengths
                history = [x[:k] for x, k in zip(history, keep)]
                once()
            new = [[rng.randrange(50)] for _ in range(rows)]
            history = [x + y for x, y in zip(history, new)]
        lengths = plan([0] * rows, 1).lengths
        assert int(state[1]) == total - rows
        once()


def test_fork_blocks_owned_table_on_its_own(res):
    """the owned table and the spare blocks: changed where a block is copied, left where there is nothing to copy or no block for it"""
    bs, w = 16, 3
    c = filled(res, 40, 1, bs, 64, "int8", 1)
    table = ints([[i, 10 + i, -1] for i in range(2 * w)])
    owned = torch.full((2 * w, 5), -7, dtype=I32, device="cuda")[:, :3]  # rows of a wider table
    owned.copy_(ints([[i, 20 + i, -1] for i in range(2 * w)]))
    lengths, spare = ints([20] * w + [32] * w), ints([30, -1, 40, 33, 34, 35])
    parents = ints([[2, 0, 1], [1, 1, 5]])
    t, l, s = decoding.fork_blocks(res, [c], table, lengths, spare, parents, owned_table=owned)
    assert t.tolist() == [[2, 30, -1], [0, -1, -1], [1, -1, -1], [4, 14, -1], [4, 14, -1], [5, 15, -1]]
    assert owned.tolist() == [[0, 30, -1], [1, 21, -1], [2, 22, -1], [3, 23, -1], [4, 24, -1], [5, 25, -1]]
    assert s.tolist() == [20, -1, 40, 33, 34, 35] and l.tolist() == lengths.tolist()
    assert owned._base[:, 3:].eq(-7).all()
    with pytest.raises(ValueError):
        decoding.fork_blocks(res, [c], table, lengths, spare, parents, owned_table=owned[:, :2])
    with pytest.raises(TypeError):
        decoding.fork_blocks(res, [c], table, lengths, spare, parents, owned_table=owned.long())


@pytest.mark.parametrize("n, total, cols", [(1, 1, 1 << 20), (3, 7, 300000), (1500, 5, 4000)])
def test_plan_blocks_given_back_more_than_there_are(res, n, total, cols):
    """lengths that claim many times the ring's blocks: what is returned goes round, the count stays within the ring, and what
    lies around it is left alone"""
    table = torch.arange(cols, dtype=I32, device="cuda").repeat(n, 1)
    ring = torch.full((total + 2,), -9, dtype=I32, device="cuda")
    state = torch.tensor([total - 1, total], dtype=torch.int64, device="cuda")
    p = decoding.plan_blocks(res, table, ints([cols] * n), ints([0] * n), ring[1:-1], state, 1, 3)
    assert p.free_state.tolist() == [total - 1, total] and p.lengths.tolist() == [0] * n and p.granted.tolist() == [1] * n
    assert ring[0] == -9 and ring[-1] == -9 and bool(((ring[1:-1] >= 0) & (ring[1:-1] < cols)).all())


@pytest.mark.parametrize("n", [1023, 1024, 1025])
@pytest.mark.parametrize("tokens", [1, 40])
def test_plan_blocks_around_a_thread_per_request(res, n, tokens):
    """where the plan goes from one workgroup to the general kernels, with few and many slots"""
    import random
    from test_gpu_decoding import plan_both
    rng = random.Random(n + tokens)
    cols, bs = 5, 16
    total = 3 * n
    ring = list(range(total))
    rng.shuffle(ring)
    table = [[-1] * cols for _ in range(n)]
    lens, state = [0] * n, [total - 5, total]
    for step in range(3):
        new = [rng.choice([x + tokens if x + tokens <= cols * bs else 0, max(x - 20, 0), x]) for x in lens]
        lens, state = plan_both(res, table, None, lens, new, ring, state, bs, n * tokens)


# ------------------------------------------------------------------------------------------------ adding
@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("scale", [1e-40, 2.0 ** -149, 2.0 ** -126, 3e-20, 2.0 ** 127, 3e38])
def test_add_over_any_scale(res, code, scale):
    """zeros, then numbers, added behind tokens whose scale is subnormal, no power of two or the largest there is"""
    for bs, d in ((16, 64), (64, 128)):
        c = filled(res, 3, 2, bs, d, code, 1)
        if scale > 1e30:  # (the old values stay within fp32)
            c.k_codes.zero_()
            c.v_codes.zero_()
        c.k_scales.fill_(scale)
        c.v_scales.fill_(scale)
        old = [c.k_codes.double().clone(), c.v_codes.double().clone()]
        x = torch.zeros((2, 2, d), device="cuda").bfloat16()
        c.add(x, x, ints([bs + 3, bs + 9]))
        k, v = c.k_codes.double(), c.v_codes.double()
        assert bool((k[1, :, [3, 9]] == 0).all()) and bool((v[1, :, :, [3, 9]] == 0).all())
        assert bool((c.k_scales == scale).all()) and bool((c.v_scales == scale).all())
        old[0][1, :, [3, 9]], old[1][1, :, :, [3, 9]] = 0.0, 0.0
        assert torch.equal(k, old[0]) and torch.equal(v, old[1])
        # numbers: the scale is the larger of the old one and their power of two; a code is off by half a step of it
        x = torch.randn((2, 2, d), device="cuda").bfloat16()
        c.add(x, x, ints([bs + 4, 2 * bs + 1]))
        got, _ = c.reconstruct(ints([1, 2]))
        e = torch.stack([got[0, :, 4], got[1, :, 1]]).double() - x.double()
        s = torch.stack([c.k_scales[1], c.k_scales[2]]).double()[:, :, None]
        # (1 / scale and the product are rounded first: 2^-23 of the code)
        room = (s * 2 ** -10 + x.double().abs() * 2 ** -4 if code == "e4m3" else s * 0.5) + x.double().abs() * 2 ** -22
        assert bool((e.abs() <= room).all())


# ------------------------------------------------------------------------------------------------ refusals
def test_gradients_are_not_dropped_on_the_device(res):
    c = filled(res, 4, 2, 16, 64, "e4m3", 0)
    x = torch.randn((1, 2, 64), device="cuda").half()
    g = x.clone().requires_grad_()
    table, n, parents = ints([[0, 1]]), ints([3]), ints([[1, 0]])
    logits, scores = torch.randn((1, 2, 5), device="cuda"), torch.zeros((1, 2), device="cuda")
    state = torch.randn((1, 2, 7), device="cuda")
    calls = [lambda f: c.attend(f(x), table, n), lambda f: c.attend(x, table, n, out=f(x.clone())), lambda f: c.add(f(x), x, n),
             lambda f: c.add(x, f(x), n), lambda f: decoding.beam_select(res, f(logits), scores, 2),
             lambda f: decoding.beam_select(res, logits, f(scores), 2), lambda f: decoding.reorder_beams(res, [state, f(state)], parents)]
    for call in calls:
        with pytest.raises(ValueError, match="gradient"):
            call(lambda t: t.clone().requires_grad_())
        want = call(lambda t: t)
        with torch.no_grad():
            got = call(lambda t: t.clone().requires_grad_())
        for a, b in zip(got if isinstance(got, (list, tuple)) else [got], want if isinstance(want, (list, tuple)) else [want]):
            assert a is None or torch.equal(a, b)
    assert g.grad is None


def test_reorder_complex_states(res):
    """complex rows are reordered as bytes; a lazy conjugate, whose memory holds other numbers, is refused"""
    z = torch.randn((2, 3, 5), dtype=torch.complex64, device="cuda")
    p = ints([[2, 0, 1], [1, 1, 2]])
    for t in (z, z.conj().resolve_conj(), z.conj().imag.resolve_neg()):
        assert torch.equal(decoding.reorder_beams(res, [t], p)[0], t[torch.arange(2, device="cuda")[:, None], p.long()])
    for t in (z.conj(), z.conj().imag):
        with pytest.raises(ValueError, match="lazily"):
            decoding.reorder_beams(res, [t], p)


def test_attend_out_that_overlaps_is_refused(res):
    c, table = paged(res, [20, 20, 20], 16, 1, 64, "e4m3", 0)
    q, lens = torch.randn((3, 4, 64), device="cuda").half(), ints([20, 20, 20])
    base = torch.zeros(4096, device="cuda").half()
    want = c.attend(q, table, lens)
    for stride in ((0, 64, 1), (256, 0, 1), (256, 63, 1), (255, 64, 1), (64, 64, 1), (63, 192, 1), (64, 191, 1)):
        with pytest.raises(ValueError, match="overlap"):
            c.attend(q, table, lens, out=base.as_strided((3, 4, 64), stride))
    for stride in ((256, 64, 1), (300, 67, 1), (64, 192, 1), (70, 400, 1)):
        out = base.as_strided((3, 4, 64), stride)
        assert c.attend(q, table, lens, out=out) is out and torch.equal(out, want)
    # one row or one head: the other stride does not matter
    for shape, stride in (((1, 4, 64), (0, 64, 1)), ((3, 1, 64), (64, 0, 1)), ((1, 1, 64), (0, 0, 1))):
        out = base.as_strided(shape, stride)
        x = q[:shape[0], :shape[1]]
        assert torch.equal(c.attend(x, table[:shape[0]], lens[:shape[0]], out=out), want[:shape[0], :shape[1]])
    with pytest.raises(ValueError, match="overlap"):
        c.attend(q[:, :1], table, lens, out=base.as_strided((3, 1, 64), (32, 0, 1)))
    with pytest.raises(ValueError, match="overlap"):
        c.attend(q[:1], table[:1], lens[:1], out=base.as_strided((1, 4, 64), (0, 32, 1)))


def test_wrong_kinds_are_type_errors(res):
    """what is no tensor, or no cache, is a TypeError like a wrong dtype"""
    logits, scores = torch.zeros((1, 2, 5), device="cuda"), torch.zeros((1, 2), device="cuda")
    for bad in ([[True, False]], scores, 1):
        with pytest.raises(TypeError):
            decoding.beam_select(res, logits, scores, 2, finished=bad)
    c = filled(res, 4, 1, 16, 64, "int8", 0)
    args = (ints([[0], [1]]), ints([3, 3]), ints([2, 3]), ints([[0, 1]]))
    for bad in ([c, None], [c.k_codes], 3):
        with pytest.raises(TypeError):
            decoding.fork_blocks(res, bad, *args)
    with pytest.raises(ValueError):
        decoding.fork_blocks(res, [], *args)
    decoding.fork_blocks(res, (x for x in [c]), *args)  # any iterable


# ------------------------------------------------------------------------------------------------ beams
def _log_sums_less(rows):
    """rows [n, v]: fp32 scores that take nearly all of each row's best value away, so that the fp32 results keep the digits of
    the log-sum's error; the exact values that they leave"""
    top = rows.double().amax(-1)
    lse = torch.logsumexp(rows.double(), -1)
    s = (lse - top).float()
    return s, s.double() + top - lse


@pytest.mark.parametrize("far", [-0.5, -3.0, -7.7, -10.0, -11.3, -12.9, -14.2, -16.0])
@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
def test_beam_select_one_token_dominates(res, far, dt):
    """One token at 0, the others at `far`, 1000 of them: 16 of a lane at most, one step.  Lanes without the token have exact terms
    (2^0).  In its lane a term is off by |far| (2^-23 + 2^-26) and 2^-23; four terms are added in fp32, two roundings of 2^-24 of
    at most 1 + 3 e^far; sums beyond that are in 64 bits."""
    for pos in (0, 5, 500, 999):
        x = torch.full((1, 1, 1000), far, device="cuda").to(dt)
        x[0, 0, pos] = 0
        e = math.exp(float(x[0, 0, pos - 1]))
        s, want = _log_sums_less(x[0])
        got, _, tok = decoding.beam_select(res, x, s[None], 1)
        tol = (2 ** -23 * (1 + 3 * e) + 15 * e * (abs(far) * (2 ** -23 + 2 ** -26) + 2 ** -23)) / (1 + 999 * e) + 2 ** -45
        assert int(tok) == pos and abs(float(got.double() - want)) <= tol, (pos, float(got.double() - want), tol)


@pytest.mark.parametrize("v", [1000, 32000, 128001])
@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
def test_beam_select_log_sums(res, v, dt):
    """Rows of all kinds.  A term is off by |x - max| (2^-23 + 2^-26) (its own exponential's argument and those that rescale the
    sums it is in: their differences add up) and by 2^-23 for each of them, at most one a step: 2^-23 (3 + steps) with the sums of four"""
    g = torch.Generator(device="cuda")
    g.manual_seed(v)
    n = torch.randn((12, v), generator=g, device="cuda")
    up = torch.linspace(-20, 0, v, device="cuda")
    rows = torch.stack([n[0], n[1] * 3, n[2] * 10, n[3] * 0.1, n[4].exp(), -(n[5].abs()) * 4, up, up.flip(0), up * 3, n[6] * 3 + 100,
                        n[7] * 30 - 1000, torch.zeros_like(up)]).to(dt)
    for row in rows:
        s, want = _log_sums_less(row[None])
        got, _, _ = decoding.beam_select(res, row[None, None], s[None], 1)
        d = row.double() - row.double().max()
        p = d.exp()
        steps = min(v // 1024 + 1, 8 + v // 4096)
        tol = float((p * -d).sum() / p.sum()) * (2 ** -23 + 2 ** -26) + 2 ** -23 * (3 + steps) + 2 ** -45
        assert abs(float(got.double() - want)) <= tol


def test_beam_select_beams_that_are_close(res):
    """beams whose values differ by less than an fp32 sum of 16 tells, in both orders"""
    x = torch.full((1, 2, 1000), -math.inf, device="cuda")
    x[0, 0, :2] = 0.0                  # log-sum log 2
    for far, pos in ((-10.0, 700), (-11.3, 5), (-11.3, 700), (-12.9, 999), (-7.7, 0)):
        x[0, 1] = far
        x[0, 1, pos] = 0.0
        lse = torch.logsumexp(x[0].double(), -1)
        for gap in (-3e-7, 3e-7):
            s = (lse + torch.tensor([0.0, gap], device="cuda").double()).float()
            exact = s.double() - lse
            assert 2.4e-7 < abs(float(exact[0] - exact[1])) < 3.6e-7
            _, parents, _ = decoding.beam_select(res, x, s[None], 1)
            assert int(parents) == int(exact.argmax()), (far, pos, gap)


def test_numbers_past_32_bits_are_refused(res):
    """they would reach the library without their upper halves"""
    logits, scores = torch.randn((1, 2, 50), device="cuda"), torch.zeros((1, 2), device="cuda")
    done = torch.tensor([[True, False]], device="cuda")
    for kw in (dict(pad_token=2 ** 32 + 3), dict(pad_token=50), dict(pad_token=-1), dict(num_beams=2 ** 32 + 2), dict(num_beams=65), dict(num_beams=0)):
        with pytest.raises(ValueError):
            decoding.beam_select(res, **{**dict(logits=logits, scores=scores, num_beams=2, finished=done), **kw})
    table, n, ring, state = ints([[-1] * 4]), ints([0]), ints([0, 1, 2]), torch.tensor([0, 3], device="cuda")
    for bs, room in ((2 ** 32 + 16, 4), (0, 4), (-16, 4), (16, -1), (16, 2 ** 32 + 4)):
        with pytest.raises(ValueError):
            decoding.plan_blocks(res, table, n, ints([3]), ring, state, bs, room)
    # a bound on the queries may be any number
    c, table = paged(res, [40], 16, 1, 64, "e4m3", 0)
    q = torch.randn((40, 2, 64), device="cuda").half()
    want = c.attend(q, table, ints([40]), query_offsets=ints([0, 40]))
    for most in (2 ** 32 + 1, 2 ** 40, 41):
        assert torch.equal(c.attend(q, table, ints([40]), query_offsets=ints([0, 40]), max_queries=most), want)
