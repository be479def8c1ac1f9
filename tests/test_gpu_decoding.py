"""GPU tests of the decoding operators (faiss_amd/decoding.py) against plain implementations in 64 bits.

Tolerances of the attention, per output element.  With A = sum_j p_j |v_j| / sum_j p_j:
  * probabilities (times their value's scale) are rounded to fp16: at most 2^-11 of each, together 2^-11 A, and where they are
    below fp16's normal numbers by 2^-25 in units in which the row's largest is at least 2^6: 2^-31 max_j p_j s_j per code;
  * a score's fp32 sum over D products and its scaling are off by at most (D + 8) 2^-24 B, B = scale max_j sum_d |q_d k_jd| (and
    2 steps for the exponential), which changes numerator and denominator by that factor: 2 ((D + 8) B + 4) 2^-24 A;
  * sums over N tokens in fp32: lanes add 16 at a time, matrix steps 32, chunks are joined: less than (N / 16 + 300) 2^-24 A;
  * the result is rounded to its type: half a step, eps / 2 |o| (and the smallest subnormal).
bf16 queries lose nothing but what is 2^-35 below a row's largest element."""
import math

import pytest
import torch

import faiss_amd
from faiss_amd import decoding

pytestmark = pytest.mark.gpu
QMAX = {"e4m3": 448.0, "int8": 127.0}
I32 = torch.int32


def ints(x, dev="cuda"):
    return torch.tensor(x, dtype=I32, device=dev)


def values(cache, page, head):
    """keys, values [block_size, head_dim] of a block in 64 bits"""
    k = cache.k_codes[page, head].double() * cache.k_scales[page, head].double()
    v = cache.v_codes[page, head].double() * cache.v_scales[page, head].double()
    return k, v.T


def filled(res, n, h, bs, d, code, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    c = decoding.PagedCache(res, n, bs, h, d, code)
    for t in (c.k_codes, c.v_codes):
        x = torch.randn(t.shape, generator=g, device="cuda")
        t.copy_((x * 60).clamp(-448, 448).to(t.dtype) if code == "e4m3" else (x * 30).round().clamp(-127, 127).to(t.dtype))
    for t in (c.k_scales, c.v_scales):  # any positive scales, not only the powers of two that add() makes
        t.copy_(torch.rand(t.shape, generator=g, device="cuda") * 0.02 + 0.002)
    return c


def reference(cache, q, table, lens, offs, scale, causal):
    """out, lse, tolerance (all float64) of every row; rows of no request stay NaN"""
    t, hq, d = q.shape
    bs, hk = cache.block_size, cache.num_heads
    out = torch.full((t, hq, d), float("nan"), dtype=torch.float64, device=q.device)
    lse = torch.full((t, hq), float("nan"), dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    kk = cache.k_codes.double() * cache.k_scales.double()[:, :, None, None]
    vv = (cache.v_codes.double() * cache.v_scales.double()[:, :, None, None]).transpose(2, 3)
    vc, vs = cache.v_codes.double().abs().transpose(2, 3), cache.v_scales.double()
    for b, n in enumerate(lens):
        a, e = (offs[b], offs[b + 1]) if offs is not None else (b, b + 1)
        nq = e - a
        pages = table[b, :(n + bs - 1) // bs].long()
        for h in range(hk):
            k = kk[pages, h].reshape(-1, d)[:n]
            v = vv[pages, h].reshape(-1, d)[:n]
            codes, each = vc[pages, h].reshape(-1, d)[:n], vs[pages, h].repeat_interleave(bs)[:n]
            g = hq // hk
            x = q[a:e, h * g:(h + 1) * g].double().reshape(nq * g, d)
            z = x @ k.T * scale
            size = (x.abs() @ k.abs().T * scale).amax(-1, keepdim=True) if n else torch.zeros((nq * g, 1), dtype=torch.float64, device=q.device)
            see = torch.full((nq * g, 1), n, device=q.device)
            if causal:
                see = (n - nq + 1 + torch.arange(nq, device=q.device)).repeat_interleave(g)[:, None]
            z = z.masked_fill(torch.arange(n, device=q.device)[None] >= see, -math.inf)
            empty = see <= 0
            if n == 0:
                o, l, big, low = x * 0, x[:, 0] * 0 - math.inf, x * 0, x * 0
            else:
                m = z.amax(-1, keepdim=True)
                p = torch.where(empty, torch.zeros_like(z), (z - m).exp())
                s = p.sum(-1, keepdim=True)
                o = torch.where(empty, torch.zeros_like(x), p @ v / s)
                big = torch.where(empty, torch.zeros_like(x), p @ v.abs() / s)
                low = torch.where(empty, torch.zeros_like(x), 2 ** -31 * (p * each).amax(-1, keepdim=True) * codes.sum(0) / s)
                l = torch.where(empty[:, 0], torch.full_like(s[:, 0], -math.inf), m[:, 0] + s[:, 0].log())
            eps = torch.finfo(q.dtype).eps / 2
            f = 2 ** -11 + 2 * ((d + 8) * size + 4) * 2 ** -24 + (n / 16 + 300) * 2 ** -24
            out[a:e, h * g:(h + 1) * g] = o.reshape(nq, g, d)
            lse[a:e, h * g:(h + 1) * g] = l.reshape(nq, g)
            tol[a:e, h * g:(h + 1) * g] = ((f * big + low) * (1 + eps) + eps * o.abs() + torch.finfo(q.dtype).smallest_normal * eps).reshape(nq, g, d)
    return out, lse, tol


def paged(res, lens, bs, hk, d, code, seed, extra=3):
    """a cache and a table that scatters the requests' blocks"""
    need = [(n + bs - 1) // bs for n in lens]
    total = sum(need) + extra
    c = filled(res, total, hk, bs, d, code, seed)
    g = torch.Generator()
    g.manual_seed(seed)
    perm = torch.randperm(total, generator=g).to(I32)
    table = torch.full((len(lens), max(need + [1]) + 2), -1, dtype=I32)
    at = 0
    for i, m in enumerate(need):
        table[i, :m] = perm[at:at + m]
        at += m
    return c, table.cuda()


def check(got, lse, want, wl, tol, name=""):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (name, int(bad.sum()), float((got.double() - want).abs().max()), bad.nonzero()[:4].tolist())
    if lse is not None:
        fin = torch.isfinite(wl)
        assert torch.equal(torch.isfinite(lse), fin)
        # a log-sum is off by the scores' error and the sums' (relative) error; both are below 2^-11 here
        assert float((lse.double() - wl)[fin].abs().max() if fin.any() else 0.0) < 2 ** -11, name


CASES = [
    # code, type, dim, block, heads, kv heads, lengths, queries (None: one each), causal
    ("e4m3", torch.bfloat16, 128, 16, 8, 2, [1], None, True),
    ("e4m3", torch.bfloat16, 128, 16, 32, 8, [0, 1, 15, 16, 17, 63, 64, 65, 255, 257, 1000], None, True),
    ("int8", torch.float16, 64, 32, 4, 4, [31, 0, 33, 300, 2], None, True),
    ("int8", torch.bfloat16, 96, 64, 6, 2, [500, 63, 64, 65, 4097], None, True),
    ("e4m3", torch.float16, 192, 128, 16, 1, [1, 129, 2000], None, True),
    ("e4m3", torch.bfloat16, 256, 256, 20, 1, [255, 256, 257, 5000], None, True),     # 20 heads of one: two row tiles
    ("int8", torch.bfloat16, 128, 16, 71, 1, [77, 1500], None, True),                 # more heads than a row tile of 32
    ("e4m3", torch.bfloat16, 128, 16, 8, 2, [5, 100, 640], [5, 3, 4], True),          # drafts; a whole prompt
    ("int8", torch.float16, 128, 64, 8, 2, [70, 3, 900], [6, 6, 7], True),            # three rows of the second see nothing
    ("e4m3", torch.float16, 64, 16, 4, 2, [200, 40], [100, 40], False),
    ("e4m3", torch.bfloat16, 128, 64, 8, 2, [700, 0, 1, 333], [257, 0, 1, 333], True),
    ("int8", torch.bfloat16, 256, 32, 4, 2, [600, 130], [70, 130], True),
    ("int8", torch.float16, 96, 128, 3, 3, [1031, 200], [200, 130], True),
    ("e4m3", torch.bfloat16, 192, 16, 2, 1, [333], [333], True),
    ("e4m3", torch.float16, 128, 16, 4, 1, [40], [60], True),                         # more queries than tokens
    ("e4m3", torch.bfloat16, 128, 64, 8, 8, [9000, 20000, 33], None, True),           # split contexts
    ("int8", torch.bfloat16, 64, 16, 8, 1, [30001], [129], True),                     # split contexts, many rows
]


@pytest.mark.parametrize("i", range(len(CASES)))
def test_attend(res, i):
    code, dt, d, bs, hq, hk, lens, nq, causal = CASES[i]
    c, table = paged(res, lens, bs, hk, d, code, i)
    offs = None
    if nq is not None:
        offs = [0]
        for x in nq:
            offs.append(offs[-1] + x)
    t = offs[-1] if offs else len(lens)
    g = torch.Generator(device="cuda")
    g.manual_seed(100 + i)
    q = (torch.randn((t, hq, d), generator=g, device="cuda") * 1.5).to(dt)
    scale = 1 / math.sqrt(d)
    got, lse = c.attend(q, table, ints(lens), query_offsets=None if offs is None else ints(offs), causal=causal, return_lse=True)
    want, wl, tol = reference(c, q, table, lens, offs, scale, causal)
    check(got, lse, want, wl, tol, CASES[i])
    again = c.attend(q, table, ints(lens), query_offsets=None if offs is None else ints(offs), causal=causal)
    assert torch.equal(got, again)  # no order depends on chance
    if nq is not None:  # a bound that is tight, and one that is too low, cost time at most
        for most in (max(nq), 1):
            other = c.attend(q, table, ints(lens), query_offsets=ints(offs), causal=causal, max_queries=most)
            check(other, None, want, None, tol, (CASES[i], most))


def test_attend_strides_padding_and_scale(res):
    """views of a fused projection, a wider table, out of another layout; rows behind the last request stay as they were"""
    lens, nq = [300, 90, 17], [40, 1, 17]
    c, table = paged(res, lens, 16, 2, 64, "e4m3", 5)
    wide = torch.full((3, table.shape[1] + 7), -1, dtype=I32, device="cuda")
    wide[:, :table.shape[1]] = table
    qkv = torch.randn((70, 3, 8, 64), device="cuda").bfloat16()
    q = qkv[:, 1]
    odd = torch.randn((70, 8, 67), device="cuda").bfloat16()[:, :, 1:65]  # rows on odd addresses
    offs = [0, 40, 41, 58]
    near = torch.full((70, 8, 67), 7.0, device="cuda").bfloat16()
    c.attend(q, table, ints(lens), query_offsets=ints(offs), out=near[:, :, 1:65])  # out on odd addresses
    want, _, tol = reference(c, q[:58], table, lens, offs, 1 / 8, True)
    check(near[:58, :, 1:65], None, want, None, tol)
    assert bool((near[58:] == 7).all()) and bool((near[:, :, 0] == 7).all()) and bool((near[:, :, 65:] == 7).all())
    for x, sc in ((q, 0.3), (odd, 0.0), (q.transpose(0, 1).contiguous().transpose(0, 1), -0.125)):
        out = torch.full((8, 70, 64), 7.0, device="cuda").bfloat16().transpose(0, 1)
        got = c.attend(x, wide[:, :table.shape[1]], ints(lens), query_offsets=ints(offs), scale=sc, out=out)
        assert got is out and bool((out[58:] == 7).all())
        want, wl, tol = reference(c, x[:58], table, lens, offs, sc, True)
        # (the tolerance's score term takes |scale|)
        check(out[:58], None, want, None, tol.abs() if sc >= 0 else reference(c, -x[:58], table, lens, offs, -sc, True)[2], sc)


def test_attend_sees_nothing_behind_the_last_token(res):
    """codes and scales behind a request's tokens may be anything; so may blocks of nobody"""
    lens = [33, 1, 64]
    for code in ("e4m3", "int8"):
        c, table = paged(res, lens, 64, 2, 128, code, 9)
        q = torch.randn((3, 4, 128), device="cuda").bfloat16()
        want = c.attend(q, table, ints(lens))
        raw_k, raw_v = c.k_codes.view(torch.uint8), c.v_codes.view(torch.uint8)
        for b, n in enumerate(lens):
            page = int(table[b, 0])
            raw_k[page, :, n:] = 0x7f
            raw_v[page, :, :, n:] = 0xff
        used = set(table[:, 0].tolist())
        for p in range(c.num_blocks):
            if p not in used:
                c.k_scales[p] = float("nan")
                c.v_scales[p] = float("inf")
                raw_v[p] = 0x7f
        assert torch.equal(c.attend(q, table, ints(lens)), want)


@pytest.mark.parametrize("lens, nq", [([5000, 3, 700], None), ([700, 40, 3000], [300, 1, 17])])
def test_attend_in_place(res, lens, nq):
    """the results may take the queries' place: a workgroup reads no rows but its own"""
    c, table = paged(res, lens, 32, 2, 64, "int8", 9)
    offs = None if nq is None else [0, nq[0], nq[0] + nq[1], sum(nq)]
    q = torch.randn((len(lens) if nq is None else sum(nq), 8, 64), device="cuda").half()
    offsets = None if offs is None else ints(offs)
    want = c.attend(q, table, ints(lens), query_offsets=offsets)
    got = c.attend(q, table, ints(lens), query_offsets=offsets, out=q)
    assert got is q and torch.equal(got, want)


def test_attend_masked_scales(res):
    """a block whose scales are no numbers touches the rows that see it, and no others"""
    lens = [40]
    c, table = paged(res, lens, 16, 1, 64, "e4m3", 3)
    q = torch.randn((40, 2, 64), device="cuda").half()
    offs = ints([0, 40])
    want, _, tol = reference(c, q, table, lens, [0, 40], 1 / 8, True)
    # (an infinite scale of keys makes scores of -inf too, which are tokens of probability zero)
    for s, bad in ((c.k_scales, float("nan")), (c.v_scales, float("nan")), (c.v_scales, float("inf"))):
        old = s.clone()
        s[int(table[0, 2])] = bad
        got = c.attend(q, table, ints(lens), query_offsets=offs)
        s.copy_(old)
        # (not the same bits: values are accumulated in units of the largest scale)
        check(got[:32], None, want[:32], None, tol[:32])
        assert not bool(torch.isfinite(got[32:]).all(-1).any())


@pytest.mark.parametrize("nq, g", [(5, 2), (200, 1)])
def test_attend_masked_nan_codes(res, nq, g):
    """a NaN code of a key or a value reaches the rows that see its token, and no others"""
    lens = [300]
    c, table = paged(res, lens, 16, 1, 64, "e4m3", 3)
    q = torch.randn((nq, g, 64), device="cuda").bfloat16()
    offs = ints([0, nq])
    want, _, tol = reference(c, q, table, lens, [0, nq], 1 / 8, True)
    at = 300 - 3  # seen by the last three rows
    page, off = int(table[0, at // 16]), at % 16
    for codes, where in ((c.k_codes, (page, 0, off, 7)), (c.v_codes, (page, 0, 50, off))):
        raw = codes.view(torch.uint8)
        old = int(raw[where])
        for code in (0x7f, 0xff):
            raw[where] = code
            got = c.attend(q, table, ints(lens), query_offsets=offs)
            check(got[:nq - 3], None, want[:nq - 3], None, tol[:nq - 3])
            assert bool(got[nq - 3:, :, 50].isnan().all())
        raw[where] = old


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("nq", [1, 40])
def test_attend_scales_far_apart(res, code, nq):
    """blocks whose value scales lie up to 2^90 apart, and rows that see next to nothing of the large ones (probability and scale
    share an fp32 exponent of 2^-126 ..., which is where the limit of 2^100 comes from)"""
    lens = [160]
    c, table = paged(res, lens, 16, 1, 64, code, 5)
    far = [2.0 ** e for e in (-3, -45, 20, -30, 0, -40, 45, -20, -40, 5)]
    for i, x in enumerate(far):
        c.v_scales[int(table[0, i])] = x
    g = torch.Generator(device="cuda")
    g.manual_seed(nq)
    q = (torch.randn((nq, 4, 64), generator=g, device="cuda") * 2).half()
    for scale, lift in ((1 / 8, None), (1 / 8, 3), (1 / 8, 7), (4.0, 1)):
        old = c.k_codes.clone()
        if lift is not None:  # one block has nearly all the probability
            c.k_codes.view(torch.uint8)[int(table[0, lift])] = (q[0, 0].float() * 8).round().clamp(-100, 100).to(c.k_codes.dtype).view(torch.uint8)
        offs = ints([0, nq])
        want, wl, tol = reference(c, q, table, lens, [0, nq], scale, False)
        got, lse = c.attend(q, table, ints(lens), query_offsets=offs, scale=scale, causal=False, return_lse=True)
        # (beyond the type's range both are infinite)
        fits = want.abs() < torch.finfo(q.dtype).max * 0.999
        assert bool(((got.double() - want).abs() <= tol)[fits].all()), (code, scale, lift)
        assert bool((lse.double() - wl).abs().max() < 2 ** -9)
        c.k_codes.copy_(old)


def test_attend_zero_and_negative_scales(res):
    """values of a zero scale are zero whatever their codes; a negative scale counts as no number"""
    lens = [100, 100]
    c, table = paged(res, lens, 16, 2, 64, "int8", 4)
    c.v_scales[table[0, 1].long()] = 0.0
    c.k_scales[table[0, 2].long()] = 0.0
    for nq in (1, 40):
        q = torch.randn((2 * nq, 4, 64), device="cuda").half()
        offs = ints([0, nq, 2 * nq])
        want, _, tol = reference(c, q, table, lens, [0, nq, 2 * nq], 1 / 8, True)
        check(c.attend(q, table, ints(lens), query_offsets=offs), None, want, None, tol)
        for s in (c.k_scales, c.v_scales):
            old = s.clone()
            s[table[1, 0].long()] *= -1
            got = c.attend(q, table, ints(lens), query_offsets=offs)
            s.copy_(old)
            check(got[:nq], None, want[:nq], None, tol[:nq])
            assert bool(got[nq:].isnan().all())


def test_attend_bad_blocks_and_lengths(res):
    """a row that reaches a block that does not exist is NaN; the others are what they were"""
    lens = [100, 100, 100, 100]
    c, table = paged(res, lens, 16, 2, 64, "int8", 4)
    q = torch.randn((4, 4, 64), device="cuda").half()
    want = c.attend(q, table, ints(lens))
    bad = table.clone()
    bad[0, 6] = -1
    bad[1, 0] = c.num_blocks
    bad[3, 7] = -5  # not reached
    got = c.attend(q, bad, ints(lens))
    assert bool(got[:2].isnan().all()) and torch.equal(got[2:], want[2:])
    # lengths that the table cannot hold, and negative ones
    got = c.attend(q, table[:, :7].contiguous(), ints([100, 113, 2 ** 31 - 1, -3]))
    assert torch.equal(got[0], want[0]) and bool(got[1:3].isnan().all()) and bool((got[3] == 0).all())
    # offsets out of range are clamped: the call writes nothing outside `out`
    out = torch.full((6, 4, 64), 3.0, device="cuda").half()
    c.attend(q, table, ints(lens), query_offsets=ints([-7, 2, 2, 3, 900]), out=out[:4])
    assert bool((out[4:] == 3).all())


def test_attend_no_number_in_queries(res):
    lens = [70, 70]
    c, table = paged(res, lens, 16, 2, 64, "e4m3", 6)
    q = torch.randn((2, 4, 64), device="cuda").bfloat16()
    want = c.attend(q, table, ints(lens))
    q[0, 1, 5] = float("nan")
    got = c.attend(q, table, ints(lens))
    assert bool(got[0, 1].isnan().all())
    keep = torch.ones((2, 4), dtype=torch.bool)
    keep[0, 1] = False
    assert torch.equal(got[keep], want[keep])


def test_attend_extreme_queries(res):
    """bf16 queries beyond fp16's range on both sides"""
    lens = [90, 90, 90]
    c, table = paged(res, lens, 32, 1, 64, "e4m3", 8)
    q = torch.randn((3, 4, 64), device="cuda").bfloat16()
    q[0] *= 2.0 ** 60
    q[1] *= 2.0 ** -100
    q[2, :, ::2] *= 2.0 ** -20
    scale = 1 / math.sqrt(64)
    got = c.attend(q, table, ints(lens))
    want, _, tol = reference(c, q, table, lens, None, scale, True)
    # scores of 2^60 leave one token: softmax picks it exactly in either arithmetic unless the two best are closer than fp32 tells
    check(got[1:], None, want[1:], None, tol[1:])
    assert bool(torch.isfinite(got).all())


def test_attend_beyond_32_bits(res):
    """blocks more than 2^32 bytes into the cache"""
    bs, h, d = 64, 8, 128
    n = (2 ** 32 // (bs * h * d)) + 40
    c = decoding.PagedCache(res, n, bs, h, d, "int8")
    small = filled(res, 8, h, bs, d, "int8", 1)
    at = torch.tensor([n - 1, 3, n - 5, n - 2, 0, n - 9, n // 2, n - 3], device="cuda")
    for name in ("k_codes", "v_codes", "k_scales", "v_scales"):
        getattr(c, name)[at] = getattr(small, name)
    lens = [8 * bs - 3]
    q = torch.randn((1, 8, d), device="cuda").bfloat16()
    near = small.attend(q, torch.arange(8, dtype=I32, device="cuda")[None], ints(lens))
    far = c.attend(q, at.to(I32)[None], ints(lens))
    assert torch.equal(near, far)
    k = torch.randn((3, h, d), device="cuda").bfloat16()
    slots = ints([(n - 7) * bs, (n - 7) * bs + 1, (n - 4) * bs])
    c.add(k, k, slots)
    kk, vv = c.reconstruct(ints([n - 7, n - 4]))
    assert torch.equal(kk, vv)
    assert bool(((kk[0, :, :2] - k[:2].float().transpose(0, 1)).abs().amax() < 0.05)) and bool((kk[0, :, 2:] == 0).all())


# ------------------------------------------------------------------------------------------------ adding and reading
def nearest(x, code):
    if code == "int8":
        return torch.round(x)
    _, e = torch.frexp(x)
    step = torch.exp2((e.double() - 1).clamp(min=-6) - 3)
    return torch.round(x / step) * step


def add_reference(kv, scales, x, slots, bs, code):
    """values [n, h, bs, d] (codes as float64) and scales (float64) after adding x [tokens, h, d]"""
    last = {}
    for t, s in enumerate(slots):
        if 0 <= s < kv.shape[0] * bs:
            last[s] = t
    pages = {}
    for s, t in last.items():
        pages.setdefault(s // bs, []).append((s % bs, t))
    for p, at in pages.items():
        off = [o for o, _ in at]
        new = x[[t for _, t in at]].double().transpose(0, 1)  # [h, tokens, d]
        for h in range(x.shape[1]):
            old = 0.0 if 0 in off else float(scales[p, h])
            amax = float(new[h].abs().max()) if bool(torch.isfinite(new[h]).all()) else math.nan
            if math.isnan(amax) or not (0 <= old < math.inf):
                after = math.nan
            else:
                after = max(old, 2.0 ** max(math.ceil(math.log2(amax / QMAX[code])), -126) if amax > 0 else 0.0)
            if 0 in off:
                kv[p, h] = 0
            elif after == after and after > 0 and old != after:
                kv[p, h] = nearest(kv[p, h] * (old / after), code)
            elif after == 0:
                kv[p, h] = 0
            kv[p, h][off] = nearest(new[h] / after, code) if after == after and after > 0 else torch.zeros_like(new[h])
            scales[p, h] = after


def add_both(res, c, k, v, slots):
    """add on the device and in the reference; everything has to be equal, codes and scales"""
    kk, ks = c.k_codes.double().cpu(), c.k_scales.double().cpu()
    vv, vs = c.v_codes.double().cpu().transpose(2, 3).contiguous(), c.v_scales.double().cpu()
    add_reference(kk, ks, k.cpu(), slots, c.block_size, c.code)
    add_reference(vv, vs, v.cpu(), slots, c.block_size, c.code)
    c.add(k, v, ints(slots))
    assert torch.equal(c.k_scales.double().cpu().nan_to_num(-1), ks.nan_to_num(-1))
    assert torch.equal(c.v_scales.double().cpu().nan_to_num(-1), vs.nan_to_num(-1))
    assert torch.equal(c.k_codes.double().cpu(), kk)
    assert torch.equal(c.v_codes.double().cpu().transpose(2, 3), vv)


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("bs, h, d, dt", [(16, 2, 128, torch.bfloat16), (64, 3, 96, torch.float16), (256, 1, 64, torch.bfloat16),
                                          (32, 5, 256, torch.float16), (128, 2, 192, torch.bfloat16)])
def test_add(res, code, bs, h, d, dt):
    g = torch.Generator(device="cuda")
    g.manual_seed(bs + d)
    c = decoding.PagedCache(res, 9, bs, h, d, code)
    rnd = lambda n, s: (torch.randn((n, 3, h, d), generator=g, device="cuda") * s).to(dt)  # noqa: E731
    # a prompt over two and a half blocks, then tokens that grow, that are small, that begin a block, that are skipped
    n = 2 * bs + bs // 2 + 1
    x = rnd(n, 1.0)
    add_both(res, c, x[:, 0], x[:, 2], [4 * bs + i for i in range(bs)] + [bs + i for i in range(bs)] + [7 * bs + i for i in range(n - 2 * bs)])
    for scale, slots in ((5.0, [7 * bs + n - 2 * bs, 4 * bs + 3, -1]), (0.01, [7 * bs + n - 2 * bs + 1, 8 * bs, 9 * bs]),
                         (100.0, [8 * bs + 1, 2 ** 31 - 1, -2 ** 31]), (1.0, [4 * bs, 5, 4 * bs + 1]),
                         (3.0, [bs + 2, 7 * bs + 1, bs + 2, 8 * bs + 2, bs + 1])):  # a slot twice: the last wins; blocks in turn
        x = rnd(len(slots), scale)
        add_both(res, c, x[:, 1], x[:, 0], slots)
    # zeros, and the largest and smallest numbers of the type
    x = rnd(4, 1.0) * 0
    add_both(res, c, x[:, 0], x[:, 1], [2 * bs, 2 * bs + 1, 3 * bs, 2 * bs + 2])
    big, tiny = torch.finfo(dt).max, torch.finfo(dt).smallest_normal
    x[0, :, 0, 0], x[1, :, 0, 1], x[2], x[3, :, :, ::2] = big, -big, tiny, -tiny
    add_both(res, c, x[:, 0], x[:, 1], [2 * bs + 3, 3 * bs + 1, 6 * bs, 6 * bs + 1])
    # what is no number makes the block's scale none, until the block is begun anew
    x = rnd(3, 1.0)
    x[0, 0, 0, 7], x[1, 1, h - 1, 3] = float("inf"), float("nan")
    add_both(res, c, x[:, 0], x[:, 1], [6 * bs + 2, 3 * bs + 2, 2 * bs + 4])
    x = rnd(2, 1.0)
    add_both(res, c, x[:, 0], x[:, 1], [6 * bs + 3, 3 * bs + 3])
    add_both(res, c, x[:, 0], x[:, 1], [6 * bs, 3 * bs])


def test_add_nothing_and_many(res):
    c = decoding.PagedCache(res, 70, 16, 2, 64, "e4m3")
    x = torch.randn((1000, 2, 64), device="cuda").bfloat16()
    c.add(x[:0], x[:0], ints([]))
    g = torch.Generator()
    g.manual_seed(0)
    add_both(res, c, x, x.flip(0), torch.randperm(1120, generator=g)[:1000].tolist())  # no order at all


@pytest.mark.parametrize("bs, d, n", [(16, 64, 3000), (128, 256, 1500), (64, 96, 1025)])
def test_add_long_calls_and_odd_addresses(res, bs, d, n):
    """calls of more than a thousand tokens, whose workgroups share the scan for a block's tokens; rows that start anywhere"""
    g = torch.Generator(device="cuda")
    g.manual_seed(n)
    blocks = -(-n // bs) + 3
    for code in ("e4m3", "int8"):
        c = decoding.PagedCache(res, blocks, bs, 3, d, code)
        x = torch.randn((n, 2, 3, d + 3), generator=g, device="cuda").half()
        k, v = x[:, 0, :, 1:d + 1], x[:, 1, :, 2:d + 2]
        o = torch.Generator()
        o.manual_seed(bs)
        # runs of a block's slots, and a tail in no order that comes back to their blocks
        slots = [2 * bs + i for i in range(n - 70)] + torch.randint(0, blocks * bs, (70,), generator=o).tolist()
        add_both(res, c, k, v, slots)


@pytest.mark.parametrize("bs, h, d", [(16, 2, 64), (64, 1, 128), (256, 2, 96)])
@pytest.mark.parametrize("n", [512, 513, 2500])
def test_add_listed_blocks(res, bs, h, d, n):
    """around the number of tokens from which a call's blocks are listed: requests that take turns, skipped slots, the same slot
    again at the call's other end, a second call that comes back to the blocks"""
    g = torch.Generator(device="cuda")
    g.manual_seed(n + bs)
    blocks = -(-n // bs) + 4
    c = decoding.PagedCache(res, blocks, bs, h, d, "e4m3")
    k, v = (torch.randn((n, h, d), generator=g, device="cuda").bfloat16() for _ in range(2))
    half = n // 2
    slots = [(i // 2 if i % 2 else half + i // 2) for i in range(n)]
    slots[5], slots[n // 3], slots[n - 2], slots[n - 1] = -1, blocks * bs, 2**31 - 1, slots[0]
    add_both(res, c, k, v, slots)
    o = torch.Generator()
    o.manual_seed(n)
    again = torch.randperm(blocks * bs, generator=o)[:n].tolist()
    add_both(res, c, 2 * v, k, again + again[:max(0, n - len(again))])


@pytest.mark.parametrize("n", [300, 1000])
def test_add_captured(res, n):
    c = decoding.PagedCache(res, 80, 16, 2, 64, "int8")
    want = decoding.PagedCache(res, 80, 16, 2, 64, "int8")
    slots = ints(list(range(40, 40 + n)))
    k, v = torch.zeros((n, 2, 64), device="cuda").half(), torch.zeros((n, 2, 64), device="cuda").half()
    c.add(k, v, slots)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.add(k, v, slots)
    want.add(k, v, slots)
    for i in range(4):
        g = torch.Generator(device="cuda")
        g.manual_seed(i)
        k.copy_(torch.randn((n, 2, 64), generator=g, device="cuda") * 2**i)
        v.copy_(torch.randn((n, 2, 64), generator=g, device="cuda") * 2**i)
        slots.copy_(ints(torch.randperm(1280, generator=torch.Generator().manual_seed(i))[:n].tolist()))
        graph.replay()
        torch.cuda.synchronize()
        want.add(k, v, slots)
        for a, b in ((c.k_codes, want.k_codes), (c.v_codes, want.v_codes), (c.k_scales, want.k_scales), (c.v_scales, want.v_scales)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_reconstruct(res, code):
    for bs, h, d in ((16, 3, 64), (64, 2, 96), (256, 1, 256)):
        c = filled(res, 5, h, bs, d, code, bs)
        blocks = [3, 0, 3, 4]
        for dt in (torch.float32, torch.float16, torch.bfloat16):
            k, v = c.reconstruct(ints(blocks + [-1, 5]), dt)
            for i, p in enumerate(blocks):
                for hh in range(h):
                    wk, wv = values(c, p, hh)
                    # one product in fp32, one rounding to the type
                    assert torch.equal(k[i, hh], wk.float().to(dt)) and torch.equal(v[i, hh], wv.float().to(dt))
            assert bool(k[4:].isnan().all()) and bool(v[4:].isnan().all())
    k, v = c.reconstruct(ints([]))
    assert k.shape[0] == 0


# ------------------------------------------------------------------------------------------------ block tables
def plan_reference(table, owned, old, new, ring, state, bs, room):
    total, cols = len(ring), len(table[0]) if table else 0
    head, count = state
    taken = asked = tokens = given = 0
    off, slots, granted, lens = [0], [], [], []
    pushes = []
    for b in range(len(old)):
        ok = 0 <= old[b] <= cols * bs and 0 <= new[b] <= cols * bs
        have, want = -(-old[b] // bs), -(-new[b] // bs)
        need, tok = (want - have, max(new[b] - old[b], 0)) if ok else (0, 0)
        asked += max(need, 0)
        tokens += tok
        g = ok and (tok == 0 or (asked <= count and tokens <= room))
        granted.append(int(g))
        lens.append(new[b] if g else old[b])
        if g:
            for i in range(max(need, 0)):
                p = ring[(head + taken) % total]
                taken += 1
                table[b][have + i] = p
                if owned:
                    owned[b][have + i] = p
            for i in range(max(-need, 0)):
                pushes.append((owned or table)[b][want + i])
            for i in range(tok):
                pos = old[b] + i
                p = table[b][pos // bs]
                slots.append(p * bs + pos % bs if 0 <= p < total else -1)
        off.append(len(slots))
    for p in pushes:
        ring[(head + count + given) % total] = p
        given += 1
    return lens, [(head + taken) % total, min(count - taken + given, total)], off, slots + [-1] * (room - len(slots)), granted


def plan_both(res, table, owned, old, new, ring, state, bs, room, inplace=False):
    t, r, o, s = ints(table).reshape(len(old), -1), ints(ring), ints(old), torch.tensor(state, dtype=torch.int64, device="cuda")
    w = ints(owned) if owned else None
    kw = dict(lengths_out=o, free_state_out=s) if inplace else {}
    p = decoding.plan_blocks(res, t, o, ints(new), r, s, bs, room, owned_table=w, **kw)
    lens, st, off, slots, granted = plan_reference(table, owned, list(old), new, ring, state, bs, room)
    assert p.lengths.tolist() == lens and p.free_state.tolist() == st
    assert p.query_offsets.tolist() == off and p.slots.tolist() == slots and p.granted.tolist() == granted
    assert t.tolist() == table and r.tolist() == ring
    if owned:
        assert w.tolist() == owned
    if inplace:
        assert o.tolist() == lens and s.tolist() == st
    return lens, st


@pytest.mark.parametrize("n, bs, cols, steps, room", [(1, 16, 4, 12, 70), (7, 16, 9, 20, 200), (50, 64, 5, 8, 5000), (1500, 16, 6, 4, 40000),
                                                      (2, 1, 30, 6, 70)])
def test_plan_blocks(res, n, bs, cols, steps, room):
    """requests that grow, shrink, finish and come again; blocks and slots run short"""
    import random
    rng = random.Random(n)
    total = max(3, int(n * cols * 0.6))
    ring = list(range(total))
    rng.shuffle(ring)
    table = [[-1] * cols for _ in range(n)]
    owned = [[-1] * cols for _ in range(n)] if n % 2 else None
    lens, state = [0] * n, [total // 2, total]
    for step in range(steps):
        new = [rng.choice([x + 1, x, 0, rng.randint(0, cols * bs), min(x + bs, cols * bs), max(x - 3, 0)]) for x in lens]
        for i in range(n // 9):
            new[rng.randrange(n)] = rng.choice([-1, cols * bs + 1, 2 ** 31 - 1])
        lens, state = plan_both(res, table, owned, lens, new, ring, state, bs, room, inplace=step % 2 == 1)
        held = sorted(p for b in range(n) for p in (owned or table)[b][:-(-lens[b] // bs)])
        free = sorted(ring[(state[0] + i) % total] for i in range(state[1]))
        assert sorted(held + free) == list(range(total))  # every block once


def test_plan_blocks_refuses_on_the_device(res):
    # no blocks left; no slots left; a table that names no block; an empty batch
    plan_both(res, [[0, 1], [2, -1]], None, [32, 16], [32, 17], [7, 7, 7, 7], [1, 0], 16, 5)
    plan_both(res, [[0, 1], [2, -1], [3, -1]], None, [20, 5, 0], [22, 9, 1], [4, 5, 6, 7, 8], [3, 2], 16, 4)
    plan_both(res, [[9, 1]], None, [5], [8], [0, 1, 2], [0, 1], 16, 5)
    t = torch.zeros((0, 3), dtype=I32, device="cuda")
    p = decoding.plan_blocks(res, t, ints([]), ints([]), ints([1, 2]), torch.tensor([1, 1], device="cuda"), 16, 4)
    assert p.query_offsets.tolist() == [0] and p.slots.tolist() == [-1] * 4 and p.free_state.tolist() == [1, 1]


# ------------------------------------------------------------------------------------------------ beams
def beam_reference(logits, scores, keep, finished, pad):
    x = logits.double().cpu()
    n, w, v = x.shape
    lse = torch.logsumexp(x, -1, keepdim=True)
    val = scores.double().cpu()[:, :, None] + (x - lse)
    if finished is not None:
        f = finished.bool().cpu()
        val[f] = -math.inf
        val[:, :, pad][f] = scores.double().cpu()[f]
    val = torch.where(val > -math.inf, val, torch.full_like(val, -math.inf)).reshape(n, w * v)
    s, i = torch.sort(val, dim=1, descending=True, stable=True)
    k = min(keep, w * v)
    s, i = s[:, :k], i[:, :k]
    none = s == -math.inf
    s = torch.cat([s, torch.full((n, keep - k), -math.inf, dtype=torch.float64)], 1)
    pad1 = torch.full((n, keep - k), -1)
    return s, torch.cat([torch.where(none, -1, i // v), pad1], 1), torch.cat([torch.where(none, -1, i % v), pad1], 1)


def beam_check(res, logits, scores, keep, finished=None, pad=0):
    s, p, t = decoding.beam_select(res, logits, scores, keep, finished=finished, pad_token=pad)
    ws, wp, wt = beam_reference(logits, scores, keep, finished, pad)
    assert torch.equal(p.cpu().long(), wp) and torch.equal(t.cpu().long(), wt)
    fin = torch.isfinite(ws)
    assert torch.equal(torch.isfinite(s.cpu()), fin)
    # the log-sum is off by ~1e-7 at most (exponentials and lane sums in fp32), the result is rounded to fp32
    err = (s.cpu().double() - ws).abs()[fin]
    assert not fin.any() or bool((err <= 2 ** -22 + 2 ** -24 * ws[fin].abs()).all())


@pytest.mark.parametrize("n, w, v, keep, dt", [
    (1, 1, 1, 1, torch.float32), (1, 4, 32000, 4, torch.float32), (3, 5, 1001, 10, torch.bfloat16), (2, 64, 777, 64, torch.float16),
    (4, 8, 128001, 16, torch.bfloat16), (40, 3, 63, 6, torch.float16), (2, 2, 5, 64, torch.float32), (1, 7, 4096, 1, torch.float16),
    (300, 2, 2049, 2, torch.float32)])
def test_beam_select(res, n, w, v, keep, dt):
    g = torch.Generator(device="cuda")
    g.manual_seed(v)
    # distinct values of a type with few digits still tie often inside a row: ties go to the lowest token
    x = (torch.randn((n, w, v), generator=g, device="cuda") * 3).to(dt)
    s = -torch.rand((n, w), generator=g, device="cuda") * 5
    beam_check(res, x, s, keep)
    f = torch.rand((n, w), generator=g, device="cuda") < 0.4
    beam_check(res, x, s, keep, finished=f, pad=v - 1)
    beam_check(res, x, s, keep, finished=(f * 3).to(torch.uint8), pad=v // 2)


def test_beam_select_ties_and_order(res):
    # constant rows, sorted rows, equal beams, the best ones side by side in one lane
    for v in (70, 5000, 40000):
        beam_check(res, torch.zeros((2, 3, v), device="cuda"), torch.zeros((2, 3), device="cuda"), 12)
        up = torch.arange(v, device="cuda").float()[None, None].repeat(1, 4, 1) / v
        beam_check(res, up, torch.zeros((1, 4), device="cuda"), 9)
        beam_check(res, -up.half(), torch.tensor([[0.0, -1.0, 0.0, -2.0]], device="cuda"), 64)
        x = torch.randn((1, 2, v), device="cuda")
        x[0, 0, v // 2:v // 2 + 40] = 50.0 + torch.arange(min(40, v - v // 2), device="cuda") % 7
        beam_check(res, x, torch.zeros((1, 2), device="cuda"), 33)


def test_beam_select_masks(res):
    v = 3001
    x = torch.randn((4, 3, v), device="cuda")
    x[0, 0] = -math.inf                       # nothing left of a beam
    x[0, 1, 10:] = -math.inf                  # ten tokens
    x[1, :, 5:] = torch.finfo(torch.float32).min
    x[2, 1, 7] = math.nan
    x[2, 2, 7] = math.inf
    x[3] = -math.inf
    s = torch.zeros((4, 3), device="cuda")
    s[1, 2] = -math.inf                       # a dead beam
    for keep in (4, 20):
        beam_check(res, x, s, keep)
        h = x.clone().clamp(min=-6e4).half()
        h[0, 0], h[0, 1, 10:], h[3] = -math.inf, -math.inf, -math.inf
        beam_check(res, h, s, keep)


def test_beam_select_strides(res):
    x = torch.randn((3, 5, 2, 1030), device="cuda").bfloat16()
    s = -torch.rand((3, 5), device="cuda")
    for view in (x[:, :, 1, 3:1004], x[:, :, 0, 1:], x[:, :, 1].transpose(0, 1)[:3, :3]):
        beam_check(res, view, s[:, :view.shape[1]].contiguous(), 7)


@pytest.mark.parametrize("shape, dt", [((3,), torch.bfloat16), ((1,), torch.int8), ((8191,), torch.bfloat16), ((4, 33, 128), torch.float32),
                                       ((20000,), torch.uint8), ((), torch.int64), ((5, 0), torch.float32)])
def test_reorder_beams(res, shape, dt):
    n, w = 5, 3
    x = torch.randint(-100, 100, (n, w) + shape, device="cuda").to(dt)
    wide = torch.randint(-100, 100, (n, w + 2, 2) + shape, device="cuda").to(dt)[:, 1:4, 1]
    for k in (3, 7):
        p = torch.randint(-1, w + 1, (n, k), device="cuda", dtype=I32)
        ok = (p >= 0) & (p < w)
        row = torch.arange(n, device="cuda")[:, None]
        got = decoding.reorder_beams(res, [x, wide, x[:, :1].expand(x.shape)], p)
        for g, t in zip(got, (x, wide, x[:, :1].expand(x.shape))):
            want = t[row, p.long().clamp(0, w - 1)]
            want[~ok] = 0
            assert g.dtype == t.dtype and torch.equal(g, want)


def test_reorder_many_states(res):
    states = [torch.randn((2, 4, 1 + 17 * i), device="cuda") for i in range(150)]
    p = ints([[3, 3, 0, 1], [2, 2, 2, 2]])
    for g, t in zip(decoding.reorder_beams(res, states, p), states):
        assert torch.equal(g, t[torch.arange(2, device="cuda")[:, None], p.long()])
    assert decoding.reorder_beams(res, [], p) == []


@pytest.mark.parametrize("layers, bs, d, lens", [(1, 16, 64, [40, 16, 0]), (40, 32, 96, [31, 70, 64])])
def test_fork_blocks(res, layers, bs, d, lens):
    n, w, cols = len(lens), 4, 6
    rows = n * w
    caches = [filled(res, rows * (cols + 1), 2, bs, d, "e4m3" if i % 2 else "int8", i) for i in range(layers)]
    perm = torch.randperm(rows * (cols + 1)).to(I32).cuda()
    table, spare = perm[:rows * cols].reshape(rows, cols).contiguous(), perm[rows * cols:].clone()
    lengths = ints([l for l in lens for _ in range(w)])
    parents = ints([[3, 0, 0, 1], [1, 1, 7, -1], [2, 3, 0, 0]])
    before = [[t.clone() for t in (c.k_codes, c.v_codes, c.k_scales, c.v_scales)] for c in caches]
    t2, l2, s2 = decoding.fork_blocks(res, caches, table, lengths, spare, parents)
    for r in range(rows):
        b, j = divmod(r, w)
        p = int(parents[b, j])
        src = b * w + p if 0 <= p < w else r
        length = lens[b]
        assert int(l2[r]) == length
        want = table[src].clone()
        if length % bs:
            col = length // bs
            want[col] = spare[r]
            assert int(s2[r]) == int(table[r, col])
            for c, old in zip(caches, before):
                for now, was in zip((c.k_codes, c.v_codes, c.k_scales, c.v_scales), old):
                    assert torch.equal(now[int(spare[r])].view(torch.uint8), was[int(table[src, col])].view(torch.uint8))
        else:
            assert int(s2[r]) == int(spare[r])
        assert torch.equal(t2[r], want)
    # every block that was not a spare one is what it was
    for c, old in zip(caches, before):
        assert torch.equal(c.k_codes[table.flatten().long()].view(torch.uint8), old[0][table.flatten().long()].view(torch.uint8))
    # a spare block that does not exist
    t3, _, _ = decoding.fork_blocks(res, caches[:1], table, lengths, torch.full_like(spare, -1), parents)
    assert int(t3[0, lens[0] // bs]) == -1


# ------------------------------------------------------------------------------------------------ together, streams, graphs
def test_beam_decoding_over_a_paged_cache(res):
    """prompt, then steps of plan / add / attend / select / fork / reorder; each beam's context is followed on the host"""
    torch.manual_seed(0)
    n, w, h, hq, d, bs, layers, vocab = 2, 3, 2, 4, 64, 16, 2, 50
    rows, cols = n * w, 8
    emb = torch.randn((vocab, 2, h, d), device="cuda").bfloat16()  # a token's keys and values
    head = torch.randn((hq * d, vocab), device="cuda")
    total = rows * (cols + 1)
    caches = [decoding.PagedCache(res, total, bs, h, d, c) for c in ("e4m3", "int8")][:layers]
    pages = torch.randperm(total).to(I32).cuda()
    spare0, ring = pages[:rows].clone(), torch.cat([pages[rows:], torch.full((rows,), -1, dtype=I32, device="cuda")])
    state = torch.tensor([0, total - rows], dtype=torch.int64, device="cuda")
    view = torch.full((rows, cols), -1, dtype=I32, device="cuda")
    owned, lengths, spare = view.clone(), torch.zeros(rows, dtype=I32, device="cuda"), spare0.clone()
    history = [[int(x) for x in torch.randint(0, vocab, (21,))] for _ in range(n) for _ in range(w)]
    history = [list(history[(r // w) * w]) for r in range(rows)]  # the beams of an item share its prompt
    new = [list(x) for x in history]
    scores = torch.tensor([[0.0] + [-math.inf] * (w - 1)] * n, device="cuda")
    told = torch.zeros((n, w, 0), dtype=I32, device="cuda")
    for step in range(30):
        want = ints([len(x) for x in history])
        p = decoding.plan_blocks(res, view, lengths, want, ring, state, bs, sum(map(len, new)) + 2, owned_table=owned, free_state_out=state)
        lengths = p.lengths
        assert p.granted.tolist() == [1] * rows
        tok = torch.tensor([t for x in new for t in x] + [0, 0], device="cuda")
        q = torch.randn((tok.numel(), hq, d), device="cuda").bfloat16()
        outs = []
        for c in caches:
            c.add(emb[tok, 0], emb[tok, 1], p.slots)
            outs.append(c.attend(q, view, lengths, query_offsets=p.query_offsets))
        # the cache holds each beam's own context: codes are within half a step of the tokens' values (a step twice: a scale that
        # grew has rounded them again)
        for c, out in zip(caches, outs):
            for r in range(rows):
                m = len(history[r])
                k, v = c.reconstruct(view[r, :-(-m // bs)])
                k, v = (x.transpose(1, 2).reshape(-1, h, d)[:m] for x in (k, v))
                e = emb[torch.tensor(history[r], device="cuda")].float()
                room = 2 ** -3 * e.abs() + 0.02 if c.code == "e4m3" else 0.07
                assert bool(((k - e[:, 0]).abs() <= room if c.code == "int8" else ((k - e[:, 0]).abs() <= room[:, 0])).all())
                assert bool(((v - e[:, 1]).abs() <= room if c.code == "int8" else ((v - e[:, 1]).abs() <= room[:, 1])).all())
            o, _, tol = reference(c, q[:-2], view, want.tolist(), p.query_offsets.tolist(), 1 / math.sqrt(d), True)
            check(out[:-2], None, o, None, tol, step)
        last = outs[0][p.query_offsets[1:].long() - 1].float().reshape(n, w, hq * d)
        logits = (last @ head) * 3
        wp = beam_reference(logits, scores, w, None, 0)
        scores, parents, tokens = decoding.beam_select(res, logits, scores, w)
        assert torch.equal(parents.cpu().long(), wp[1]) and torch.equal(tokens.cpu().long(), wp[2])
        told = torch.cat([decoding.reorder_beams(res, [told], parents)[0], tokens[:, :, None]], 2)
        view, lengths, spare = decoding.fork_blocks(res, caches, view, lengths, spare, parents)
        history = [history[(r // w) * w + int(parents[r // w, r % w])] + [int(tokens[r // w, r % w])] for r in range(rows)]
        new = [[x[-1]] for x in history]
    assert told.shape[2] == 30 and [x[21:] for x in history] == told.reshape(rows, -1).tolist()
    # everything goes back: the blocks that each row was given, whoever's table names them now
    p = decoding.plan_blocks(res, view, lengths, torch.zeros_like(lengths), ring, state, bs, 1, owned_table=owned, free_state_out=state)
    free = sorted(ring[(int(state[0]) + i) % total].item() for i in range(int(state[1])))
    assert free == sorted(pages[rows:].tolist())


def test_calls_follow_the_current_stream_and_keep_the_device(res):
    lens = [3000, 77]
    c, table = paged(res, lens, 16, 2, 128, "e4m3", 1)
    q = torch.randn((2, 8, 128), device="cuda").bfloat16()
    want = c.attend(q, table, ints(lens))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a = torch.randn((4096, 4096), device="cuda")
        for _ in range(8):
            a = a @ a * 1e-4
        late = q + (a[0, 0] * 0).nan_to_num().bfloat16()  # ready only when the products are
        got = c.attend(late, table, ints(lens))
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    assert torch.cuda.current_device() == 0


def test_captured_into_a_graph(res):
    """a decoding step in a graph, replayed with other inputs, eager work between the replays; two graphs side by side"""
    n, h, hq, d, bs, cols = 3, 2, 8, 128, 16, 300
    total = n * cols
    torch.manual_seed(1)

    def make(code):
        c = filled(res, total, h, bs, d, code, 3)
        st = dict(c=c, table=torch.full((n, cols), -1, dtype=I32, device="cuda"), lengths=ints([0, 0, 0]), new=ints([0, 0, 0]),
                  ring=torch.randperm(total).to(I32).cuda(), state=torch.tensor([5, total], dtype=torch.int64, device="cuda"),
                  k=torch.randn((n, h, d), device="cuda").bfloat16(), q=torch.randn((n, hq, d), device="cuda").bfloat16(),
                  scores=torch.zeros((1, n), device="cuda"), head=torch.randn((d, 400), device="cuda"))
        # a long context to begin with
        p = decoding.plan_blocks(res, st["table"], st["lengths"], ints([4000, 30, 15]), st["ring"], st["state"], bs, 5000,
                                 lengths_out=st["lengths"], free_state_out=st["state"])
        x = torch.randn((5000, h, d), device="cuda").bfloat16()
        c.add(x, x, p.slots)
        return st

    def step(st):
        p = decoding.plan_blocks(res, st["table"], st["lengths"], st["new"], st["ring"], st["state"], bs, n, lengths_out=st["lengths"],
                                 free_state_out=st["state"])
        st["c"].add(st["k"], st["k"], p.slots)
        o = st["c"].attend(st["q"], st["table"], st["lengths"])
        sel = decoding.beam_select(res, (o.float()[:, 0] @ st["head"])[None], st["scores"], n)
        return (o, p.slots) + sel + tuple(decoding.reorder_beams(res, [o[None]], sel[1]))

    a, b = make("e4m3"), make("int8")
    ea, eb = make("e4m3"), make("int8")  # the same, for the eager results
    for x, y in ((a, ea), (b, eb)):
        for key in ("table", "lengths", "ring", "state", "k", "q", "head"):
            y[key].copy_(x[key])
        for name in ("k_codes", "v_codes", "k_scales", "v_scales"):
            getattr(y["c"], name).copy_(getattr(x["c"], name))
    graphs = []
    for st in (a, b):
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            out = step(st)
        graphs.append((g, out))
    for it in range(6):
        for st, e, (g, out) in ((a, ea, graphs[0]), (b, eb, graphs[1])):
            k, q = torch.randn((n, h, d), device="cuda").bfloat16(), torch.randn((n, hq, d), device="cuda").bfloat16()
            for x in (st, e):
                x["k"].copy_(k)
                x["q"].copy_(q)
                x["new"].copy_(x["lengths"] + 1)
            g.replay()
            want = step(e)
            torch.cuda.synchronize()
            for i, (x, y) in enumerate(zip(out, want)):
                assert torch.equal(x, y), (it, i)
            assert torch.equal(st["table"], e["table"]) and torch.equal(st["state"], e["state"])


def test_refusals_on_the_device(res):
    c = filled(res, 4, 2, 16, 64, "e4m3", 0)
    q, t, l = torch.zeros((1, 4, 64), device="cuda").half(), torch.zeros((1, 4), dtype=I32, device="cuda"), ints([3])
    for bad in (dict(q=q.cpu()), dict(block_table=t.cpu()), dict(lengths=l.long()), dict(q=q.float()), dict(q=q[:, :3]),
                dict(q=q[:, :, :32]), dict(lengths=ints([1, 2])), dict(q=q.repeat(2, 1, 1)), dict(query_offsets=ints([0, 1, 1])),
                dict(out=q.bfloat16()), dict(out=q[:, :2]), dict(scale=float("nan")), dict(block_table=t.expand(1, 4)[:, ::2])):
        with pytest.raises((ValueError, TypeError, faiss_amd.FaissAmdError)):
            c.attend(**{**dict(q=q, block_table=t, lengths=l), **bad})
    with pytest.raises(faiss_amd.FaissAmdError):
        decoding.beam_select(res, torch.zeros((1, 65, 10), device="cuda"), torch.zeros((1, 65), device="cuda"), 2)
    with pytest.raises(ValueError):
        decoding.PagedCache(res, 4, 24, 2, 64)
    with pytest.raises(ValueError):
        decoding.reorder_beams(res, [torch.zeros((2, 3, 4), device="cuda").transpose(2, 1)], ints([[0], [0]]))
    # host memory and a workspace that is too small are errors of the library
    import ctypes
    lib = faiss_amd.load_library()
    host = torch.zeros(64, dtype=I32)
    assert lib.faiss_amd_PagedCache_reconstruct(res._h, c._ref, 1, host.data_ptr(), 1, q.data_ptr(), q.data_ptr(), 0, None) == -2
    assert b"device memory" in lib.faiss_amd_get_last_error() or b"resources' device" in lib.faiss_amd_get_last_error()
    a = decoding._BeamStruct(q.data_ptr(), 8, 8, t.data_ptr(), None, q.data_ptr(), q.data_ptr(), q.data_ptr(), 8, 1, 1, 1, 0, 2, 0, q.data_ptr(), 1)
    assert lib.faiss_amd_beam_select(res._h, ctypes.byref(a), None) == -2 and b"workspace" in lib.faiss_amd_get_last_error()


def test_add_without_workspace_is_refused(res):
    c = decoding.PagedCache(res, 40, 16, 1, 64)
    x, slots = torch.zeros((513, 1, 64), device="cuda").half(), ints(list(range(513)))
    a = decoding._AddStruct(x.data_ptr(), x.data_ptr(), 64, 64, 64, 64, slots.data_ptr(), 513, decoding._HALF[torch.float16], 0, None)
    with pytest.raises(RuntimeError, match="workspace must be provided"):
        decoding._check(c._lib.faiss_amd_PagedCache_add(res._h, c._ref, decoding._byref(a), None))
