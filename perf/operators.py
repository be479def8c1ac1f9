"""Workloads of the decoding operators: block planning, the 8-bit paged cache, attention over it, beam selection, reordering.

``own`` selects who computes a pass: the plain torch forms below (False) or the kernels of faiss_amd.decoding (True)."""
import math

import torch

own = False

QMAX = {"e4m3": 448.0, "int8": 127.0}
DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CODE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
DEV = "cuda"


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a scheduler's step between two decoding steps: every request grows by one token, a sixteenth of them need a block
        dict(name="plan_step", op="plan", batch=256, block=16, longest=4096, grow=1, leave=0),
        # admission of prompts while finished requests return their blocks
        dict(name="plan_prompts", op="plan", batch=64, block=64, longest=8192, grow=6000, leave=9),
        # the keys and values of one decoding step of a full batch
        dict(name="add_step", op="add", tokens=256, each=1, heads=8, dim=128, block=16, code="e4m3", dtype="bf16"),
        # the keys and values of a batch of prompts, ragged behind their last full block
        dict(name="add_prompts", op="add", tokens=16389, each=2731, heads=8, dim=128, block=64, code="int8", dtype="fp16"),
        # one user, one token: the smallest call, where latency counts
        dict(name="attend_token", op="attend", batch=1, queries=1, longest=1000, ragged=False, heads=32, kv_heads=8, dim=128,
             block=16, code="e4m3", dtype="bf16"),
        # a serving batch of ragged contexts, one token each
        dict(name="attend_batch", op="attend", batch=64, queries=1, longest=16384, ragged=True, heads=32, kv_heads=8, dim=128,
             block=64, code="e4m3", dtype="bf16"),
        # few very long contexts behind one shared key-value head
        dict(name="attend_long", op="attend", batch=3, queries=1, longest=131071, ragged=False, heads=16, kv_heads=1, dim=256,
             block=32, code="int8", dtype="fp16"),
        # prompts in chunks behind earlier chunks
        dict(name="attend_prompt", op="attend", batch=4, queries=2048, longest=8192, ragged=True, heads=16, kv_heads=4, dim=128,
             block=64, code="e4m3", dtype="bf16"),
        # one sentence, four beams
        dict(name="beams_one", op="beams", batch=1, beams=4, keep=4, vocab=32000, dtype="fp32", finished=False),
        # a translation batch over a large vocabulary; twice the beams are kept, as programs do that set finished ones aside
        dict(name="beams_batch", op="beams", batch=64, beams=8, keep=16, vocab=128001, dtype="bf16", finished=True),
        # recurrent and convolution states of a small decoder's beams, layer by layer
        dict(name="reorder_states", op="reorder", batch=16, beams=5, layers=6, width=8191),
        # beams over the paged cache: tables change hands, partly filled blocks are copied
        dict(name="fork_blocks", op="fork", batch=32, beams=8, layers=8, heads=8, dim=128, block=64, longest=4000, code="e4m3"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "add", "attend", "attend", "beams", "reorder", "fork"])
    block = rng.choice([16, 32, 64, 128])
    code = rng.choice(["e4m3", "int8"])
    dtype = rng.choice(["bf16", "fp16"])
    dim = rng.choice([64, 96, 128, 192, 256])
    if op == "plan":
        longest = _log(rng, 64, 16384)
        return dict(op=op, batch=_log(rng, 1, 1000), block=block, longest=longest, grow=_log(rng, 1, min(longest, 512)),
                    leave=rng.randint(0, 5))
    if op == "add":
        tokens = _log(rng, 1, 16389)
        return dict(op=op, tokens=tokens, each=rng.choice([1, _log(rng, 1, tokens)]), heads=rng.choice([1, 2, 3, 8]), dim=dim,
                    block=block, code=code, dtype=dtype)
    if op == "attend":
        kv = rng.choice([1, 2, 3, 8])
        queries = rng.choice([1, 1, rng.randint(2, 9), _log(rng, 16, 1500)])
        longest = queries + _log(rng, 1, 30000)
        batch, heads = _log(rng, 1, 48), kv * rng.choice([1, 3, 4, 8])
        while batch > 1 and (batch * longest * kv > 500000 or batch * queries * longest * heads * dim > 2 ** 36):
            batch //= 2
        while batch * queries * longest * heads * dim > 2 ** 36:
            queries, longest = queries // 2, longest // 2 + 1
        return dict(op=op, batch=batch, queries=queries, longest=longest, ragged=rng.random() < 0.7, heads=heads, kv_heads=kv, dim=dim,
                    block=block, code=code, dtype=dtype)
    if op == "beams":
        beams = rng.choice([1, 3, 4, 8, 12])
        batch = _log(rng, 1, 64)
        vocab = _log(rng, 100, 128001)
        while batch > 1 and batch * beams * vocab > 2 ** 25:
            batch //= 2
        return dict(op=op, batch=batch, beams=beams, keep=beams * rng.choice([1, 2]), vocab=vocab,
                    dtype=rng.choice(["bf16", "fp16", "fp32"]), finished=rng.random() < 0.5)
    if op == "reorder":
        return dict(op=op, batch=_log(rng, 1, 64), beams=rng.choice([2, 3, 5, 8]), layers=rng.randint(1, 12), width=_log(rng, 1, 16384))
    return dict(op=op, batch=_log(rng, 1, 32), beams=rng.choice([2, 3, 4, 8]), layers=rng.randint(1, 8), heads=rng.choice([1, 3, 8]),
                dim=dim, block=block, longest=_log(rng, 20, 4000), code=code)


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _blocks(length, block):
    return (length + block - 1) // block


def _context_lengths(case, seed):
    """lengths of the contexts, drawn on the host so that work() and prepare() agree"""
    c = torch.Generator()
    c.manual_seed(seed * 7919 + 13)
    n, longest = case["batch"], case["longest"]
    low = case.get("queries", 1)
    if not case.get("ragged", True):
        return [longest - i for i in range(n)] if longest - n >= low else [longest] * n
    u = torch.rand(n, generator=c)
    lens = [max(low, int(round(longest * (0.25 + 0.75 * float(x))))) for x in u]
    lens[0] = longest
    return lens


def _query_counts(case):
    """queries of each request of a ragged prompt batch: the full chunk, and shorter last chunks"""
    n, q = case["batch"], case["queries"]
    if q == 1 or not case["ragged"]:
        return [q] * n
    return [max(1, q - (q // (n + 1)) * i) for i in range(n)]


def _codes(shape, code, g):
    x = torch.randn(shape, generator=g, device=DEV, dtype=torch.float16)
    if code == "e4m3":
        return (x * 60.0).clamp(-448, 448).to(torch.float8_e4m3fn)
    return (x * 30.0).round().clamp(-127, 127).to(torch.int8)


def _cache(blocks, heads, block, dim, code, g):
    """codes and scales of a cache that decoding has filled: unit keys and values, a power of two per block and head"""
    k = _codes((blocks, heads, block, dim), code, g)
    v = _codes((blocks, heads, dim, block), code, g)
    low = -7 if code == "e4m3" else -6
    ks = torch.exp2(torch.randint(low, low + 3, (blocks, heads), generator=g, device=DEV).float())
    vs = torch.exp2(torch.randint(low, low + 3, (blocks, heads), generator=g, device=DEV).float())
    return dict(k=k, v=v, ks=ks, vs=vs)


def _wrap(res, c):
    from faiss_amd.decoding import PagedCache
    return PagedCache.wrap(res, c["k"], c["v"], c["ks"], c["vs"])


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case=case)
    if own:
        import faiss_amd
        s["res"] = faiss_amd.StandardGpuResources(torch.cuda.current_device())
    op = case["op"]
    if op == "plan":
        c = torch.Generator()
        c.manual_seed(seed)
        n, block, longest, grow = case["batch"], case["block"], case["longest"], case["grow"]
        old = torch.randint(0, longest - min(grow, longest) + 1, (n,), generator=c, dtype=torch.int64)
        if grow == 1:
            new = old + 1
        else:
            new = old + torch.randint(0, min(grow, longest) + 1, (n,), generator=c, dtype=torch.int64)
        for i in range(min(case["leave"], n - 1)):
            new[(i * 7) % n] = 0
        have = (old + block - 1) // block
        width = _blocks(longest, block)
        total = int(n * width * 1.25) + 8
        pages = torch.randperm(total, generator=c).to(torch.int32)
        table = torch.full((n, width), -1, dtype=torch.int32)
        at = 0
        for i in range(n):
            m = int(have[i])
            table[i, :m] = pages[at:at + m]
            at += m
        free = total - at
        head = total // 3
        ring = torch.full((total,), -1, dtype=torch.int32)
        ring[(head + torch.arange(free)) % total] = pages[at:]
        s.update(table=table.to(DEV), old=old.to(torch.int32).to(DEV), new=new.to(torch.int32).to(DEV), ring=ring.to(DEV),
                 state=torch.tensor([head, free], dtype=torch.int64, device=DEV),
                 room=n * min(grow, longest) + 3)
        return s
    if op == "add":
        tokens, each, block, heads, dim = case["tokens"], case["each"], case["block"], case["heads"], case["dim"]
        dt = DTYPE[case["dtype"]]
        c = torch.Generator()
        c.manual_seed(seed)
        starts = list(range(0, tokens, each))
        slots, touched, page = [], [], 0
        for i, t0 in enumerate(starts):
            m = min(each, tokens - t0)
            first = (7 * i + 3) % block
            n = _blocks(first + m, block)
            # blocks of a request lie anywhere in the cache: strides that do not repeat
            ids = list(range(page, page + n))
            page += n
            touched += ids
            slots += [(ids[(first + j) // block], (first + j) % block) for j in range(m)]
        perm = torch.randperm(page, generator=c)
        sl = torch.tensor([int(perm[p]) * block + o for p, o in slots], dtype=torch.int32)
        s["cache"] = _cache(page, heads, block, dim, case["code"], g)
        # keys and values as they leave a fused projection: views of one matrix
        qkv = torch.randn((tokens, 3, heads, dim), generator=g, device=DEV, dtype=torch.float32).to(dt)
        s.update(key=qkv[:, 1], value=qkv[:, 2], slots=sl.to(DEV), touched=perm[torch.tensor(touched)].to(torch.int32).to(DEV))
        if own:
            s["handle"] = _wrap(s["res"], s["cache"])
        return s
    if op == "attend":
        lens, qn = _context_lengths(case, seed), _query_counts(case)
        block, n = case["block"], case["batch"]
        need = [_blocks(l, block) for l in lens]
        total = sum(need) + 5
        c = torch.Generator()
        c.manual_seed(seed)
        pages = torch.randperm(total, generator=c).to(torch.int32)
        table = torch.full((n, max(need)), -1, dtype=torch.int32)
        at = 0
        for i, m in enumerate(need):
            table[i, :m] = pages[at:at + m]
            at += m
        off = [0]
        for m in qn:
            off.append(off[-1] + m)
        dt = DTYPE[case["dtype"]]
        s["cache"] = _cache(total, case["kv_heads"], block, case["dim"], case["code"], g)
        s.update(q=torch.randn((off[-1], case["heads"], case["dim"]), generator=g, device=DEV, dtype=torch.float32).to(dt),
                 table=table.to(DEV), lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
                 off=torch.tensor(off, dtype=torch.int32, device=DEV), host_lens=lens, host_off=off)
        if own:
            s["handle"] = _wrap(s["res"], s["cache"])
        return s
    if op == "beams":
        n, w, v = case["batch"], case["beams"], case["vocab"]
        x = torch.randn((n, w, v), generator=g, device=DEV, dtype=torch.float32) * 3.0
        s.update(logits=x.to(DTYPE[case["dtype"]]), scores=-torch.rand((n, w), generator=g, device=DEV) * 8.0,
                 finished=(torch.rand((n, w), generator=g, device=DEV) < 0.2) if case["finished"] else None)
        return s
    n, w, layers = case["batch"], case["beams"], case["layers"]
    s["parents"] = torch.randint(0, w, (n, w), generator=g, device=DEV, dtype=torch.int32)
    if op == "reorder":
        s["states"] = [torch.randn((n, w, case["width"] + 3 * i), generator=g, device=DEV, dtype=torch.float32).to(
            torch.float32 if i % 2 else torch.bfloat16) for i in range(layers)]
        return s
    rows, block = n * w, case["block"]
    lens = _context_lengths(dict(batch=n, longest=case["longest"]), seed)
    width = _blocks(max(lens) + 1, block)
    c = torch.Generator()
    c.manual_seed(seed)
    # a prompt's full blocks are shared by its beams; each beam has its own last block and a spare one
    need = [l // block for l in lens]
    total = sum(need) + 2 * rows
    pages = torch.randperm(total, generator=c).to(torch.int32)
    table = torch.full((n, w, width), -1, dtype=torch.int32)
    at = 0
    for i, m in enumerate(need):
        table[i, :, :m] = pages[at:at + m]
        at += m
        for j in range(w):
            table[i, j, m] = pages[at + j] if lens[i] % block else -1
        at += w
    s.update(table=table.reshape(rows, width).to(DEV), spare=pages[at:at + rows].clone().to(DEV),
             lens=torch.tensor(lens, dtype=torch.int32).repeat_interleave(w).to(DEV))
    s["caches"] = [_cache(total, case["heads"], block, case["dim"], case["code"], g) for _ in range(layers)]
    if own:
        s["handles"] = [_wrap(s["res"], c) for c in s["caches"]]
    return s


# ------------------------------------------------------------------------------------------------ the plain forms
def _plain_plan(s):
    block = s["case"]["block"]
    table, ring = s["table"], s["ring"]
    total, (n, width) = ring.numel(), table.shape
    old, new = s["old"].long(), s["new"].long()
    head, count = s["state"][0], s["state"][1]
    have, want = (old + block - 1) // block, (new + block - 1) // block
    ok = (old >= 0) & (new >= 0) & (old <= width * block) & (new <= width * block)
    take = torch.where(ok, (want - have).clamp(min=0), 0)
    tokens = torch.where(ok, (new - old).clamp(min=0), 0)
    ct, cn = take.cumsum(0), tokens.cumsum(0)
    granted = ok & ((tokens == 0) | ((ct <= count) & (cn <= s["room"])))
    take, tokens = torch.where(granted, take, 0), torch.where(granted, tokens, 0)
    give = torch.where(granted, (have - want).clamp(min=0), 0)
    # blocks taken from the ring's front, in request order
    col = torch.arange(width, device=table.device)
    fresh = (col >= have[:, None]) & (col < (have + take)[:, None])
    src = (head + (take.cumsum(0) - take)[:, None] + col - have[:, None]) % total
    gone = (col >= want[:, None]) & (col < (want + give)[:, None])
    dst = (head + count + (give.cumsum(0) - give)[:, None] + col - want[:, None]) % total
    filled = torch.where(fresh, ring[src], table)
    ring = ring.scatter(0, dst[gone], table[gone])
    off = torch.cat([torch.zeros(1, dtype=torch.int64, device=table.device), tokens.cumsum(0)])
    t = torch.arange(s["room"], device=table.device)
    b = (torch.searchsorted(off, t, right=True) - 1).clamp(max=n - 1)
    pos = torch.where(t < off[-1], old[b] + t - off[b], 0)
    slot = filled[b, pos // block].long() * block + pos % block
    state = torch.stack([(head + take.sum()) % total, count - take.sum() + give.sum()])
    return dict(table=filled, ring=ring, lengths=torch.where(granted, new, old).int(), state=state, offsets=off.int(),
                slots=torch.where(t < off[-1], slot, -1).int(), granted=granted.int())


def _exponent(amax, code):
    """smallest e with amax <= QMAX 2^e"""
    f, x = torch.frexp(amax)
    top = 9 if code == "e4m3" else 7
    return (x - top + (f > QMAX[code] / 2.0 ** top).int()).clamp(min=-126)


def _requantise(values, inverse, code):
    x = values * inverse
    return x.to(torch.float8_e4m3fn) if code == "e4m3" else x.round().to(torch.int8)


def _take(codes, at):
    """codes[at] by way of their bytes"""
    return codes.view(torch.uint8)[at].view(codes.dtype)


def _plain_add_one(codes, scales, x, page, offset, touched, code):
    """codes [blocks, heads, block, dim] with their scales; x [tokens, heads, dim] stored at (page, offset)"""
    blocks, heads, block, _ = codes.shape
    x = x.float()
    amax = torch.zeros((blocks, heads), device=x.device).index_reduce_(0, page, x.abs().amax(-1), "amax", include_self=True)
    written = torch.zeros((blocks, block), dtype=torch.bool, device=x.device)
    written[page, offset] = True
    fresh, hit = written[:, 0], written.any(1)
    scale = torch.where(amax > 0, torch.exp2(_exponent(amax, code).float()), torch.zeros_like(amax))
    before = torch.where(fresh[:, None], torch.zeros_like(scales), scales)
    after = torch.where(hit[:, None], torch.maximum(before, scale), scales)
    ratio = torch.where(after > 0, before / after, torch.zeros_like(after))
    p = touched.long()
    raw = codes.view(torch.uint8)
    raw[p] = _requantise(_take(codes, p).float(), ratio[p][:, :, None, None], code).view(torch.uint8)
    inverse = torch.where(after > 0, 1.0 / after, torch.zeros_like(after))
    raw[page, :, offset] = _requantise(x, inverse[page][:, :, None], code).view(torch.uint8)
    scales.copy_(after)
    return _take(codes, p).float() * after[p][:, :, None, None]


def _plain_add(s):
    case, c = s["case"], s["cache"]
    slots = s["slots"].long()
    page, offset = slots // case["block"], slots % case["block"]
    k = _plain_add_one(c["k"], c["ks"], s["key"], page, offset, s["touched"], case["code"])
    v = _plain_add_one(c["v"].transpose(2, 3), c["vs"], s["value"], page, offset, s["touched"], case["code"])
    dt = DTYPE[case["dtype"]]
    return dict(k=k.to(dt), v=v.to(dt), ks=c["ks"], vs=c["vs"])


def _values(c, pages, dtype):
    """keys and values [kv heads, tokens, dim] of the blocks"""
    k = _take(c["k"], pages).to(dtype) * c["ks"][pages].to(dtype)[:, :, None, None]
    v = _take(c["v"], pages).to(dtype) * c["vs"][pages].to(dtype)[:, :, None, None]
    n, h, b, d = k.shape
    return k.permute(1, 0, 2, 3).reshape(h, n * b, d), v.permute(1, 0, 3, 2).reshape(h, n * b, d)


def _plain_attend(s):
    case, c, q = s["case"], s["cache"], s["q"]
    hq, hk, d, block = case["heads"], case["kv_heads"], case["dim"], case["block"]
    out = torch.empty_like(q)
    for i, length in enumerate(s["host_lens"]):
        a, b = s["host_off"][i], s["host_off"][i + 1]
        k, v = _values(c, s["table"][i, :_blocks(length, block)].long(), torch.float32)
        k, v = k[:, :length], v[:, :length]
        x = q[a:b].float().permute(1, 0, 2).reshape(hk, (hq // hk) * (b - a), d)
        p = torch.matmul(x, k.transpose(1, 2).contiguous()) * (1.0 / math.sqrt(d))
        if b - a > 1:
            row = torch.arange(b - a, device=q.device).repeat(hq // hk)
            p.masked_fill_(torch.arange(length, device=q.device)[None] > (length - (b - a) + row)[:, None], float("-inf"))
        p = torch.exp(p - p.amax(-1, keepdim=True))
        o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
        out[a:b] = o.reshape(hq, b - a, d).permute(1, 0, 2).to(q.dtype)
    return out


def _plain_beams(s):
    # in 64 bits: which candidate comes first hangs on differences that 32 bits lose
    x = s["logits"].double()
    n, w, v = x.shape
    m = x.amax(-1, keepdim=True)
    value = s["scores"].double()[:, :, None] + (x - (m + torch.exp(x - m).sum(-1, keepdim=True).log()))
    if s["finished"] is not None:
        rest = torch.full_like(value, float("-inf"))
        rest[:, :, 0] = s["scores"].double()
        value = torch.where(s["finished"][:, :, None], rest, value)
    value = value.reshape(n, w * v)
    at = torch.arange(w * v, device=x.device)
    best, where = [], []
    for _ in range(s["case"]["keep"]):
        top = value.amax(1, keepdim=True)
        i = torch.where(value == top, at, w * v).amin(1, keepdim=True)
        best.append(top)
        where.append(i)
        value.scatter_(1, i, float("-inf"))
    best, where = torch.cat(best, 1), torch.cat(where, 1)
    none = best == float("-inf")
    return (best.float(), torch.where(none, -1, where // v).int(), torch.where(none, -1, where % v).int())


def _plain_reorder(s):
    p = s["parents"].long()
    row = torch.arange(p.shape[0], device=p.device)[:, None]
    return [x[row, p] for x in s["states"]]


def _plain_fork(s):
    case = s["case"]
    n, w, block = case["batch"], case["beams"], case["block"]
    parent = (torch.arange(n, device=DEV)[:, None] * w + s["parents"].long()).reshape(-1)
    table, spare, lens = s["table"][parent], s["spare"], s["lens"][parent]
    tail, last = (lens % block) != 0, (lens // block).long()
    row = torch.arange(n * w, device=DEV)
    last = last.clamp(max=table.shape[1] - 1)
    src = table[row, last].long()
    for c in s["caches"]:
        for name in ("k", "v", "ks", "vs"):
            t = c[name]
            raw = t if name in ("ks", "vs") else t.view(torch.uint8)
            keep = tail.reshape((-1,) + (1,) * (raw.dim() - 1))
            raw[spare.long()] = torch.where(keep, raw[src.clamp(min=0)], raw[spare.long()])
    table[row, last] = torch.where(tail, spare, table[row, last])
    left = torch.where((s["lens"] % block) != 0, s["table"][row, (s["lens"] // block).long().clamp(max=table.shape[1] - 1)], -1)
    return table, lens, torch.where(tail, left, spare), [_plain_blocks(c, spare) for c in s["caches"]]


def _plain_blocks(c, pages):
    p = pages.long()
    return (_widen(c["k"], c["ks"], p), _widen(c["v"], c["vs"], p).transpose(2, 3).contiguous())


def _widen(codes, scales, p):
    return (_take(codes, p).float() * scales[p][:, :, None, None]).to(torch.bfloat16)


# ------------------------------------------------------------------------------------------------ a pass
def run(state):
    s, case = state, state["case"]
    op = case["op"]
    if not own:
        return dict(plan=_plain_plan, add=_plain_add, attend=_plain_attend, beams=_plain_beams, reorder=_plain_reorder,
                    fork=_plain_fork)[op](s)
    from faiss_amd import decoding
    if op == "plan":
        p = decoding.plan_blocks(s["res"], s["table"], s["old"], s["new"], s["ring"], s["state"], case["block"], s["room"])
        return dict(table=s["table"], ring=s["ring"], lengths=p.lengths, state=p.free_state, offsets=p.query_offsets,
                    slots=p.slots, granted=p.granted)
    if op == "add":
        h = s["handle"]
        h.add(s["key"], s["value"], s["slots"])
        k, v = h.reconstruct(s["touched"], DTYPE[case["dtype"]])
        return dict(k=k, v=v, ks=h.k_scales, vs=h.v_scales)
    if op == "attend":
        if case["queries"] == 1:
            return s["handle"].attend(s["q"], s["table"], s["lens"])
        return s["handle"].attend(s["q"], s["table"], s["lens"], query_offsets=s["off"], max_queries=case["queries"])
    if op == "beams":
        return decoding.beam_select(s["res"], s["logits"], s["scores"], case["keep"], finished=s["finished"])
    if op == "reorder":
        return decoding.reorder_beams(s["res"], s["states"], s["parents"])
    table, lens, spare = decoding.fork_blocks(s["res"], s["handles"], s["table"], s["lens"], s["spare"], s["parents"])
    return table, lens, spare, [h.reconstruct(s["spare"], torch.bfloat16) for h in s["handles"]]


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "plan":
        n, block = case["batch"], case["block"]
        tokens = n if case["grow"] == 1 else n * min(case["grow"], case["longest"]) // 2
        return dict(bytes=n * 20 + (n * min(case["grow"], case["longest"]) + 3) * 4 + _blocks(tokens, block) * 8 + 32, flops=0)
    if op == "add":
        n, h, d = case["tokens"], case["heads"], case["dim"]
        blocks = -(-n // case["each"]) * _blocks(min(case["each"], n) + case["block"] // 2, case["block"])
        return dict(bytes=2 * h * (n * d * 3 + blocks * (4 + case["block"] * d * 3)) + 4 * n, flops=2 * n * h * d * 4)
    if op == "attend":
        lens, qn = _context_lengths(case, 0), _query_counts(case)
        d, hq, hk = case["dim"], case["heads"], case["kv_heads"]
        seen = sum(m * l - m * (m - 1) // 2 for l, m in zip(lens, qn))
        return dict(bytes=sum(lens) * hk * d * 2 + sum(_blocks(l, case["block"]) for l in lens) * (hk * 8 + 4) + sum(qn) * hq * d * 4,
                    flops=4 * seen * hq * d)
    if op == "beams":
        size = {"fp32": 4, "bf16": 2, "fp16": 2}[case["dtype"]]
        rows = case["batch"] * case["beams"]
        return dict(bytes=rows * case["vocab"] * size + rows * 4 + case["batch"] * case["keep"] * 12, flops=rows * case["vocab"] * 4)
    rows = case["batch"] * case["beams"]
    if op == "reorder":
        each = [(case["width"] + 3 * i) * (4 if i % 2 else 2) for i in range(case["layers"])]
        return dict(bytes=2 * rows * sum(each) + rows * 4, flops=0)
    page = 2 * case["heads"] * (case["block"] * case["dim"] + 4)
    width = _blocks(case["longest"] + 1, case["block"])
    # the copied blocks, and the values that are read back from them
    return dict(bytes=rows * (case["layers"] * page * 5 + width * 8 + 24), flops=0)


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    op = case["op"]
    if op in ("plan", "reorder", "fork"):
        return None  # integers and copies
    s = prepare(case, seed)
    if op == "beams":
        return _exact_beams(s)
    if op == "add":
        return _exact_add(s)
    return _exact_attend(s)


def _exact_beams(s):
    x = s["logits"].double()
    n, w, v = x.shape
    logp = x - torch.logsumexp(x, -1, keepdim=True) + s["scores"].double()[:, :, None]
    if s["finished"] is not None:
        f = s["finished"]
        logp[f] = float("-inf")
        first = logp[:, :, 0]
        first[f] = s["scores"].double()[f]
    best = torch.topk(logp.reshape(n, w * v), min(s["case"]["keep"], w * v), dim=1).values
    return best, None, None


def _exact_add(s):
    """block by block on the host: the powers of two and the nearest codes by their definition"""
    case, c = s["case"], s["cache"]
    block, code = case["block"], case["code"]
    if case["tokens"] > 4096:
        return None
    slots = s["slots"].cpu().tolist()
    by = {}
    for t, x in enumerate(slots):
        by.setdefault(x // block, []).append((x % block, t))
    out = []
    for name, scales, x in (("k", "ks", s["key"]), ("v", "vs", s["value"])):
        codes = c[name] if name == "k" else c[name].transpose(2, 3)
        val, sc = codes.float().double().cpu(), c[scales].double().cpu()
        x = x.double().cpu()
        for page, at in by.items():
            off = torch.tensor([o for o, _ in at])
            new = x[torch.tensor([t for _, t in at])]  # [tokens, heads, dim]
            amax = new.abs().amax((0, 2))
            step = torch.where(amax > 0, torch.exp2(torch.ceil(torch.log2(amax / QMAX[code])).clamp(min=-126)), amax)
            kept = torch.zeros_like(sc[page]) if 0 in off.tolist() else sc[page]
            grown = torch.maximum(kept, step)
            safe = torch.where(grown > 0, grown, torch.ones_like(grown))[:, None, None]
            val[page] = _nearest(val[page] * kept[:, None, None] / safe, code)
            val[page][:, off] = _nearest(new.transpose(0, 1) / safe, code)
            sc[page] = grown
        p = s["touched"].long().cpu()
        out.append(((val[p] * sc[p][:, :, None, None]).to(DEV), sc.to(DEV)))
    return dict(k=out[0][0], v=out[1][0], ks=out[0][1], vs=out[1][1])


def _nearest(x, code):
    if code == "int8":
        return torch.round(x)
    _, e = torch.frexp(x)
    step = torch.exp2((e.double() - 1).clamp(min=-6) - 3)  # spacing of the codes around x
    return torch.round(x / step) * step


def _exact_attend(s):
    case, c = s["case"], s["cache"]
    hq, hk, d, block = case["heads"], case["kv_heads"], case["dim"], case["block"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    for i, length in enumerate(s["host_lens"]):
        a, b = s["host_off"][i], s["host_off"][i + 1]
        pages = s["table"][i, :_blocks(length, block)].long()
        pos = torch.arange(length, device=DEV)
        for h in range(hk):
            k = (_take(c["k"], (pages, h)).double() * c["ks"][pages, h].double()[:, None, None]).reshape(-1, d)[:length]
            v = (_take(c["v"], (pages, h)).double() * c["vs"][pages, h].double()[:, None, None]).transpose(1, 2).reshape(-1, d)[:length]
            for r in range(h * (hq // hk), (h + 1) * (hq // hk)):
                z = s["q"][a:b, r].double() @ k.T / math.sqrt(d)
                z[pos[None] > (length - (b - a) + torch.arange(b - a, device=DEV))[:, None]] = float("-inf")
                out[a:b, r] = torch.softmax(z, -1) @ v
    return out
