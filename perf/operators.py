"""Cases and plain forms of the paged 4-bit KV cache and of token scoring.

Operators: ``append`` (quantise keys / values into cache pages, read back what they hold), ``attend`` (attention over the
pages), ``pages`` (forking rows with copy on write; evicting rows, compacting the pool and admitting new rows) and ``score``
(log probabilities of given tokens, entropy and the top alternatives).

A page holds 64 tokens.  The block of one (layer, page, KV head) is one run of bytes:
key codes [64, hd/2], value codes [64, hd/2], key scales [64, hd/32] bfloat16, value scales [64, hd/32] bfloat16.
Channel 2j of a token is the low nibble of byte j, channel 2j + 1 the high one; a value is (nibble - 8) * scale of its 32
channels; the scale is amax / 7 rounded to 4 significant bits.
"""
import math

import torch

own = False

PAGE = 64
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one token of one chat row early in its answer: latency alone
        dict(name="attend one row", op="attend", rows=1, s=1, hq=32, hkv=8, hd=128, ctx=129, window=0, dtype="bf16"),
        # a decode step of the default serving batch (16 rows, up to 512 + 256 tokens), ragged
        dict(name="attend decode batch", op="attend", rows=16, s=1, hq=32, hkv=8, hd=128, ctx=768, window=0, dtype="bf16"),
        # long documents: 32 rows of up to 16384 tokens, ragged
        dict(name="attend long rows", op="attend", rows=32, s=1, hq=32, hkv=8, hd=128, ctx=16384, window=0, dtype="bf16"),
        # float32 with one query head per KV head, an odd context
        dict(name="attend f32 heads", op="attend", rows=3, s=1, hq=8, hkv=8, hd=64, ctx=2001, window=0, dtype="f32"),
        # a prompt chunk of 512 tokens over what the rows hold already
        dict(name="attend prompt chunk", op="attend", rows=2, s=512, hq=32, hkv=8, hd=128, ctx=4096, window=0, dtype="bf16"),
        # four drafted tokens a row checked at once, sliding window, wide heads
        dict(name="attend draft window", op="attend", rows=8, s=4, hq=16, hkv=8, hd=256, ctx=8192, window=1024, dtype="bf16"),
        # the keys and values of one decode step
        dict(name="append one token", op="append", rows=64, s=1, hkv=8, hd=128, ctx=700, dtype="bf16"),
        # the keys and values of a ragged batch of prompts
        dict(name="append prompts", op="append", rows=16, s=512, hkv=8, hd=128, ctx=512, dtype="bf16"),
        # four beams a prompt step on from their first beam: shared last pages are copied before they are written
        dict(name="pages fork beams", op="pages", what="fork", rows=16, beam=4, layers=4, hkv=8, hd=128, ctx=650),
        # half of the rows end, the pool is compacted, new rows take their places
        dict(name="pages evict compact", op="pages", what="evict", rows=32, beam=1, layers=8, hkv=8, hd=128, ctx=2000),
        # seven rows of one step scored, float32, a small vocabulary
        dict(name="score step f32", op="score", rows=7, vocab=50304, top=5, dtype="f32"),
        # the tokens of two prompts of 512 scored
        dict(name="score prompts", op="score", rows=1024, vocab=128256, top=20, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "append", "pages", "score"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "score":
        vocab = rng.choice([1003, 32000, 50304, 128256, 262144, _log_int(rng, 300, 200000)])
        rows = _log_int(rng, 1, 1024)
        while rows * vocab * (2 if dtype == "bf16" else 4) > 1024 * 128256 * 2:
            rows = max(1, rows // 2)
        return dict(op=op, rows=rows, vocab=vocab, top=rng.randint(0, 32), dtype=dtype)
    hq, hkv, hd = rng.choice([(32, 8, 128), (8, 8, 64), (16, 8, 256), (64, 8, 128), (6, 3, 64), (12, 2, 128), (5, 1, 256)])
    rows = _log_int(rng, 1, 64)
    if op == "append":
        s = rng.choice([1, 1, _log_int(rng, 2, 2048)])
        while rows * s * hkv * hd > 16 * 512 * 8 * 128:
            s = max(1, s // 2)
            rows = rows if s > 1 else min(rows, 64)
        return dict(op=op, rows=rows, s=s, hkv=hkv, hd=hd, ctx=s + rng.randint(0, 700), dtype=dtype)
    if op == "pages":
        what = rng.choice(["fork", "evict"])
        beam = rng.choice([2, 3, 4, 8]) if what == "fork" else 1
        rows = max(2, min(rows, 32)) * 1
        rows = max(beam, rows // beam * beam) if what == "fork" else rows // 2 * 2
        ctx, layers = _log_int(rng, 3, 2000), rng.randint(1, 8)
        while rows * ctx * layers * hkv * hd > 32 * 2000 * 8 * 8 * 128:
            ctx = max(3, ctx // 2)
        return dict(op=op, what=what, rows=rows, beam=beam, layers=layers, hkv=hkv, hd=hd, ctx=ctx)
    s = rng.choice([1, 1, 1, rng.randint(2, 16), _log_int(rng, 17, 512)])
    ctx = max(s, _log_int(rng, 1, 16384))
    window = rng.choice([0, 0, 0, _log_int(rng, 1, 4096)])
    while (rows * ctx * hkv * hd > 32 * 16384 * 8 * 128 // (4 if dtype == "f32" else 1)
           or rows * s * ctx * hq * hd > 2 * 512 * 4096 * 32 * 128 // (4 if dtype == "f32" else 1)):
        rows, ctx = (rows // 2, ctx) if rows > 1 else (1, ctx // 2)
        s = min(s, ctx)
    return dict(op=op, rows=rows, s=s, hq=hq, hkv=hkv, hd=hd, ctx=ctx, window=window, dtype=dtype)


def _block(hd):
    return PAGE * hd + PAGE * (hd // 32) * 4


def _lens(case):
    """Row lengths: the first row is the longest, the others between half of it and all of it."""
    n, ctx, s = case["rows"], case["ctx"], case.get("s", 1)
    return [ctx - (r * 2654435761 % 1000) * (ctx - max(s, (ctx + 1) // 2)) // 1000 for r in range(n)]


def _counts(case):
    """Tokens of the current call a row has: ragged where it has several; in a larger batch the last row is idle."""
    n, s = case["rows"], case["s"]
    c = [s if r % 3 == 0 else max(1, s - (r * 37) % s) for r in range(n)]
    if n >= 8:
        c[-1] = 0
    return c


def work(case):
    op, rows = case["op"], case["rows"]
    if op == "score":
        nv = rows * case["vocab"]
        return {"bytes": nv * (2 if case["dtype"] == "bf16" else 4) + rows * (16 + 8 * case["top"]), "flops": 6 * nv}
    hkv, hd = case["hkv"], case["hd"]
    token = 2 * hkv * (hd // 2 + hd // 16)
    if op == "append":
        n, size = sum(_counts(case)), 2 if case["dtype"] == "bf16" else 4
        whole = rows * case["s"]
        return {"bytes": n * 2 * hkv * hd * size + 2 * n * token + whole * 2 * hkv * hd * size, "flops": 12 * n * 2 * hkv * hd}
    if op == "pages":
        page = case["layers"] * hkv * _block(hd)
        per_row = [-(-x // PAGE) for x in _page_lens(case)]
        if case["what"] == "fork":
            copied = (rows - rows // case["beam"]) if _page_lens(case)[0] % PAGE else 0
        else:
            copied = sum(per_row) // 2
        return {"bytes": 2 * copied * page + 16 * sum(per_row), "flops": 0}
    size = 2 if case["dtype"] == "bf16" else 4
    keys = read = 0
    for n, c in zip(_lens(case), _counts(case)):
        if c == 0:
            continue
        w = case["window"] or n
        keys += sum(min(n - c + i + 1, w) for i in range(c))
        read += n - max(0, n - c + 1 - w)
    whole = rows * case["s"]
    return {"bytes": read * token + 2 * whole * case["hq"] * hd * size, "flops": 4 * keys * case["hq"] * hd}


# ---------------------------------------------------------------------------------------------- inputs
def _page_lens(case):
    """Of the page cases: the same length in every row of a group of beams, never a whole number of pages unless ctx is one."""
    return [case["ctx"]] * case["rows"]


def _pool(gen, layers, pages, hkv, hd):
    """Pages of random finite content: codes of -7..7 and scales of 4 significant bits between 1/32 and 1/2."""
    shape = (layers, pages, hkv)
    nib = torch.randint(1, 16, shape + (2, PAGE * hd), generator=gen, device=DEV, dtype=torch.uint8)
    nib = (nib[..., 0, :] | (nib[..., 1, :] << 4)).to(torch.uint8)
    n = 2 * PAGE * (hd // 32)
    scale = (1 + torch.randint(0, 8, shape + (n,), generator=gen, device=DEV) / 8) * torch.exp2(
        torch.randint(-5, -1, shape + (n,), generator=gen, device=DEV).float())
    return torch.cat([nib, scale.to(torch.bfloat16).view(torch.uint8)], dim=-1).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    op, rows = case["op"], case["rows"]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    if op == "score":
        x = torch.randn(rows, case["vocab"], generator=gen, device=DEV) * 3
        x[:, ::17] = x[:, ::17] - 8
        if rows > 2:  # a row that a filter has been over
            x[1, 5::2] = float("-inf")
        ids = torch.randint(0, case["vocab"], (rows,), generator=gen, device=DEV, dtype=torch.int32)
        return dict(case=case, logits=x.to(DTYPES[case["dtype"]]), ids=ids)
    hkv, hd = case["hkv"], case["hd"]
    lens = _page_lens(case) if op == "pages" else _lens(case)
    used = [-(-n // PAGE) for n in lens]
    layers = case.get("layers", 1)
    width = max(used) + 2
    st = dict(case=case, head_dim=hd)
    if op == "pages":
        # page j of row r, as rows that grow together take them; spare pages behind
        total = sum(used) + 2 * rows
        table = [[j * rows + r if j < used[r] else -1 for j in range(width)] for r in range(rows)]
        st["table"] = i32(table)
        group = torch.arange(rows, device=DEV, dtype=torch.int32)
        st["parents"] = group // case["beam"] * case["beam"]
        st["half"] = [(group % 2 == 0), (group % 2 == 1)]
        st["admit"] = [x.to(torch.int32) * case["ctx"] for x in st["half"]]
        st["turn"] = 0
    else:
        total = sum(used) + 3
        order = torch.randperm(total, generator=gen, device=DEV).to(torch.int32)
        at = torch.cumsum(i32([0] + used), 0)[:-1, None] + torch.arange(width, device=DEV)[None]
        there = torch.arange(width, device=DEV)[None] < i32(used)[:, None]
        st["table"] = torch.where(there, order[at.clamp(max=total - 1)], -1).to(torch.int32).contiguous()
    st["pages"] = _pool(gen, layers, total, hkv, hd)
    st["lengths"] = i32(lens)
    st["counts"] = i32(_counts(case)) if op != "pages" else i32([0] * rows)
    refs = torch.zeros(total + 1, dtype=torch.int32, device=DEV)
    refs.index_add_(0, torch.where(st["table"] < 0, total, st["table"]).reshape(-1).long(),
                    torch.ones(rows * width, dtype=torch.int32, device=DEV))
    st["refs"] = refs[:total].contiguous()
    if op == "attend":
        st["q"] = (torch.randn(rows, case["s"], case["hq"], hd, generator=gen, device=DEV) * 1.5).to(DTYPES[case["dtype"]])
    if op == "append":
        shape = (rows, case["s"], hkv, hd)
        for name, size in (("k", 2.0), ("v", 0.3)):
            x = torch.randn(shape, generator=gen, device=DEV) * size
            x[..., 3] *= 8  # a channel that stands out
            st[name] = x.to(DTYPES[case["dtype"]])
        st["start"] = (st["lengths"] - st["counts"]).to(torch.int32)
    return st


# ---------------------------------------------------------------------------------------------- plain forms
def _codes(blk, hd, which):
    """(nibble - 8) * scale in 32 bits of gathered blocks [..., block] -> [..., 64, hd]."""
    lead, half, per = blk.shape[:-1], PAGE * hd // 2, PAGE * (hd // 32) * 2
    b = blk[..., which * half:(which + 1) * half].reshape(lead + (PAGE, hd // 2))
    n = torch.stack([b & 15, b >> 4], dim=-1).reshape(lead + (PAGE, hd // 32, 32)).to(torch.float32) - 8
    at = 2 * half + which * per
    s = blk[..., at:at + per].contiguous().view(torch.bfloat16).reshape(lead + (PAGE, hd // 32, 1)).to(torch.float32)
    return (n * s).reshape(lead + (PAGE, hd))


def _rows_of(pages, table, hd, which):
    """The rows' keys (0) or values (1): [R, Hkv, T, hd] of a layer's pages [N, Hkv, block]."""
    x = _codes(pages[table.clamp(min=0).long()], hd, which)          # [R, P, Hkv, 64, hd]
    R, P, H = x.shape[:3]
    return x.permute(0, 2, 1, 3, 4).reshape(R, H, P * PAGE, hd)


def _plain_attend(st):
    case, hd, q = st["case"], st["head_dim"], st["q"]
    R, S, Hq, _ = q.shape
    k, v = (_rows_of(st["pages"][0], st["table"], hd, w) for w in (0, 1))
    Hkv, T = k.shape[1], k.shape[2]
    G = Hq // Hkv
    qq = q.to(torch.float32).reshape(R, S, Hkv, G, hd).permute(0, 2, 3, 1, 4).reshape(R, Hkv, G * S, hd)
    sc = torch.matmul(qq, k.transpose(-1, -2)) * (hd ** -0.5)
    i = torch.arange(S, device=q.device, dtype=torch.int32)[None]
    pos = st["lengths"][:, None] - st["counts"][:, None] + i                       # [R, S]
    key = torch.arange(T, device=q.device, dtype=torch.int32)[None, None]
    see = (key <= pos[..., None]) & (i < st["counts"][:, None])[..., None]
    if case["window"]:
        see = see & (key > pos[..., None] - case["window"])
    see = see[:, None, None].expand(R, 1, G, S, T).reshape(R, 1, G * S, T)
    sc = sc.masked_fill(~see, float("-inf"))
    m = sc.amax(-1, keepdim=True)
    e = torch.exp(sc - torch.where(torch.isfinite(m), m, 0.0))
    p = e / e.sum(-1, keepdim=True).clamp(min=1e-30)
    o = torch.matmul(p, v).reshape(R, Hkv, G, S, hd).permute(0, 3, 1, 2, 4).reshape(R, S, Hq, hd)
    return o.to(q.dtype)


def _quantise(x):
    """nibbles and scales (float32, 4 significant bits) of [..., hd]."""
    g = x.to(torch.float32).reshape(x.shape[:-1] + (x.shape[-1] // 32, 32))
    top = g.abs().amax(-1, keepdim=True)
    bits = torch.div(top, torch.full_like(top, 7)).view(torch.int32)  # by a tensor: a true division, which ties need
    bits = (bits + 0x7FFFF + ((bits >> 20) & 1)) & ~0xFFFFF
    s = bits.view(torch.float32)
    n = torch.where(s > 0, torch.round(g / torch.where(s > 0, s, 1.0)).clamp(-7, 7), 0.0) + 8
    return n.to(torch.uint8).reshape(x.shape), s[..., 0]


def _plain_append(st):
    hd, pages, table = st["head_dim"], st["pages"][0], st["table"]
    R, S, H, _ = st["k"].shape
    half = PAGE * hd // 2
    per = PAGE * (hd // 32) * 2
    i = torch.arange(S, device=pages.device)[None]
    pos = st["start"][:, None].long() + i
    ok = i < st["counts"][:, None]
    page = torch.gather(table, 1, torch.where(ok, pos // PAGE, 0)).long()
    page = torch.where(ok, page, _lowest_free(st["refs"])[0].long())  # what is not there goes to a free page, unchanged
    head, slot = torch.arange(H, device=pages.device)[None, None], (pos % PAGE)[..., None]
    base = (page[..., None] * H + head) * pages.shape[2]                            # [R, S, H]
    flat = pages.view(-1)
    for which, x in ((0, st["k"]), (1, st["v"])):
        n, s = _quantise(x)
        by = n[..., 0::2] | (n[..., 1::2] << 4)
        at = base + which * half + slot * (hd // 2)
        idx = at[..., None] + torch.arange(hd // 2, device=pages.device)
        old = flat[idx]
        flat[idx] = torch.where(ok[..., None, None], by, old)
        sb = s.to(torch.bfloat16).view(torch.uint8)
        at = base + 2 * half + which * per + slot * (hd // 16)
        idx = at[..., None] + torch.arange(hd // 16, device=pages.device)
        old = flat[idx]
        flat[idx] = torch.where(ok[..., None, None], sb, old)
    at = torch.where(ok, pos, 0)[:, None, :, None].expand(R, H, S, hd)
    live = ok[:, :, None, None]
    got = [torch.gather(_rows_of(pages, table, hd, w), 2, at).permute(0, 2, 1, 3) for w in (0, 1)]
    return [torch.where(live, x, 0.0).to(st["k"].dtype) for x in got]


def _lowest_free(refs):
    """Page ids, the free ones first, ascending."""
    return torch.sort((refs != 0).to(torch.int32), stable=True).indices.to(torch.int32)


def _plain_recount(st):
    total = st["refs"].shape[0]
    held = torch.where(st["table"] < 0, total, st["table"]).reshape(-1).long()
    refs = torch.zeros(total + 1, dtype=torch.int32, device=held.device)
    refs.index_add_(0, held, torch.ones_like(held, dtype=torch.int32))
    st["refs"].copy_(refs[:total])


def _plain_extend(st, counts):
    """Room for counts[r] more tokens: new pages, lowest first, rows in order, a shared page that is written on copied first."""
    table, refs, lens, pages = st["table"], st["refs"], st["lengths"], st["pages"]
    R, P = table.shape
    last = torch.where(lens % PAGE != 0, lens // PAGE, 0).long()
    part = torch.gather(table, 1, last[:, None])[:, 0]
    part = torch.where((lens % PAGE != 0) & (counts > 0), part, -1)
    row = torch.arange(R, device=table.device)
    same = (part[:, None] == part[None]) & (part >= 0)[:, None]
    before = (same & (row[None] < row[:, None])).sum(1)
    copy = (part >= 0) & (refs[part.clamp(min=0).long()] - before > 1)
    new = torch.where(counts > 0, (lens + counts + PAGE - 1) // PAGE - (lens + PAGE - 1) // PAGE, 0)
    need = new + copy
    first = torch.cumsum(need, 0) - need
    free = _lowest_free(refs)
    j = torch.arange(P, device=table.device)[None]
    at = (lens[:, None] + PAGE - 1) // PAGE
    fresh = (j >= at) & (j < at + new[:, None])
    pick = (first + copy)[:, None] + (j - at)
    table.copy_(torch.where(fresh, free[pick.clamp(0, free.shape[0] - 1).long()], table))
    dst = torch.where(copy, free[first.clamp(max=free.shape[0] - 1).long()], part)
    src = torch.arange(pages.shape[1] + 1, device=table.device)
    src[torch.where(copy, dst, pages.shape[1]).long()] = part.clamp(min=0).long()
    pages.copy_(pages[:, src[:-1]])
    table.scatter_(1, last[:, None], torch.where(copy, dst, torch.gather(table, 1, last[:, None])[:, 0])[:, None])
    lens.add_(counts)
    st["counts"].copy_(counts)
    _plain_recount(st)


def _plain_shorten(st, lens):
    keep = torch.arange(st["table"].shape[1], device=lens.device)[None] < ((lens + PAGE - 1) // PAGE)[:, None]
    st["table"].copy_(torch.where(keep, st["table"], -1))
    st["lengths"].copy_(lens)
    st["counts"].zero_()
    _plain_recount(st)


def _plain_fork(st, parents):
    st["table"].copy_(st["table"][parents.long()])
    st["lengths"].copy_(st["lengths"][parents.long()])
    st["counts"].zero_()
    _plain_recount(st)


def _plain_compact(st):
    """The used pages at or above the number of used pages go to the free ones below it, both ascending."""
    refs, pages = st["refs"], st["pages"]
    total = refs.shape[0]
    ids = torch.arange(total, device=refs.device)
    n = (refs != 0).sum()
    mover, hole = (refs != 0) & (ids >= n), (refs == 0) & (ids < n)
    rank = torch.cumsum(mover, 0) - 1
    holes = torch.sort((~hole).to(torch.int32), stable=True).indices
    to = torch.where(mover, holes[rank.clamp(min=0)], ids)
    src = torch.arange(total + 1, device=refs.device)
    src[torch.where(mover, to, total)] = ids
    pages.copy_(pages[:, src[:total]])
    st["table"].copy_(torch.where(st["table"] < 0, -1, to[st["table"].clamp(min=0).long()].to(torch.int32)))
    _plain_recount(st)
    return n.to(torch.int32).reshape(1)


def _plain_score(st):
    x, top = st["logits"].to(torch.float32), st["case"]["top"]
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    z = e.sum(-1, keepdim=True)
    lz = torch.log(z)
    ent = lz[:, 0] - torch.where(e > 0, e * d, 0.0).sum(-1) / z[:, 0]
    lp = (torch.gather(d, 1, st["ids"][:, None].long()) - lz)[:, 0]
    bits = (x + 0.0).view(torch.int32).to(torch.int64)
    key = torch.where(bits < 0, -(bits & 0x7FFFFFFF) - 1, bits) * (1 << 20) + (
        (1 << 20) - 1 - torch.arange(x.shape[1], device=x.device))
    best = (1 << 20) - 1 - (torch.topk(key, top, dim=-1).values % (1 << 20))
    return [lp, ent, torch.gather(d, 1, best) - lz, best.to(torch.int32)]


# ---------------------------------------------------------------------------------------------- run
def _cache(st):
    if "cache" not in st:
        from jaxml_b200 import PagedKVCache
        st["cache"] = PagedKVCache(pages=st["pages"], table=st["table"], lengths=st["lengths"], counts=st["counts"],
                                   refs=st["refs"], head_dim=st["head_dim"])
    return st["cache"]


def _state(st, *more):
    return [st["table"], st["lengths"], st["refs"], st["pages"].view(torch.int32), *more]


def run(st):
    case = st["case"]
    op = case["op"]
    if op == "score":
        if own:
            from jaxml_b200.sampling import token_log_probs
            return list(token_log_probs(st["logits"], st["ids"], top_n=case["top"]))
        return _plain_score(st)
    if op == "attend":
        return _cache(st).attend(0, st["q"], sliding_window=case["window"] or None) if own else _plain_attend(st)
    if op == "append":
        if own:
            c = _cache(st)
            c.append(0, st["k"], st["v"])
            return list(c.read(0, st["start"], case["s"], dtype=st["k"].dtype))
        return _plain_append(st)
    if case["what"] == "fork":
        if own:
            c = _cache(st)
            c.fork(st["parents"])
            c.extend(1)
            c.rollback(1)
        else:
            _plain_fork(st, st["parents"])
            _plain_extend(st, torch.ones_like(st["lengths"]))
            _plain_shorten(st, st["lengths"] - 1)
        return _state(st)
    gone, admit = st["half"][st["turn"]], st["admit"][st["turn"]]
    st["turn"] = 1 - st["turn"]
    if own:
        c = _cache(st)
        c.free(gone)
        n = c.compact()
        c.extend(admit)
    else:
        _plain_shorten(st, torch.where(gone, 0, st["lengths"]))
        n = _plain_compact(st)
        _plain_extend(st, admit)
    return _state(st, n)


# ---------------------------------------------------------------------------------------------- exact
def _unpack64(pages, hd, which):
    """[N, Hkv, 64, hd] in 64 bits of a layer's blocks."""
    N, H = pages.shape[:2]
    codes = pages[..., which * 32 * hd:(which + 1) * 32 * hd].reshape(N, H, 64, hd // 2).to(torch.int64)
    out = torch.empty(N, H, 64, hd, dtype=torch.float64, device=pages.device)
    out[..., 0::2] = (codes % 16 - 8).double()
    out[..., 1::2] = (codes // 16 - 8).double()
    first = 64 * hd + which * 4 * hd
    scales = pages[..., first:first + 4 * hd].contiguous().view(torch.bfloat16).reshape(N, H, 64, hd // 32).double()
    return out * scales.repeat_interleave(32, dim=-1)


def _exact_attend(st):
    case, hd, q = st["case"], st["head_dim"], st["q"].double()
    R, S, Hq, _ = q.shape
    out = torch.zeros(R, S, Hq, hd, dtype=torch.float64, device=q.device)
    G = Hq // case["hkv"]
    for r, (n, c) in enumerate(zip(_lens(case), _counts(case))):
        if c == 0:
            continue
        held = st["pages"][0][st["table"][r, : -(-n // 64)].long()]
        k, v = (_unpack64(held, hd, w).transpose(0, 1).reshape(case["hkv"], -1, hd)[:, :n] for w in (0, 1))
        for h in range(Hq):
            s = q[r, :c, h] @ k[h // G].T / math.sqrt(hd)
            gap = (n - c + torch.arange(c, device=q.device))[:, None] - torch.arange(n, device=q.device)[None]
            hidden = (gap < 0) | (gap >= (case["window"] or n + 1))
            out[r, :c, h] = torch.softmax(s.masked_fill(hidden, float("-inf")), dim=-1) @ v[h // G]
    return out


def _exact_append(st):
    out = []
    live = (torch.arange(st["case"]["s"], device=DEV)[None] < st["counts"][:, None])[..., None, None]
    for name in ("k", "v"):
        x = st[name].double().unflatten(-1, (-1, 32))
        top = x.abs().amax(-1, keepdim=True)
        mant, exp = torch.frexp(torch.div(top, torch.full_like(top, 7)))
        step = torch.ldexp(torch.round(mant * 16) / 16, exp)
        n = torch.where(step > 0, torch.round(x / step.clamp(min=1e-300)), 0.0).clamp(-7, 7)
        out.append(torch.where(live, (n * step).flatten(-2), 0.0))
    return out


def _exact_score(st):
    case = st["case"]
    parts = [[], [], []]
    for x, ids in zip(st["logits"].split(64), st["ids"].split(64)):
        x = x.double()
        lp = torch.log_softmax(x, -1)
        p = lp.exp()
        parts[0].append(lp.gather(1, ids[:, None].long())[:, 0])
        parts[1].append(-torch.where(p > 0, p * lp, 0.0).sum(-1))
        parts[2].append(torch.sort(lp, dim=-1, descending=True, stable=True).values[:, :case["top"]])
    return [torch.cat(p) for p in parts] + [None]


def exact(case, seed):
    if case["op"] == "pages":
        return None  # whole numbers and moved bytes: nothing is computed
    st = prepare(case, seed)
    return {"attend": _exact_attend, "append": _exact_append, "score": _exact_score}[case["op"]](st)
