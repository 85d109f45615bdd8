"""The operators for several answers to one prompt that are timed, in their plain form and as the
library's calls.

A case is a dict of plain values. Its "op" names the operator:

  fork      kvpages.free, fork, grow, copy   answers that ended leave their pages; sequences that
                                             share a prompt's pages; pages for their next tokens
  compact   kvpages.compact, copy            the pages in use moved to the front of the cache
  shared    kvcache.attention(shared=)       attention of sequences with a common front, read once
  score     kvcache.attention(softcap=,      scores capped by a tanh or lowered with the distance,
            slopes=, first=, prefix=)        rows bound to a document, prompts seen whole
  sample    sampling.sample                  the next token of every row from given numbers

Layouts. Cache: k uint8 [pages, heads, block, d] and v uint8 [pages, heads, d, block], e4m3
codes, with float32 scales [pages, heads] that are powers of two. table int32 [sequences, pages
of each], -1: no page. refs int32 [pages]: how many entries of the table hold a page.
"""
import math
import random

import torch

own = False

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
I32 = dict(dtype=torch.int32, device="cuda")


def listed():
    heads = dict(hkv=8, d=128, block=16, dtype="bf16")
    score = dict(window=0, cap=0.0, bias=False, docs=False, prefix=False)
    return [
        # one prompt of some hundred tokens answered four times: the calls' own latency
        dict(name="fork-prompt", op="fork", parents=1, each=4, top=700, hkv=2, d=64, block=32),
        # sixteen prompts of up to 4096 tokens, sixteen answers to each: a full server starts anew
        dict(name="fork-server", op="fork", parents=16, each=16, top=4096, hkv=8, d=128, block=16),
        # a cache of which half is left in pieces after a day's answers
        dict(name="compact", op="compact", pages=4096, part=0.5, seqs=48, hkv=8, d=128, block=16),
        # a token each of eight answers to one short question, a small model in float16
        dict(name="shared-answers", op="shared", groups=1, each=8, front=1008, own=150, new=1, hq=4,
             hkv=2, d=80, block=16, dtype="f16"),
        # a token each of 64 answers over one long document
        dict(name="shared-document", op="shared", groups=1, each=64, front=32768, own=512, new=1,
             hq=32, **heads),
        # four system prompts, eight questions of up to 300 tokens to each, as they come in
        dict(name="shared-questions", op="shared", groups=4, each=8, front=4096, own=300, new=300,
             hq=16, **heads),
        # a token of each of 32 sequences, scores lowered with the distance
        dict(name="score-tokens", op="score", b=32, top=4096, new=1, hq=16, **heads,
             **{**score, "bias": True}),
        # three short prompts with capped scores in a window, whole prompts seen, float16
        dict(name="score-short", op="score", b=3, top=333, new=100, hq=4, hkv=1, d=64, block=32,
             dtype="f16", **{**score, "cap": 20.0, "window": 200, "prefix": True}),
        # a packed row of documents of up to 8192 tokens, each seen by its own rows, capped scores
        dict(name="score-documents", op="score", b=2, top=8192, new=4096, hq=16, **heads,
             **{**score, "cap": 30.0, "docs": True}),
        # one row's next token: temperature, the 50 likeliest, nine tenths of the mass
        dict(name="sample-token", op="sample", rows=1, vocab=151936, dtype="bf16", mixed=False),
        # 40 rows of a small ragged vocabulary in float32, each with its own settings
        dict(name="sample-few", op="sample", rows=40, vocab=32001, dtype="f32", mixed=True),
        # the next tokens of 256 answers, each with its own settings
        dict(name="sample-server", op="sample", rows=256, vocab=151936, dtype="bf16", mixed=True),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(("fork", "compact", "shared", "shared", "score", "score", "sample", "sample"))
    hkv, d, block = rng.choice((1, 2, 4, 8)), rng.choice((64, 80, 128)), rng.choice((16, 32, 64))
    if op == "fork":
        return dict(op=op, parents=_log(rng, 1, 16), each=_log(rng, 1, 16), top=_log(rng, 16, 4096),
                    hkv=hkv, d=d, block=block)
    if op == "compact":
        pages = _log(rng, 64, 4096)
        return dict(op=op, pages=pages, part=rng.choice((0.1, 0.3, 0.5, 0.7, 0.9)),
                    seqs=_log(rng, 1, max(1, pages // 32)), hkv=hkv, d=d, block=16)
    if op == "sample":
        dtype = rng.choice(("bf16", "f16", "f32"))
        return dict(op=op, rows=_log(rng, 1, 128 if dtype == "f32" else 256),
                    vocab=_log(rng, 100, 151936), dtype=dtype, mixed=rng.random() < 0.7)
    heads = dict(hq=hkv * rng.choice((1, 2, 4)), hkv=hkv, d=d, block=block,
                 dtype=rng.choice(("bf16", "f16")))
    if op == "shared":
        new = rng.choice((1, 1, 1, 4, 60))
        return dict(op=op, groups=rng.choice((1, 1, 2, 4)), each=_log(rng, 2, 16 if new < 60 else 8),
                    front=block * _log(rng, 4, (8192 if new < 60 else 2048) // block),
                    own=max(new, _log(rng, 1, 512)), new=new, **heads)
    few = rng.random() < 0.5
    b = _log(rng, 1, 32) if few else rng.choice((1, 2))
    return dict(op=op, b=b, top=_log(rng, 64, 4096 if few else 2048),
                new=rng.choice((1, 1, 1, 4)) if few else _log(rng, 24, 1024),
                window=rng.choice((0, 0, 500)), cap=rng.choice((0.0, 15.0, 50.0)),
                bias=rng.random() < 0.5, docs=rng.random() < 0.4, prefix=rng.random() < 0.4, **heads)


# ------------------------------------------------------------------ what a case holds


def _dice(c):
    """A generator of its own for each case's lengths: fixed by the case alone."""
    return random.Random(repr(sorted((k, v) for k, v in c.items() if k != "name")))


def _lengths(c):
    """(tokens, new rows) of each sequence of an attention case, and its groups' common tokens."""
    rng = _dice(c)
    if c["op"] == "shared":
        n = c["groups"] * c["each"]
        own = [c["own"] if i == 0 else _log(rng, 1, c["own"]) for i in range(n)]
        front = [c["front"] if g == 0 else c["block"] * _log(rng, 1, c["front"] // c["block"])
                 for g in range(c["groups"])]
        held = [front[i // c["each"]] + o for i, o in enumerate(own)]
        return held, [min(o, c["new"]) for o in own], front
    held = [c["top"] if i == 0 else _log(rng, max(1, c["top"] // 16), c["top"])
            for i in range(c["b"])]
    return held, [min(h, c["new"]) for h in held], None


def _ranges(c):
    """For every row of an attention case its position, and the first and last token it sees."""
    held, new, _ = _lengths(c)
    rng = _dice(dict(c, ranges=1))
    rows, prefixes = [], []
    for length, n in zip(held, new):
        starts = [0]
        while c.get("docs") and starts[-1] < length:
            starts.append(starts[-1] + _log(rng, max(1, length // 32), max(1, length // 2)))
        prefix = rng.randrange(length + 1) if c.get("prefix") else 0
        prefixes.append(prefix)
        at = 0
        for p in range(length - n, length):
            while at + 1 < len(starts) and starts[at + 1] <= p:
                at += 1
            first = starts[at]
            lo = max(first, p - c["window"] + 1 if c.get("window") else 0)
            rows.append((p, first, lo, max(p, prefix - 1)))
    return rows, prefixes


def _offsets(counts):
    total, at = 0, [0]
    for n in counts:
        total += n
        at.append(total)
    return at


def _cache(s, g, pages, c):
    """Codes of normal values and scales around 2^-8, as a cache holds them."""
    h, d, blk = c["hkv"], c["d"], c["block"]
    for key, shape in (("k", (pages, h, blk, d)), ("v", (pages, h, d, blk))):
        t = torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16) * 80
        s[key] = t.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    for key in ("ks", "vs"):
        e = torch.randint(-9, -6, (pages, h), generator=g, device="cuda")
        s[key] = ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _prepare_fork(c, s, g):
    """Prompts' pages anywhere in the cache, their children's rows of the table empty."""
    rng, blk = _dice(c), c["block"]
    lens = [c["top"] if i == 0 else _log(rng, max(1, c["top"] // 8), c["top"])
            for i in range(c["parents"])]
    n, each = c["parents"], c["each"]
    cap = -(-c["top"] // blk) + 1
    need = [-(-t // blk) for t in lens]
    pages = sum(need) + n * each + 3
    _cache(s, g, pages, c)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    s["refs"] = torch.zeros(pages, **I32)
    s["refs"][order[:sum(need)].long()] = 1
    s["table"] = torch.full((n * (1 + each), cap), -1, **I32)
    at = 0
    for i, m in enumerate(need):
        s["table"][i, :m] = order[at:at + m]
        at += m
    s["lens"] = torch.tensor(lens + [lens[i // each] for i in range(n * each)], **I32)
    s["parents"] = torch.tensor([i // each for i in range(n * each)], **I32)
    s["children"] = torch.tensor([n + i for i in range(n * each)], **I32)
    s["new"] = torch.tensor([0] * n + [1] * (n * each), **I32)


def _prepare_compact(c, s, g):
    """Sequences of mixed lengths, two of them with a common front, over pages anywhere."""
    rng, pages = _dice(c), c["pages"]
    used = max(1, int(pages * c["part"]))
    _cache(s, g, pages, c)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)[:used]
    cuts = sorted(rng.randrange(used + 1) for _ in range(c["seqs"] - 1))
    ends = list(zip([0] + cuts, cuts + [used]))
    cap = max(b - a for a, b in ends)
    s["table"] = torch.full((len(ends) + 1, cap), -1, **I32)
    s["refs"] = torch.zeros(pages, **I32)
    s["refs"][order.long()] = 1
    for i, (a, b) in enumerate(ends):
        s["table"][i, :b - a] = order[a:b]
    a, b = ends[0]
    half = (b - a) // 2  # forked from the first sequence
    s["table"][-1, :half] = order[a:a + half]
    s["refs"][order[a:a + half].long()] += 1


def _prepare_rows(c, s, g):
    held, new, front = _lengths(c)
    blk, dt = c["block"], DT[c["dtype"]]
    cap = -(-max(held) // blk)
    need = [-(-n // blk) for n in held]
    pages = sum(need) + 1
    _cache(s, g, pages, c)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    s["table"] = torch.full((len(held), cap), -1, **I32)
    at = 0
    for i, m in enumerate(need):
        s["table"][i, :m] = order[at:at + m]
        at += m
        if front:
            lead = i - i % c["each"]
            common = front[i // c["each"]] // blk
            s["table"][i, :common] = s["table"][lead, :common]
    s["held"], s["new"] = torch.tensor(held, **I32), new
    s["offsets"] = None if max(new) == min(new) == 1 else torch.tensor(_offsets(new), **I32)
    # scores deviate by about two: what a cap or a distance changes
    q = torch.randn((sum(new), c["hq"], c["d"]), generator=g, device="cuda") * 6
    s["q"] = q.to(dt)
    if front:
        s["shared"] = torch.tensor([n // blk for n in front], **I32)
        return
    rows, prefixes = _ranges(c)
    s["first"] = torch.tensor([r[1] for r in rows], **I32) if c["docs"] else None
    s["prefix"] = torch.tensor(prefixes, **I32) if c["prefix"] else None
    s["slopes"] = None
    if c["bias"]:
        x = torch.arange(c["hq"], device="cuda", dtype=torch.float32)
        s["slopes"] = torch.exp2(-8.0 * (x + 1) / c["hq"])


def _prepare_sample(c, s, g):
    """Logits as a model gives them, one in a hundred tokens forbidden."""
    rows, v = c["rows"], c["vocab"]
    x = torch.randn((rows, v), generator=g, device="cuda") * 2.5
    x = x.masked_fill(torch.rand((rows, v), generator=g, device="cuda") < 0.01, float("-inf"))
    s["logits"] = x.to(DT[c["dtype"]])
    s["u"] = torch.rand((rows,), generator=g, device="cuda")
    if not c["mixed"]:
        s.update(temperature=0.7, top_k=50, top_p=0.9, min_p=0.0)
        return

    def pick(values):
        at = torch.randint(0, len(values), (rows,), generator=g, device="cuda")
        return torch.tensor(values, device="cuda")[at]
    s["temperature"] = pick((0.0, 0.3, 0.7, 1.0, 1.0, 1.5))
    s["top_k"] = pick((0, 0, 1, 20, 50, 1000)).to(torch.int32)
    s["top_p"] = pick((1.0, 1.0, 0.5, 0.9, 0.95))
    s["min_p"] = pick((0.0, 0.0, 0.02, 0.1))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": case}
    {"fork": _prepare_fork, "compact": _prepare_compact, "shared": _prepare_rows,
     "score": _prepare_rows, "sample": _prepare_sample}[case["op"]](case, s, g)
    return s


# ------------------------------------------------------------------ plain forms (32 bits)


def _books(s, **more):
    return {"refs": s["refs"], "table": s["table"], "k": s["k"].view(torch.float8_e4m3fn),
            "v": s["v"].view(torch.float8_e4m3fn), "k_scale": s["ks"], "v_scale": s["vs"], **more}


def _copy_pages(s, src, dst):
    real = src >= 0
    a, b = src[real].long(), dst[real].long()
    for key in ("k", "v", "ks", "vs"):
        s[key][b] = s[key][a]


def _count(refs, entries, by):
    """refs += by for every entry that is a page."""
    p = entries[entries >= 0].long()
    refs.index_add_(0, p, torch.full_like(p, by, dtype=torch.int32))


def _plain_fork(s):
    c, refs, table = s["case"], s["refs"], s["table"]
    blk, cap = c["block"], s["table"].shape[1]
    kids, mums = s["children"].long(), s["parents"].long()
    _count(refs, table[kids], -1)
    at = torch.arange(cap, device=table.device)
    lens = s["lens"].long()
    front = table[mums].masked_fill(at >= ((lens[mums] + blk - 1) // blk)[:, None], -1)
    table[kids] = front
    _count(refs, front, 1)
    # pages for the next tokens: entries of [first, last] that are empty or have other holders
    new = s["new"].long()
    first, last = lens // blk, (lens + new - 1) // blk
    part = (at == first[:, None]) & (lens % blk > 0)[:, None]
    in_range = (at >= first[:, None]) & (at <= last[:, None]) & (new > 0)[:, None]
    holders = torch.where(table >= 0, refs[table.clamp(min=0).long()], torch.zeros_like(table))
    wants = in_range & ((holders > 1) | ((table < 0) & ~part))
    count = wants.sum(1) + torch.where(new > 0, (last + 1 - cap).clamp(min=0), torch.zeros_like(last))
    free = torch.nonzero(refs == 0)[:, 0]
    got = (torch.cumsum(torch.where(last < cap, count, torch.zeros_like(count)), 0) <= free.numel())
    got = got & (last < cap)
    wants = wants & got[:, None]
    old = torch.where(wants & part, table, torch.full_like(table, -1))
    _count(refs, table[wants], -1)
    where = torch.nonzero(wants)
    fresh = free[: where.shape[0]].to(torch.int32)
    table[where[:, 0], where[:, 1]] = fresh
    refs[fresh.long()] = 1
    src = old.amax(1)
    dst = torch.where((src >= 0)[:, None] & part, table, torch.full_like(table, -1)).amax(1)
    _copy_pages(s, src, dst)
    short = torch.where(got, torch.zeros_like(count), count).to(torch.int32)
    return _books(s, src=src, dst=dst, short=short)


def _plain_compact(s):
    refs, table = s["refs"].clone(), s["table"].clone()
    pages = refs.numel()
    inuse = refs > 0
    used = inuse.sum()
    at = torch.arange(pages, device=refs.device)
    a = torch.nonzero(inuse & (at >= used))[:, 0]
    b = torch.nonzero(~inuse & (at < used))[:, 0]
    to = at.to(torch.int32)
    to[a] = b.to(torch.int32)
    table = torch.where(table >= 0, to[table.clamp(min=0).long()], table)
    refs[b] = refs[a]
    refs[a] = 0
    src = torch.full((pages // 2,), -1, **I32)
    dst = src.clone()
    src[: a.numel()] = a.to(torch.int32)
    dst[: a.numel()] = b.to(torch.int32)
    _copy_pages(s, src, dst)
    return {**_books(s, src=src, dst=dst, used=used.to(torch.int32)[None]), "refs": refs, "table": table}


def _decoded(s, b, length):
    """Keys and values [heads, length, d] of a sequence in float32."""
    blk = s["case"]["block"]
    p = s["table"][b, : -(-length // blk)].long()
    k = s["k"][p].view(torch.float8_e4m3fn).float() * s["ks"][p][..., None, None]
    v = s["v"][p].view(torch.float8_e4m3fn).float() * s["vs"][p][..., None, None]
    k = k.permute(1, 0, 2, 3).reshape(k.shape[1], -1, k.shape[3])[:, :length]
    v = v.permute(1, 0, 3, 2).reshape(v.shape[1], -1, v.shape[2])[:, :length]
    return k, v


def _plain_rows(s):
    c = s["case"]
    h, d, q = c["hkv"], c["d"], s["q"]
    grp, out, r = c["hq"] // h, [], 0
    held, new, _ = _lengths(c)
    for b, (length, n) in enumerate(zip(held, new)):
        k, v = _decoded(s, b, length)
        qb = q[r:r + n].float().reshape(n, h, grp, d).permute(1, 2, 0, 3).reshape(h, grp * n, d)
        sc = torch.matmul(qb, k.transpose(1, 2).contiguous()).reshape(h, grp, n, length) * d ** -0.5
        pos = torch.arange(length - n, length, device=q.device)[:, None]
        j = torch.arange(length, device=q.device)[None, :]
        sees = j <= pos
        if c["op"] == "score":
            if c["cap"]:
                sc = c["cap"] * torch.tanh(sc / c["cap"])
            if c["bias"]:
                sc = sc - s["slopes"].view(h, grp, 1, 1) * (pos - j).abs().float()
            if c["prefix"]:
                sees = sees | (j < s["prefix"][b])
            if c["window"]:
                sees = sees & (j > pos - c["window"])
            if c["docs"]:
                sees = sees & (j >= s["first"][r:r + n, None])
        sc = sc.masked_fill(~sees, float("-inf"))
        p = torch.exp(sc - sc.amax(-1, keepdim=True))
        o = torch.matmul(p.reshape(h, grp * n, length), v) / p.sum(-1).reshape(h, grp * n, 1)
        out.append(o.reshape(h, grp, n, d).permute(2, 0, 1, 3).reshape(n, c["hq"], d))
        r += n
    return torch.cat(out).to(q.dtype)


def _plain_sample(s):
    x, rows = s["logits"].double(), s["logits"].shape[0]

    def each(name):
        return torch.as_tensor(s[name], dtype=torch.float64, device=x.device).expand(rows)[:, None]
    t, top_k, top_p, min_p = (each(n) for n in ("temperature", "top_k", "top_p", "min_p"))
    vocab = x.shape[1]
    v, at = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((v - v[:, :1]) / torch.where(t > 0, t, torch.ones_like(t)))
    rank = torch.arange(vocab, device=x.device)[None, :]
    w = torch.where((top_k <= 0) | (rank < top_k), w, torch.zeros_like(w))
    before = torch.cumsum(w, 1) - w
    total = w.sum(1, keepdim=True)
    keep = (rank == 0) | (((top_p >= 1) | (before < top_p * total)) & (w >= min_p))
    kept = torch.zeros_like(w).scatter_(1, at, torch.where(keep, w, torch.zeros_like(w)))
    mass = torch.cumsum(kept, 1)
    u = s["u"].double()[:, None] * mass[:, -1:]
    # the first token whose sum passes u times the mass kept; no temperature: the largest logit
    token = torch.searchsorted(mass, u, right=True).clamp(max=vocab - 1)
    return torch.where(t > 0, token, at[:, :1])[:, 0].to(torch.int32)


# ------------------------------------------------------------------ one pass


def run(state):
    s, c = state, state["case"]
    if own:
        from perm_amd import kvcache, kvpages, sampling
        if c["op"] == "sample":
            return sampling.sample(s["logits"], s["u"], temperature=s["temperature"],
                                   top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
        cache = kvcache.KvCache(s["k"], s["v"], s["ks"], s["vs"])
        if c["op"] == "fork":
            kvpages.free(s["refs"], s["table"], s["children"])
            kvpages.fork(s["refs"], s["table"], s["lens"], s["parents"], s["children"], c["block"])
            src, dst, short = kvpages.grow(s["refs"], s["table"], s["lens"], s["new"], c["block"])
            kvpages.copy(cache, src, dst)
            return _books(s, src=src, dst=dst, short=short)
        if c["op"] == "compact":
            refs, table = s["refs"].clone(), s["table"].clone()
            src, dst, used = kvpages.compact(refs, table)
            kvpages.copy(cache, src, dst)
            return {**_books(s, src=src, dst=dst, used=used), "refs": refs, "table": table}
        if c["op"] == "shared":
            return kvcache.attention(s["q"], cache, s["table"], s["held"], s["offsets"],
                                     shared=s["shared"])
        return kvcache.attention(s["q"], cache, s["table"], s["held"], s["offsets"],
                                 window=c["window"], softcap=c["cap"], slopes=s["slopes"],
                                 first=s["first"], prefix=s["prefix"])
    return {"fork": _plain_fork, "compact": _plain_compact, "shared": _plain_rows,
            "score": _plain_rows, "sample": _plain_sample}[c["op"]](s)


def work(case):
    c = case
    if c["op"] == "sample":
        return {"bytes": c["rows"] * c["vocab"] * SIZE[c["dtype"]], "flops": 0}
    if c["op"] in ("fork", "compact"):
        page = 2 * c["hkv"] * (c["block"] * c["d"] + 4)
        if c["op"] == "fork":
            rng, moved, ints = _dice(c), 0, 0
            for i in range(c["parents"]):
                t = c["top"] if i == 0 else _log(rng, max(1, c["top"] // 8), c["top"])
                moved += c["each"] if t % c["block"] else 0
                # a child's entries read and cleared, then written; the holders of each page twice
                ints += (2 + c["each"] * 5) * -(-t // c["block"])
            return {"bytes": 2 * moved * page + 4 * ints, "flops": 0}
        used = max(1, int(c["pages"] * c["part"]))
        # of the pages past the used ones, as many are in use as chance leaves there
        moved = used * (c["pages"] - used) // c["pages"]
        return {"bytes": 2 * moved * page + 4 * (2 * c["pages"] + 2 * used), "flops": 0}
    held, new, front = _lengths(c)
    row = c["hkv"] * c["d"]
    pairs = tokens = 0
    at, rows = 0, _ranges(c)[0]
    for length, n in zip(held, new):
        mine = [(lo, hi) for _, _, lo, hi in rows[at:at + n]]
        at += n
        pairs += sum(hi - lo + 1 for lo, hi in mine)
        end = 0
        for lo, hi in sorted(mine):
            tokens += max(0, hi + 1 - max(lo, end))
            end = max(end, hi + 1)
    if front:
        tokens -= (c["each"] - 1) * sum(front)
    return {"bytes": 2 * tokens * row + 2 * 2 * sum(new) * c["hq"] * c["d"],
            "flops": 4.0 * c["d"] * c["hq"] * pairs}


# ------------------------------------------------------------------ the definitions in 64 bits


def _values(s):
    return {"k": s["k"].view(torch.float8_e4m3fn).double(), "v": s["v"].view(torch.float8_e4m3fn).double(),
            "k_scale": s["ks"].double(), "v_scale": s["vs"].double()}


def _moved(s, pairs):
    """The cache's values after the pages of these pairs were copied, one after the other."""
    out = _values(s)
    for a, b in pairs:
        for t in out.values():
            t[b] = t[a]
    return out


def _ints(v):
    return torch.tensor(v, **I32)


def _exact_fork(c, s):
    """The books kept a sequence at a time, as one would by hand."""
    refs, table = s["refs"].tolist(), s["table"].tolist()
    lens, new, blk = s["lens"].tolist(), s["new"].tolist(), c["block"]
    for mum, kid in zip(s["parents"].tolist(), s["children"].tolist()):
        n = math.ceil(lens[mum] / blk)
        table[kid] = table[mum][:n] + [-1] * (len(table[kid]) - n)
        for p in table[kid][:n]:
            refs[p] += 1
    free = [p for p, n in enumerate(refs) if n == 0]
    held = list(refs)
    src, dst, short, pairs = [], [], [], []
    for b, row in enumerate(table):
        src.append(-1)
        dst.append(-1)
        short.append(0)
        for p in range(lens[b], lens[b] + new[b]):
            i = p // blk
            if (i > lens[b] // blk and p % blk) or (row[i] >= 0 and held[row[i]] <= 1):
                continue
            page, old = free.pop(0), row[i]
            row[i] = page
            refs[page] = 1
            if old >= 0:
                refs[old] -= 1
                if p % blk:
                    src[b], dst[b] = old, page
                    pairs.append((old, page))
            held[page] = 1
    return {"refs": _ints(refs), "table": _ints(table), **_moved(s, pairs), "src": _ints(src),
            "dst": _ints(dst), "short": _ints(short)}


def _exact_compact(c, s):
    refs, table = s["refs"].tolist(), s["table"].tolist()
    used = sum(n > 0 for n in refs)
    pairs, hole = [], 0
    for p in range(used, c["pages"]):
        if refs[p]:
            while refs[hole]:
                hole += 1
            pairs.append((p, hole))
            refs[hole], refs[p] = refs[p], 0
    to = dict(pairs)
    table = [[to.get(p, p) for p in row] for row in table]
    pad = [-1] * (c["pages"] // 2 - len(pairs))
    return {"refs": _ints(refs), "table": _ints(table), **_moved(s, pairs),
            "src": _ints([a for a, _ in pairs] + pad), "dst": _ints([b for _, b in pairs] + pad),
            "used": _ints([used])}


def _exact_rows(c, s):
    held, new, _ = _lengths(c)
    rows, _ = _ranges(c)
    lo = torch.tensor([r[2] for r in rows], device="cuda")[:, None]
    hi = torch.tensor([r[3] for r in rows], device="cuda")[:, None]
    at = torch.tensor([r[0] for r in rows], device="cuda")[:, None]
    value = _values(s)
    grp, r = c["hq"] // c["hkv"], 0
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, (length, n) in enumerate(zip(held, new)):
        j = torch.arange(length, device="cuda")
        page, slot = s["table"][b].long()[j // c["block"]], j % c["block"]
        sees = (j >= lo[r:r + n]) & (j <= hi[r:r + n])
        for h in range(c["hq"]):
            x = h // grp
            k = value["k"][page, x, slot] * value["k_scale"][page, x, None]
            v = value["v"][page, x, :, slot] * value["v_scale"][page, x, None]
            sc = (s["q"][r:r + n, h].double() @ k.t()) / math.sqrt(c["d"])
            if c.get("cap"):
                sc = torch.tanh(sc / c["cap"]) * c["cap"]
            if c.get("bias"):
                sc -= s["slopes"][h].double() * (at[r:r + n] - j).abs()
            out[r:r + n, h] = torch.softmax(sc.masked_fill(~sees, -math.inf), 1) @ v
        r += n
    return out


def _exact_sample(c, s):
    """A row at a time: the tokens by falling logit, the sums from the smallest weight on."""
    out = []

    def one(name, i):
        return s[name][i].item() if torch.is_tensor(s[name]) else s[name]
    for i in range(c["rows"]):
        x = s["logits"][i].double()
        t, k, p, m = (one(n, i) for n in ("temperature", "top_k", "top_p", "min_p"))
        if t <= 0:
            out.append(int(torch.nonzero(x == x.max())[0]))
            continue
        order = torch.argsort(-x, stable=True)
        if k > 0:
            order = order[:k]
        w = ((x[order] - x[order[0]]) / t).exp()
        if p < 1:
            after = w.flip(0).cumsum(0).flip(0)  # its own weight and those of less likely ones
            n = int((after[0] - after < p * after[0]).sum())
            order, w = order[:max(n, 1)], w[:max(n, 1)]
        n = max(1, int((w >= m).sum()))
        order, back = order[:n].sort()
        mass = w[:n][back].cumsum(0)
        out.append(int(order[min(int((mass <= s["u"][i].double() * mass[-1]).sum()), n - 1)]))
    return _ints(out)


def exact(case, seed):
    s = prepare(case, seed)
    return {"fork": _exact_fork, "compact": _exact_compact, "shared": _exact_rows,
            "score": _exact_rows, "sample": _exact_sample}[case["op"]](case, s)
