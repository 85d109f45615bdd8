"""The low-bit serving operators that are timed, in their plain form and as the library's calls.

A case is a dict of plain values. Its "op" names the operator:

  quantize   mxfp4.quantize, mxfp4.dequantize   rows into MXFP4 blocks, and the values they hold
  linear     mxfp4.linear        y = x w^T on MXFP4 weights, x quantised in the call
  write      kvcache.write       new keys and values into the paged 8-bit cache
  read       kvcache.read        a cache's keys and values back in 16 bits
  attend     kvcache.attention   attention of query rows over the 8-bit cache

Layouts. MXFP4: codes uint8 [rows, k / 2], the even column in the low four bits, and one
exponent byte (bias 127) for each 32 columns in the order the matrix cores take them: scales
uint8 [ceil(k / 128), ceil(rows / 64), 4, 16, 4], indexed by k / 128, row / 64, k / 32 % 4,
row % 16 and row / 16 % 4; 0 past the end of a row.
Cache: k uint8 [pages, heads, block, d] and v uint8 [pages, heads, d, block], e4m3 codes, with
float32 scales [pages, heads] that are powers of two. table int32 [sequences, pages of each].
"""
import random

import torch

own = False

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # one token's activations at a small model's width: the call's own latency
        dict(name="quantize-token", op="quantize", rows=1, k=1024, dtype="bf16"),
        # a wide decoder layer's largest matrix, quantised once from float32
        dict(name="quantize-weight", op="quantize", rows=14336, k=4096, dtype="f32"),
        # a generated token through the wide layer's gate matrix
        dict(name="linear-token", op="linear", m=1, n=14336, k=4096, dtype="bf16"),
        # a few sequences' tokens through a ragged projection in float16
        dict(name="linear-few", op="linear", m=17, n=1000, k=1056, dtype="f16"),
        # a prompt of 4096 tokens through the wide layer's gate matrix
        dict(name="linear-prompt", op="linear", m=4096, n=14336, k=4096, dtype="bf16"),
        # one new token of each of 64 running sequences, in pages begun earlier
        dict(name="write-tokens", op="write", b=64, top=4096, new=1, hkv=8, d=128, block=16,
             dtype="bf16"),
        # eight prompts of up to 4096 tokens into empty caches
        dict(name="write-prompts", op="write", b=8, top=0, new=4096, hkv=8, d=128, block=16,
             dtype="bf16"),
        # three short sequences of a small model read back, float16, pages of 32
        dict(name="read-short", op="read", b=3, top=333, hkv=2, d=64, block=32, dtype="f16"),
        # sixteen long sequences read back (moved to a server that keeps 16 bits)
        dict(name="read-long", op="read", b=16, top=8192, hkv=8, d=128, block=16, dtype="bf16"),
        # one generated token at the end of a very long sequence
        dict(name="attend-long", op="attend", b=1, top=131072, new=1, hq=32, hkv=8, d=128,
             block=16, window=0, dtype="bf16"),
        # one generated token of each of 64 sequences of mixed lengths
        dict(name="attend-tokens", op="attend", b=64, top=4096, new=1, hq=16, hkv=8, d=128,
             block=16, window=0, dtype="bf16"),
        # two prompts' last 4096 tokens over up to 8192: the largest
        dict(name="attend-prompt", op="attend", b=2, top=8192, new=4096, hq=16, hkv=8, d=128,
             block=16, window=0, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(("quantize", "linear", "linear", "write", "read", "attend", "attend"))
    half = rng.choice(("bf16", "f16"))
    if op == "quantize":
        return dict(op=op, rows=_log(rng, 1, 14336), k=32 * _log(rng, 4, 128),
                    dtype=rng.choice(("bf16", "f16", "f32")))
    if op == "linear":
        return dict(op=op, m=_log(rng, 1, 4096), n=_log(rng, 64, 14336),
                    k=32 * _log(rng, 4, 128), dtype=half)
    hkv, d, block = rng.choice((1, 2, 4, 8)), rng.choice((64, 80, 128)), rng.choice((16, 32, 64))
    if op == "write":
        fresh = rng.random() < 0.5
        return dict(op=op, b=_log(rng, 1, 8 if fresh else 64), top=0 if fresh else _log(rng, 16, 4096),
                    new=_log(rng, 16, 4096) if fresh else rng.choice((1, 1, 2, 5)), hkv=hkv, d=d,
                    block=block, dtype=half)
    if op == "read":
        return dict(op=op, b=_log(rng, 1, 16), top=_log(rng, 16, 8192), hkv=hkv, d=d, block=block,
                    dtype=half)
    heads = dict(hq=hkv * rng.choice((1, 2, 4)), hkv=hkv, d=d, block=block, dtype=half)
    if rng.random() < 0.5:
        return dict(op=op, b=_log(rng, 1, 64), top=_log(rng, 64, 8192), new=rng.choice((1, 1, 1, 4)),
                    window=rng.choice((0, 0, 1000)), **heads)
    return dict(op=op, b=rng.choice((1, 2)), top=_log(rng, 512, 4096), new=_log(rng, 24, 2048),
                window=rng.choice((0, 0, 500)), **heads)


def _counts(c):
    """(tokens held before, new tokens) of each sequence: ragged, and fixed by the case alone.
    A write has up to top + new tokens a sequence in the end, the others up to top."""
    rng = random.Random(c["b"] * 1000003 + c["top"] * 101 + c.get("new", 0))
    if c["op"] == "write":
        new = [c["new"] if c["new"] < 16 or i == 0 else _log(rng, c["new"] // 8, c["new"])
               for i in range(c["b"])]
        return [_log(rng, 1, c["top"]) if c["top"] else 0 for _ in new], new
    held = [c["top"] if i == 0 else _log(rng, max(1, c["top"] // 16), c["top"])
            for i in range(c["b"])]
    return held, [min(h, c.get("new", 0)) for h in held]


def _capacity(c):
    """Pages of a sequence's table row."""
    return -(-(c["top"] + (c["new"] if c["op"] == "write" else 0)) // c["block"])


def _offsets(counts):
    total, at = 0, [0]
    for n in counts:
        total += n
        at.append(total)
    return at


def _activations(g, rows, cols, dtype):
    """Normal rows with log-normal channel scales, the largest channels far above the rest."""
    scale = torch.exp(torch.randn((cols,), generator=g, device="cuda"))
    return (torch.randn((rows, cols), generator=g, device="cuda") * scale).to(dtype)


def _nibbles(g, rows, k):
    return torch.randint(0, 256, (rows, k // 2), generator=g, device="cuda", dtype=torch.uint8)


def _two(e):
    """2^e of whole numbers, exactly, in 64 bits (-1022 <= e <= 1023)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": c}
    if c["op"] == "quantize":
        if c["dtype"] == "f32":
            s["x"] = torch.randn((c["rows"], c["k"]), generator=g, device="cuda") * 0.02
        else:
            s["x"] = _activations(g, c["rows"], c["k"], DT[c["dtype"]])
        return s
    if c["op"] == "linear":
        s["x"] = _activations(g, c["m"], c["k"], DT[c["dtype"]])
        # weights as a quantiser leaves them: any code, block exponents around 2^-7
        s["codes"] = _nibbles(g, c["n"], c["k"])
        s["scales"] = torch.randint(117, 122, (-(-c["k"] // 128), -(-c["n"] // 64), 4, 16, 4),
                                    generator=g, device="cuda", dtype=torch.uint8)
        s["scales"][c["k"] // 128:, :, c["k"] // 32 % 4:] = 0
        return s
    held, new = _counts(c)
    cap, h, d, blk = _capacity(c), c["hkv"], c["d"], c["block"]
    pages = c["b"] * cap + 1
    codes = []
    for shape in ((pages, h, blk, d), (pages, h, d, blk)):
        t = torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16) * 80
        codes.append(t.to(torch.float8_e4m3fn).view(torch.uint8))
    s["k"], s["v"] = codes
    s["ks"], s["vs"] = (_two(torch.randint(-9, -6, (pages, h), generator=g, device="cuda")).float()
                        for _ in range(2))
    perm = torch.randperm(pages, generator=g, device="cuda")
    s["table"] = perm[: c["b"] * cap].reshape(c["b"], cap).to(torch.int32)
    s["held"] = torch.tensor(held, dtype=torch.int32, device="cuda")
    dt = DT[c["dtype"]]
    if c["op"] == "read":
        s["offsets"] = torch.tensor(_offsets(held), dtype=torch.int32, device="cuda")
        s["total"] = sum(held)
        return s
    s["offsets"] = torch.tensor(_offsets(new), dtype=torch.int32, device="cuda")
    if c["op"] == "write":
        shape = (sum(new), h, d)
        # a key's channels differ in size; values are even
        s["k_new"] = _activations(g, shape[0], h * d, dt).reshape(shape)
        s["v_new"] = torch.randn(shape, generator=g, device="cuda").to(dt)
    else:
        s["q"] = torch.randn((sum(new), c["hq"], d), generator=g, device="cuda").to(dt)
        s["max_new"] = max(new)
    return s


# ------------------------------------------------------------------ plain forms (32 bits)


def _pow2(byte):
    """2^(byte - 127) of uint8 exponent bytes; NaN for 255."""
    b = byte.to(torch.int32)
    bits = torch.where(b == 0, torch.full_like(b, 1 << 22), b << 23)
    f = bits.view(torch.float32)
    return torch.where(b == 255, torch.full_like(f, float("nan")), f)


def _mx_values(x):
    """float32 [rows, k]: what x's MXFP4 blocks hold."""
    b = x.float().reshape(x.shape[0], -1, 32)
    amax = b.abs().amax(-1, keepdim=True)
    e = torch.frexp(amax).exponent - 3
    e = torch.where(amax == 0, torch.full_like(e, -127), e.clamp(-127, 127))
    bad = ~torch.isfinite(amax)
    v = b.abs() * _pow2((127 - e).to(torch.uint8))
    q = torch.where(v < 2, torch.round(v * 2) / 2,
                    torch.where(v < 4, torch.round(v), (torch.round(v / 2) * 2).clamp(max=6)))
    y = torch.copysign(q, b) * _pow2((e + 127).to(torch.uint8))
    return torch.where(bad, torch.full_like(y, float("nan")), y).reshape(x.shape)


def _mx_decode(codes, scales, k):
    """float32 [rows, k] of stored codes and scale bytes."""
    lut = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
    nib = torch.stack([codes & 15, codes >> 4], dim=-1).reshape(codes.shape[0], -1, 32)
    by_row = scales.permute(1, 4, 3, 0, 2).flatten(3).flatten(0, 2)[: codes.shape[0], : k // 32]
    return (lut[nib.int()] * _pow2(by_row)[..., None]).reshape(codes.shape[0], k)


def _e4m3_scale(amax):
    """The smallest power of two 2^e, -60 <= e <= 60, with amax <= 448 * 2^e."""
    f = torch.frexp(amax)
    e = f.exponent - 8 - (f.mantissa <= 0.875).int()
    e = torch.where(amax == 0, torch.full_like(e, -60), e.clamp(-60, 60))
    return _pow2((e + 127).to(torch.uint8))


def _seq_of(t, offsets):
    """The sequence of each of t rows."""
    return torch.searchsorted(offsets[1:].contiguous(), torch.arange(t, device=offsets.device),
                              right=True)


def _plain_write(s):
    c = s["case"]
    blk, t = c["block"], s["k_new"].shape[0]
    seq = _seq_of(t, s["offsets"])
    held = s["held"].long()
    pos = held[seq] + torch.arange(t, device=seq.device) - s["offsets"].long()[seq]
    page, slot = s["table"].long()[seq, pos // blk], pos % blk
    grow = (pos // blk == held[seq] // blk) & (held[seq] % blk > 0)
    # the pages begun earlier, one at most for each sequence, and the slots they hold
    old = s["table"].long().gather(1, (held // blk).clamp(max=s["table"].shape[1] - 1)[:, None])[:, 0]
    kept = torch.arange(blk, device=seq.device)[None, :] < (held % blk)[:, None]
    for new, code, scale, by_slot in ((s["k_new"], s["k"], s["ks"], True),
                                      (s["v_new"], s["v"], s["vs"], False)):
        x = new.float()
        fin = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(-1)
        top = torch.zeros_like(scale)
        top.index_reduce_(0, page, fin, "amax")
        want = _e4m3_scale(top)
        f8 = code.view(torch.float8_e4m3fn)
        wide = torch.zeros(scale.shape[0], device=scale.device).index_fill_(0, page, 1.0)[:, None] > 0
        keeps = torch.zeros(scale.shape[0], device=scale.device)
        keeps = keeps.index_reduce_(0, page, grow.float(), "amax")[:, None] > 0
        now = torch.where(wide, torch.where(keeps, torch.maximum(scale, want), want), scale)
        ratio = (scale / now)[old][:, :, None, None]
        was = f8[old].float()
        mask = kept[:, None, :, None] if by_slot else kept[:, None, None, :]
        mask = mask & keeps[old][:, :, None, None]
        code[old] = torch.where(mask, was * ratio, was).to(torch.float8_e4m3fn).view(torch.uint8)
        scale.copy_(now)
        y = (x * (1.0 / now[page])[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn)
        if by_slot:
            code[page, :, slot] = y.view(torch.uint8)
        else:
            code[page, :, :, slot] = y.view(torch.uint8)
    return _cache_out(s)


def _cache_out(s):
    return {"k": s["k"].view(torch.float8_e4m3fn), "v": s["v"].view(torch.float8_e4m3fn),
            "k_scale": s["ks"], "v_scale": s["vs"]}


def _plain_read(s):
    blk = s["case"]["block"]
    seq = _seq_of(s["total"], s["offsets"])
    pos = torch.arange(s["total"], device=seq.device) - s["offsets"].long()[seq]
    page, slot = s["table"].long()[seq, pos // blk], pos % blk
    dt = DT[s["case"]["dtype"]]
    k = s["k"][page, :, slot].view(torch.float8_e4m3fn).float() * s["ks"][page][..., None]
    v = s["v"][page, :, :, slot].view(torch.float8_e4m3fn).float() * s["vs"][page][..., None]
    return {"k": k.to(dt), "v": v.to(dt)}


def _plain_attend(s):
    c = s["case"]
    h, d, q = c["hkv"], c["d"], s["q"]
    grp, nb, qn = c["hq"] // h, c["b"], s["max_new"]
    table, lens = s["table"].long(), s["held"].long()
    off = s["offsets"].long()
    k = s["k"].view(torch.float8_e4m3fn)[table].float() * s["ks"][table][..., None, None]
    v = s["v"].view(torch.float8_e4m3fn)[table].float() * s["vs"][table][..., None, None]
    k = k.permute(0, 2, 1, 3, 4).reshape(nb, h, -1, d)
    v = v.permute(0, 2, 1, 4, 3).reshape(nb, h, -1, d)
    i = torch.arange(qn, device=q.device)
    rows = (off[:-1, None] + i).clamp(max=q.shape[0] - 1)
    qp = q[rows].float().reshape(nb, qn, h, grp, d).permute(0, 2, 3, 1, 4).reshape(nb, h, -1, d)
    sc = torch.matmul(qp, k.transpose(-1, -2)) * d ** -0.5
    pos = lens[:, None] - (off[1:] - off[:-1])[:, None] + i
    j = torch.arange(k.shape[2], device=q.device)
    sees = (j <= pos[..., None]) & (j < lens[:, None, None])
    if c["window"]:
        sees = sees & (j > pos[..., None] - c["window"])
    sees = sees[:, None, None].expand(nb, h, grp, qn, -1).reshape(sc.shape)
    sc = sc.masked_fill(~sees, float("-inf"))
    top = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    v = torch.where((j < lens[:, None])[:, None, :, None], v, torch.zeros_like(v))
    o = torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))
    o = o.reshape(nb, h, grp, qn, d).permute(0, 3, 1, 2, 4).reshape(nb * qn, c["hq"], d)
    seq = _seq_of(q.shape[0], s["offsets"])
    return o[seq * qn + torch.arange(q.shape[0], device=q.device) - off[seq]].to(q.dtype)


# ------------------------------------------------------------------ one pass


def run(state):
    s, c = state, state["case"]
    if own:
        from perm_amd import kvcache, mxfp4
        if c["op"] == "quantize":
            return mxfp4.dequantize(mxfp4.quantize(s["x"]), s["x"].dtype)
        if c["op"] == "linear":
            return mxfp4.linear(s["x"], mxfp4.MxTensor(s["codes"], s["scales"]))
        cache = kvcache.KvCache(s["k"], s["v"], s["ks"], s["vs"])
        if c["op"] == "write":
            kvcache.write(cache, s["k_new"], s["v_new"], s["table"], s["held"], s["offsets"])
            return _cache_out(s)
        if c["op"] == "read":
            k, v = kvcache.read(cache, s["table"], s["offsets"], s["total"], DT[c["dtype"]])
            return {"k": k, "v": v}
        # one row for each sequence needs no offsets
        off = None if s["max_new"] == 1 else s["offsets"]
        return kvcache.attention(s["q"], cache, s["table"], s["held"], off, window=c["window"])
    if c["op"] == "quantize":
        return _mx_values(s["x"]).to(s["x"].dtype)
    if c["op"] == "linear":
        w = _mx_decode(s["codes"], s["scales"], c["k"])
        return torch.matmul(_mx_values(s["x"]), w.t()).to(s["x"].dtype)
    return {"write": _plain_write, "read": _plain_read, "attend": _plain_attend}[c["op"]](s)


def work(case):
    c = case
    if c["op"] == "quantize":
        n = c["rows"] * c["k"]
        held = n / 2 + n / 32
        return {"bytes": 2 * (n * SIZE[c["dtype"]] + held), "flops": 0}
    if c["op"] == "linear":
        m, n, k = c["m"], c["n"], c["k"]
        return {"bytes": (m * k + m * n) * 2 + n * (k / 2 + k / 32), "flops": 2.0 * m * n * k}
    held, new = _counts(c)
    row = c["hkv"] * c["d"]
    if c["op"] == "write":
        return {"bytes": 2 * sum(new) * row * (2 + 1), "flops": 0}
    if c["op"] == "read":
        return {"bytes": 2 * sum(held) * row * (2 + 1), "flops": 0}
    pairs = read = 0
    for length, n in zip(held, new):
        w = c["window"] or length
        read += min(length, w + n - 1)
        pairs += sum(min(p + 1, w) for p in range(length - n, length))
    return {"bytes": 2 * read * row + 2 * 2 * sum(new) * c["hq"] * c["d"],
            "flops": 4.0 * c["d"] * c["hq"] * pairs}


# ------------------------------------------------------------------ the definitions in 64 bits


def _grid_round(x, mant, emin, top):
    """x on the floating grid of `mant` fraction bits, smallest exponent emin and largest value
    top, to nearest, ties to the even code, saturating."""
    _, e = torch.frexp(x)
    step = _two((e - 1).clamp(min=emin) - mant)
    return (torch.round(x / step) * step).clamp(-top, top)


def _exact_mx(x):
    b = x.double().unflatten(1, (-1, 32))
    a = b.abs().max(dim=2).values
    # bits of a: floor(log2 a) is its exponent field (64 bits hold float32's subnormals as normal)
    e = ((a.view(torch.int64) >> 52) - 1023 - 2).clamp(-127, 127)[:, :, None]
    return (_grid_round(b * _two(-e), 1, 0, 6.0) * _two(e)).flatten(1)


def _exact_scale(amax):
    """The cache's scale for a host number: 2^e with the least e, -60 <= e <= 60, that holds it."""
    e = -60
    while e < 60 and amax > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def _exact_write(c, s):
    held, new = _counts(c)
    blk, table = c["block"], s["table"].cpu().tolist()
    out = {}
    for key, x, name in (("k", s["k_new"], "ks"), ("v", s["v_new"], "vs")):
        # [pages, heads, block, d] for both, in 64 bits
        val = s[key].view(torch.float8_e4m3fn).double()
        val = val if key == "k" else val.transpose(2, 3).contiguous()
        sc, x = s[name].double(), x.double()
        tops = x.abs().amax(2)
        at = _offsets(new)
        jobs = []
        for b in range(c["b"]):
            p = held[b]
            while p < held[b] + new[b]:
                n = min(blk - p % blk, held[b] + new[b] - p)
                jobs.append((table[b][p // blk], p % blk, at[b] + p - held[b], n))
                p += n
        peak = torch.stack([tops[r:r + n].amax(0) for _, _, r, n in jobs]).cpu().tolist()
        want = torch.tensor([[_exact_scale(a) for a in row] for row in peak], dtype=torch.float64,
                            device=x.device)
        for (page, slot, r, n), w in zip(jobs, want):
            if slot:
                w = torch.maximum(w, sc[page])
                moved = val[page, :, :slot] * (sc[page] / w)[:, None, None]
                val[page, :, :slot] = _grid_round(moved, 3, -6, 448.0)
            sc[page] = w
            y = x[r:r + n].transpose(0, 1) / w[:, None, None]
            val[page, :, slot:slot + n] = _grid_round(y, 3, -6, 448.0)
        out[key] = val if key == "k" else val.transpose(2, 3).contiguous()
        out[key + "_scale"] = sc
    return out


def _exact_tokens(c, s, b, length):
    """One sequence's keys and values [heads, length, d]."""
    n = -(-length // c["block"])
    p = s["table"][b, :n].long()
    k = s["k"][p].view(torch.float8_e4m3fn).double() * s["ks"][p].double()[:, :, None, None]
    v = s["v"][p].view(torch.float8_e4m3fn).double() * s["vs"][p].double()[:, :, None, None]
    k = k.transpose(0, 1).flatten(1, 2)[:, :length]
    v = v.permute(1, 0, 3, 2).flatten(1, 2)[:, :length]
    return k, v


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "quantize":
        return _exact_mx(s["x"])
    if c["op"] == "linear":
        mag = torch.tensor(E2M1, dtype=torch.float64, device="cuda")
        w = torch.empty((c["n"], c["k"]), dtype=torch.float64, device="cuda")
        for half in (0, 1):
            nib = (s["codes"] >> (4 * half)) & 15
            w[:, half::2] = mag[(nib & 7).long()] * (1 - 2 * (nib >> 3).double())
        row = torch.arange(c["n"], device="cuda")[:, None]
        blk = torch.arange(c["k"] // 32, device="cuda")[None, :]
        e = s["scales"][blk // 4, row // 64, blk % 4, row % 16, row // 16 % 4].int() - 127
        w *= _two(e).repeat_interleave(32, dim=1)
        return _exact_mx(s["x"]) @ w.t()
    if c["op"] == "write":
        return _exact_write(c, s)
    held, new = _counts(c)
    if c["op"] == "read":
        kv = [_exact_tokens(c, s, b, n) for b, n in enumerate(held)]
        return {"k": torch.cat([k.transpose(0, 1) for k, _ in kv]),
                "v": torch.cat([v.transpose(0, 1) for _, v in kv])}
    out, r, grp = [], 0, c["hq"] // c["hkv"]
    for b, (length, n) in enumerate(zip(held, new)):
        k, v = _exact_tokens(c, s, b, length)
        o = torch.empty((n, c["hq"], c["d"]), dtype=torch.float64, device="cuda")
        for h in range(c["hq"]):
            sc = (s["q"][r:r + n, h].double() @ k[h // grp].t()) / c["d"] ** 0.5
            pos = torch.arange(length - n, length, device="cuda")[:, None]
            j = torch.arange(length, device="cuda")[None, :]
            hide = j > pos
            if c["window"]:
                hide |= j <= pos - c["window"]
            o[:, h] = torch.softmax(sc.masked_fill(hide, -torch.inf), -1) @ v[h // grp]
        out.append(o)
        r += n
    return torch.cat(out)
