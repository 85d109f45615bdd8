"""Attention over the cache with capped scores, a distance's share, documents, prefixes and pages that
sequences have in common, against the float64 definition."""
import itertools

import numpy as np
import pytest
import torch

from oracle import attention_oracle as A
from test_gpu_kvcache import HALF_ULP, _filled_cache, _i32, _offsets, kv  # noqa: F401

pytestmark = pytest.mark.gpu
HALVES = [torch.bfloat16, torch.float16]


@pytest.fixture(autouse=True)
def _fronts_apart(kv, monkeypatch, request):  # noqa: F811
    """Common pages are read apart at every size here, but where the rule for it is tested."""
    if "rule" not in request.node.name:
        monkeypatch.setattr(kv, "_front_pays", lambda *a: True)


def _check(kv, c, o, table, lens, counts, hq, dtype, rng, offsets=True, spread=1.0, slopes=None, first=None,  # noqa: F811
           prefix=None, shared=None, causal=True, window=0, scale=None, softcap=0.0):
    heads, d = o.k.shape[1], o.k.shape[3]
    rows = int(np.sum(counts))
    q = torch.from_numpy(rng.standard_normal((rows, hq, d)) * spread).to(dtype).cuda()
    args = dict(causal=causal, window=window, scale=scale, softcap=softcap,
                slopes=None if slopes is None else torch.tensor(slopes, dtype=torch.float32, device="cuda"),
                first=None if first is None else _i32(first), prefix=None if prefix is None else _i32(prefix),
                shared=None if shared is None else _i32(shared))
    off = _offsets(counts) if offsets else None
    table = np.array(table)
    if shared is not None:  # a group's rows of the table begin alike
        each = len(lens) // len(shared)
        for b in range(len(lens)):
            table[b, :max(shared[b // each], 0)] = table[b - b % each, :max(shared[b // each], 0)]
    out, lse = kv.attention(q, c, _i32(table), _i32(lens), off, return_lse=True, **args)
    again = kv.attention(q, c, _i32(table), _i32(lens), off, **args)
    assert torch.equal(again.view(torch.int16), out.view(torch.int16))
    assert out.shape == q.shape and out.dtype == dtype
    r = 0
    for b, n in enumerate(counts):
        k, v, have = (torch.from_numpy(t).cuda() for t in o.tokens(table[b], min(lens[b], table.shape[1] * o.block)))
        want, wl, bound, lb = A.attention(q[r:r + n].double(), k, v, have, lens[b], causal, window, scale, softcap,
                                          None if slopes is None else np.float32(slopes).astype(float).tolist(),
                                          None if first is None else args["first"][r:r + n],
                                          0 if prefix is None else prefix[b])
        got, gl = out[r:r + n].double(), lse[r:r + n].double()
        assert torch.equal(torch.isnan(got), torch.isnan(want)), b
        limit = bound.nan_to_num(0.0) + HALF_ULP[dtype] * want.abs().nan_to_num(0.0) * 1.01 + 2.0 ** -24
        err = (got - want).abs().nan_to_num(0.0) / limit
        assert err.numel() == 0 or float(err.max()) <= 1, (b, float(err.max()))
        # a NaN score makes the row's sum NaN on both sides
        assert torch.equal(torch.isfinite(gl), torch.isfinite(wl)), b
        fin = torch.isfinite(wl)
        assert bool(((gl - wl).abs() <= lb)[fin].all()), b
        r += n


def _many(c, counts, hq, table, window=0):
    """The call is one for the kernel of 128 rows a workgroup: pairs times the tokens they may see."""
    heads, block = c.k.shape[1:3]
    cap = table.shape[1] * block
    assert sum(counts) * hq * (min(cap, window + 128) if window else cap) > 1 << 24
    assert sum(counts) * (hq // heads) > 64 * len(counts)


def _slopes(hq):
    return [2.0 ** (-8.0 * (x + 1) / hq) for x in range(hq)]


SCORES = [dict(softcap=5.0), dict(softcap=50.0), dict(softcap=1000.0), dict(slopes=True), dict(softcap=20.0, slopes=True)]


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("scores", SCORES, ids=str)
@pytest.mark.parametrize("block,heads,d,group", [(16, 2, 128, 2), (64, 1, 80, 4), (32, 1, 256, 1), (128, 3, 16, 1)])
def test_changed_scores(kv, block, heads, d, group, scores, dtype):  # noqa: F811
    """Single tokens and ragged prompts, windows, rows of negative position, both ways to look."""
    print(f"scores {block} {heads} {d} {group} {scores} {dtype}", flush=True)
    rng = np.random.default_rng(d + group)
    hq = heads * group
    scores = dict(scores)
    if scores.get("slopes"):
        scores["slopes"] = _slopes(hq)
    lens = [1, 0, 15, 16, 33, 64, 65, 190]
    c, o, table = _filled_cache(kv, rng, lens, heads, d, block)
    ones = [1] * len(lens)
    for spread in (1.0, 6.0):
        _check(kv, c, o, table, lens, ones, hq, dtype, rng, offsets=False, spread=spread, **scores)
    counts = [1, 3, 0, 16, 40, 1, 65, 100]
    for more in (dict(), dict(window=21), dict(causal=False), dict(causal=False, window=30, scale=0.3)):
        _check(kv, c, o, table, lens, counts, hq, dtype, rng, spread=3.0, **more, **scores)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("d,scores", itertools.product((64, 96, 128, 256), [dict(), *SCORES]), ids=str)
def test_tiles_of_many_rows(kv, d, scores, dtype):  # noqa: F811
    """Prompts of hundreds of rows over thousands of tokens, in the kernel of 128 rows a workgroup: documents,
    a prefix, a window, and weights of every size."""
    print(f"many {d} {scores} {dtype}", flush=True)
    rng = np.random.default_rng(d)
    heads, hq = 1, 6
    scores = dict(scores)
    if scores.get("slopes"):
        scores["slopes"] = _slopes(hq)
    lens, counts = [3100, 1500], [900, 1300]
    c, o, table = _filled_cache(kv, rng, lens, heads, d, 16)
    cuts = [np.sort(rng.integers(0, n, 6)) for n in lens]
    first = np.concatenate([[max([0, *[x for x in cut if x <= p]]) for p in range(n - m, n)]
                            for n, m, cut in zip(lens, counts, cuts)])
    spread = 1.0 if not scores else 4.0
    for more in (dict(), dict(first=first), dict(prefix=[2800, 450]), dict(first=first, prefix=[3100, 300], window=1300),
                 dict(causal=False, window=1200)):
        if scores or more:
            _many(c, counts, hq, table, more.get("window", 0))
            _check(kv, c, o, table, lens, counts, hq, dtype, rng, spread=spread, **more, **scores)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("block,heads,d,group", [(16, 2, 128, 2), (32, 1, 64, 4), (64, 1, 112, 1)])
def test_documents_and_prefixes(kv, block, heads, d, group, dtype):  # noqa: F811
    """Rows that see nothing, bounds outside the sequence, one token, and everything."""
    print(f"masks {block} {heads} {d} {group} {dtype}", flush=True)
    rng = np.random.default_rng(block)
    lens, counts = [150, 70, 5, 33, 0, 200, 40], [150, 1, 9, 0, 3, 77, 2]
    hq, rows = heads * group, sum(counts)
    c, o, table = _filled_cache(kv, rng, lens, heads, d, block)
    firsts = [rng.integers(-5, 210, rows), np.full(rows, 2 ** 31 - 1), np.full(rows, -2 ** 31),
              np.concatenate([np.arange(n - m, n) for n, m in zip(lens, counts)])]
    prefixes = [[0, 70, 3, 10, 5, 150, -7], [2 ** 31 - 1] * 7, [-2 ** 31] * 7]
    for first, prefix, window in itertools.product([None, *firsts], [None, *prefixes], (0, 31)):
        if first is None and prefix is None:
            continue
        _check(kv, c, o, table, lens, counts, hq, dtype, rng, first=first, prefix=prefix, window=window)
    _check(kv, c, o, table, lens, counts, hq, dtype, rng, first=firsts[0], causal=False)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("block,heads,d,group", [(16, 2, 128, 2), (32, 1, 64, 8), (64, 2, 80, 1), (16, 1, 256, 3)])
def test_common_pages(kv, block, heads, d, group, dtype):  # noqa: F811
    """Groups of every kind: nothing in common, everything, fronts that end inside the rows, sequences
    shorter than the front, empty ones; one token each, and ragged rows."""
    print(f"shared {block} {heads} {d} {group} {dtype}", flush=True)
    rng = np.random.default_rng(block + d)
    hq = heads * group
    lens = [300, 257, 290, 256, 40, 0, 33, 500, 12, 130, 128, 129]
    c, o, table = _filled_cache(kv, rng, lens, heads, d, block)
    cap = table.shape[1]
    ones = [1] * 12
    counts = [1, 30, 0, 256, 5, 0, 33, 200, 3, 1, 128, 129]
    for shared in ([256 // block], [0], [cap], [1, 128 // block], [5, 0, -3, cap + 9], [2] * 6, [cap] * 12):
        _check(kv, c, o, table, lens, ones, hq, dtype, rng, offsets=False, shared=shared)
        _check(kv, c, o, table, lens, counts, hq, dtype, rng, shared=shared)
    _check(kv, c, o, table, lens, counts, hq, dtype, rng, shared=[4, 2], window=50)
    _check(kv, c, o, table, lens, counts, hq, dtype, rng, shared=[4, 2], causal=False)
    first, prefix = rng.integers(0, 260, sum(counts)), rng.integers(0, 300, 12)
    _check(kv, c, o, table, lens, counts, hq, dtype, rng, shared=[4, 2, 3], first=first, prefix=prefix)
    _check(kv, c, o, table, lens, counts, hq, dtype, rng, shared=[4, 2], softcap=8.0, slopes=_slopes(hq), window=200,
           spread=3.0)
    none = np.full_like(table, -1)
    _check(kv, c, o, none, lens, counts, hq, dtype, rng, shared=[4, 2])


@pytest.mark.parametrize("dtype", HALVES)
def test_rule_of_common_pages(kv, dtype):  # noqa: F811
    """The same answers whichever way the rule takes, on both sides of it."""
    rng = np.random.default_rng(6)
    lens = [2100 + n for n in range(24)]
    c, o, table = _filled_cache(kv, rng, lens, 1, 64, 16)
    table[:, :130] = table[0, :130]
    desc = kv._desc(c)
    assert not kv._front_pays(desc, 24, 4, 24, 1, 2144) and not kv._front_pays(desc, 2400, 4, 24, 1, 1 << 20)
    assert kv._front_pays(desc, 24, 4, 24, 1, 1 << 20) and not kv._front_pays(desc, 24, 4, 24, 24, 1 << 20)
    for counts in ([1] * 24, [5, 0, 30] * 8):
        _check(kv, c, o, table, lens, counts, 4, dtype, rng, shared=[130])
        _check(kv, c, o, table, lens, counts, 4, dtype, rng, shared=[130, 100], softcap=9.0, window=900)
    # a table wide enough for it, most of which is empty
    wide = np.full((24, 1 << 16), -1)
    wide[:, :table.shape[1]] = table
    _check(kv, c, o, wide, lens, [1] * 24, 4, dtype, rng, shared=[130])


@pytest.mark.parametrize("dtype", HALVES)
def test_common_pages_of_many_rows(kv, dtype):  # noqa: F811
    """Fronts long enough to be split among workgroups, and rows for the tiles of 128."""
    rng = np.random.default_rng(5)
    each, front, block = 6, 2048, 16
    lens = [front + n for n in (1, 100, 33, 300, 7, 64, 500, 20, 1, 90, 200, 31)]
    c, o, table = _filled_cache(kv, rng, lens, 1, 64, block)
    for g in range(2):
        table[each * g:each * (g + 1), :front // block] = table[each * g, :front // block]
    shared = [front // block, front // block - 5]
    _check(kv, c, o, table, lens, [1] * 12, 8, dtype, rng, offsets=False, shared=shared)
    counts = [1, 100, 33, 300, 7, 64, 500, 20, 1, 90, 200, 31]
    _many(c, counts, 8, table)
    _check(kv, c, o, table, lens, counts, 8, dtype, rng, shared=shared)
    _check(kv, c, o, table, lens, counts, 8, dtype, rng, shared=shared, softcap=30.0, spread=3.0)
    # the same pages, not called common: the same up to the order of sums
    q = torch.from_numpy(rng.standard_normal((12, 8, 64))).to(dtype).cuda()
    a = kv.attention(q, c, _i32(table), _i32(lens), shared=_i32(shared)).double()
    b = kv.attention(q, c, _i32(table), _i32(lens)).double()
    # weights in two terms err by 2^-17 each, results once more by half a unit in the last place of both
    assert float((a - b).abs().max()) <= 2 * HALF_ULP[dtype] * float(b.abs().max()) + 2.0 ** -14


def test_unseen_tokens_do_not_reach_a_row(kv):  # noqa: F811
    """NaN and infinities where masks hide them: before a document, after a position, past a front."""
    rng = np.random.default_rng(8)
    lens, counts = [100, 100, 37, 90], [60, 1, 37, 30]
    c, o, table = _filled_cache(kv, rng, lens, 2, 64, 16)
    for b in (1, 2, 3):
        table[b, :2] = table[0, :2]
    for b, n in enumerate(lens):  # slots past the length
        o.k[table[b][n // 16], :, n % 16:] = 127
        o.v[table[b][n // 16], :, n % 16:] = 255
    o.v[table[0][1], 0, 5, 7] = 127        # token 21 of the front
    o.k[table[0][85 // 16], 1, 85 % 16, 3] = 127
    o.v[table[3][50 // 16], 0, 50 % 16, 9] = 255
    c.k.copy_(torch.from_numpy(o.k))
    c.v.copy_(torch.from_numpy(o.v.swapaxes(2, 3).copy()))
    rows = sum(counts)
    firsts = [None, np.full(rows, 22), rng.integers(0, 60, rows), np.full(rows, 86)]
    for dtype, first, shared in itertools.product(HALVES, firsts, (None, [2], [1, 2])):
        for more in (dict(), dict(softcap=10.0), dict(slopes=_slopes(4)), dict(window=20), dict(prefix=[86, 0, 30, 60])):
            _check(kv, c, o, table, lens, counts, 4, dtype, rng, first=first, shared=shared, **more)


def test_ordered_calls_captured_and_on_streams(kv):  # noqa: F811
    """Calls whose row tiles are put in order: replayed under other documents and lengths, and two at once."""
    rng = np.random.default_rng(18)
    counts, lens = [4000, 300, 4000], [4000, 900, 4090]
    c, o, table = _filled_cache(kv, rng, lens, 4, 64, 16)
    rows, hq = sum(counts), 16
    assert rows * hq * table.shape[1] * 16 > 1 << 28 and rows * 4 // 128 * 4 >= 1024
    q = torch.from_numpy(rng.standard_normal((rows, hq, 64))).to(torch.bfloat16).cuda()
    table, held, off = _i32(table), _i32(lens), _offsets(counts)
    first = _i32(rng.integers(0, 4000, rows))

    def call():
        return kv.attention(q, c, table, held, off, first=first, softcap=20.0)
    streams = [torch.cuda.Stream() for _ in range(2)]
    alone = call()
    torch.cuda.synchronize()
    both = []
    for s in streams:
        with torch.cuda.stream(s):
            both.append([call() for _ in range(3)])
    torch.cuda.synchronize()
    for x in (*both[0], *both[1]):
        assert torch.equal(x.view(torch.int16), alone.view(torch.int16))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got.view(torch.int16), call().view(torch.int16)), i
        held -= 50
        first.copy_(_i32(np.sort(rng.integers(0, 4000 >> i, rows))))


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("many", [False, True])
def test_an_infinite_query_stays_in_its_row(kv, many, dtype):  # noqa: F811
    """Infinities and NaN in some queries, under caps and scales of every size: the other rows are as without."""
    rng = np.random.default_rng(12)
    lens, counts = ([2500], [700]) if many else ([100, 40], [9, 1])
    c, o, table = _filled_cache(kv, rng, lens, 1, 64, 16)
    rows, hq = sum(counts), 12
    q = torch.from_numpy(rng.standard_normal((rows, hq, 64))).to(dtype).cuda()
    bad = q.clone()
    bad[1, 3, 5], bad[4, 0, 0], bad[4, 7, 1] = float("inf"), float("-inf"), float("nan")
    left = torch.ones((rows, hq), dtype=torch.bool, device="cuda")
    left[1, 3] = left[4, 0] = left[4, 7] = False
    if many:
        _many(c, counts, hq, table)
    for scale, cap, slopes in itertools.product((None, 1e-13, 1e-30, 1e-37), (0.5, 30.0, 1000.0, 1e29), (None, True)):
        more = dict(scale=scale, softcap=cap, slopes=slopes and torch.tensor(_slopes(hq), device="cuda"))
        a = kv.attention(q, c, _i32(table), _i32(lens), _offsets(counts), **more)
        b = kv.attention(bad, c, _i32(table), _i32(lens), _offsets(counts), **more)
        assert bool(torch.isfinite(b[left]).all()), (scale, cap)
        # where all are small they take the shorter way together; two ways differ by less than a result's rounding
        tol = 4 * HALF_ULP[dtype] * float(a.double().abs().max())
        assert float((a[left].double() - b[left].double()).abs().max()) <= tol, (scale, cap)


def test_many_rows_that_hide_nan(kv):  # noqa: F811
    """The same in tiles of 128 rows."""
    rng = np.random.default_rng(9)
    lens, counts, hq = [1800, 1500], [500, 600], 12
    c, o, table = _filled_cache(kv, rng, lens, 1, 64, 32)
    table[1, :20] = table[0, :20]
    o.v[table[0][10], 0, 3, 7] = 127   # token 323 of both
    o.v[table[1][1200 // 32], 0, 1200 % 32, 60] = 255
    o.k[table[0][1700 // 32], 0, 1700 % 32, 1] = 127
    c.k.copy_(torch.from_numpy(o.k))
    c.v.copy_(torch.from_numpy(o.v.swapaxes(2, 3).copy()))
    for first, shared in itertools.product((None, np.repeat([324, 100], counts)), (None, [20])):
        for more in (dict(prefix=[0, 0]), dict(softcap=10.0), dict(slopes=_slopes(hq)), dict(window=1200)):
            if first is None and shared is None and "window" in more:
                continue
            _many(c, counts, hq, table, more.get("window", 0))
            _check(kv, c, o, table, lens, counts, hq, torch.bfloat16, rng, first=first, shared=shared, **more)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("scores", [dict(), dict(softcap=20.0), dict(slopes=True)], ids=str)
def test_row_tiles_in_order_of_their_work(kv, scores, dtype):  # noqa: F811
    """Thousands of rows under a table for thousands of tokens, whose row tiles run in another order: what the
    same call gives under a narrow table, and the definition. Rows of no sequence and empty rows among them."""
    rng = np.random.default_rng(17)
    hq, width = 16, 32
    scores = dict(scores)
    if scores.get("slopes"):
        scores["slopes"] = _slopes(hq)
    counts = [500, 0, 1, 300, 128, 33, 500] + [int(x) for x in rng.integers(200, 480, 26)]
    lens = [int(rng.integers(n, 513)) if n else 0 for n in counts]
    c, o, table = _filled_cache(kv, rng, lens, 4, 64, 16)
    narrow = np.full((len(lens), width), -1, np.int32)
    narrow[:, :table.shape[1]] = table[:, :width]
    wide = np.full((len(lens), 160), -1, np.int32)
    wide[:, :width] = narrow
    rows = sum(counts)
    # past 2^28 pairs under the wide table and not under the narrow one, and four workgroups a CU in both
    assert rows * hq * 160 * 16 > 1 << 28 > rows * hq * width * 16 and rows * 4 // 128 * 4 >= 1024
    first = np.concatenate([np.maximum.accumulate(rng.integers(0, 2, n) * (np.arange(n) + m - n)) if i % 3 else
                            rng.integers(0, 520, n) for i, (n, m) in enumerate(zip(counts, lens))]).astype(np.int64)
    q = torch.from_numpy(rng.standard_normal((rows + 300, hq, 64))).to(dtype).cuda()
    args = {k: torch.tensor(v, dtype=torch.float32, device="cuda") if k == "slopes" else v for k, v in scores.items()}
    for begin in (first, np.zeros_like(first)):
        more = dict(first=_i32(np.concatenate([begin, np.zeros(300, np.int64)])), **args)
        a, al = kv.attention(q, c, _i32(narrow), _i32(lens), _offsets(counts), return_lse=True, **more)
        b, bl = kv.attention(q, c, _i32(wide), _i32(lens), _offsets(counts), return_lse=True, **more)
        assert torch.equal(a.view(torch.int16), b.view(torch.int16)) and torch.equal(al, bl)
        assert not bool(b[rows:].any())
    some = slice(0, 7)
    _check(kv, c, o, wide[some], lens[some], counts[some], hq, dtype, rng, first=first[:sum(counts[some])], **scores)


def test_values_under_scales_far_apart(kv):  # noqa: F811
    """V scales from 2^-30 to 2^7 in and past the common pages, scores of hundreds."""
    rng = np.random.default_rng(7)
    c, o, table = _filled_cache(kv, rng, [190, 200], 1, 64, 16, grow=30.0)
    table[1, :6] = table[0, :6]
    for p in range(o.vs.shape[0]):
        o.vs[p] = c.v_scale[p] = 2.0 ** int(rng.integers(-30, 8))
    for counts in ([1, 1], [90, 3], [190, 200]):
        for more in (dict(shared=[6]), dict(shared=[6], softcap=30.0, scale=0.5), dict(slopes=_slopes(2), scale=1.0),
                     dict(first=[40] * sum(counts), shared=[3, 9])):
            _check(kv, c, o, table, [190, 200], counts, 2, torch.bfloat16, rng, **more)


def test_rows_of_no_sequence(kv):  # noqa: F811
    """A padded batch: rows before the first and past the last are 0, their log-sum -inf."""
    rng = np.random.default_rng(10)
    lens = [100, 70, 90, 33]
    c, o, table = _filled_cache(kv, rng, lens, 2, 64, 16)
    for n in (4, 700, 10500):
        if n == 10500:
            _many(c, [n] * 4, 4, table)
        q = torch.from_numpy(rng.standard_normal((4 * n + 20, 4, 64))).to(torch.bfloat16).cuda()
        inner = _i32([3, 3 + n, 3 + n, 3 + 3 * n, 3 + 4 * n])
        for more in (dict(softcap=9.0), dict(shared=_i32([2])), dict(shared=_i32([2, 1])),
                     dict(first=_i32(np.zeros(len(q))))):
            out, lse = kv.attention(q, c, _i32(table), _i32(lens), inner, return_lse=True, **more)
            m = {k: v[3:3 + 4 * n] if k == "first" else v for k, v in more.items()}
            want = kv.attention(q[3:3 + 4 * n], c, _i32(table), _i32(lens), inner - 3, return_lse=True, **m)
            assert torch.equal(out[3:3 + 4 * n], want[0]) and torch.equal(lse[3:3 + 4 * n], want[1])
            for part in (slice(0, 3), slice(3 + 4 * n, None)):
                assert not out[part].any() and bool((lse[part] == float("-inf")).all())
        # a sequence whose rows are not all there: it has no results, nor has its group
        past = _i32([0, n, n, 3 * n, 5 * n + 20])
        for shared, good in ((None, 3 * n), ([1, 1], n), ([1], 0)):
            more = dict(softcap=9.0) if shared is None else dict(shared=_i32(shared))
            out, lse = kv.attention(q, c, _i32(table), _i32(lens), past, return_lse=True, **more)
            assert not out[good:].any() and bool((lse[good:] == float("-inf")).all())
            if good:
                assert torch.isfinite(lse[:good][-1]).all() and out[:good][-1].any()
        nothing = kv.attention(q, c, _i32(table[:0]), _i32([]), _i32([0]), return_lse=True, softcap=1.0)
        assert not nothing[0].any() and bool((nothing[1] == float("-inf")).all())


def test_strides_and_positions_past_the_table(kv):  # noqa: F811
    rng = np.random.default_rng(11)
    lens = [100, 64]
    c, o, table = _filled_cache(kv, rng, lens, 2, 64, 16)
    wide = torch.from_numpy(rng.standard_normal((30, 12, 64))).to(torch.bfloat16).cuda()
    off, more = _i32([0, 20, 30]), dict(softcap=9.0, shared=_i32([1]))
    want = kv.attention(wide[:, :4].contiguous(), c, _i32(table), _i32(lens), off, **more)
    assert torch.equal(kv.attention(wide[:, :4], c, _i32(table), _i32(lens), off, **more), want)
    firsts = torch.zeros((60,), dtype=torch.int32, device="cuda")
    assert torch.equal(kv.attention(wide[:, :4], c, _i32(table), _i32(lens), off, first=firsts[::2], **more), want)
    # more tokens than the table's row holds
    n = table.shape[1] * 16
    for more in (dict(slopes=_slopes(4)), dict(shared=[3]), dict(first=[50, n + 5])):
        _check(kv, c, o, table, [n + 9, n + 40], [1, 1], 4, torch.bfloat16, rng, **more)


def test_answers_together(kv):  # noqa: F811
    """A prompt, forked, its answers continued a token at a time over pages in common, and the next
    tokens drawn: each step as the same sequences give it with pages of their own."""
    from perm_amd import kvpages, sampling
    g = torch.Generator(device="cuda").manual_seed(0)
    heads, hq, d, block, n, answers, vocab = 2, 8, 64, 16, 133, 5, 500
    pages = 64
    cache, own = kv.new(pages, heads, d, block), kv.new(answers * 12, heads, d, block)
    refs, table = kvpages.new(pages), torch.full((answers, 12), -1, dtype=torch.int32, device="cuda")
    own_table = torch.arange(answers * 12, dtype=torch.int32, device="cuda").view(answers, 12)
    embed = torch.randn((vocab, (hq + 2 * heads) * d), generator=g, device="cuda").to(torch.bfloat16)
    out_w = torch.randn((vocab, hq * d), generator=g, device="cuda") * 0.3
    prompt = torch.randint(0, vocab, (n,), generator=g, device="cuda")
    x = embed[prompt].view(n, -1, d)
    zero, lens = _i32([0] * answers), _i32([n] + [0] * (answers - 1))
    kvpages.grow(refs, table, zero, lens, block)
    off = _i32([0] + [n] * answers)
    kv.write(cache, x[:, hq:hq + heads], x[:, hq + heads:], table, zero, off)
    kvpages.fork(refs, table, lens, zero[1:], _i32(range(1, answers)), block)
    for b in range(answers):
        kv.write(own, x[:, hq:hq + heads], x[:, hq + heads:], own_table[b:b + 1], _i32([0]), _i32([0, n]))
    lens = _i32([n] * answers)
    shared = _i32([n // block])
    token = torch.full((answers,), 7, device="cuda")
    seen = []
    for step in range(40):
        x = embed[token].view(answers, -1, d)
        src, dst, missing = kvpages.grow(refs, table, lens, 1, block)
        kvpages.copy(cache, src, dst)
        if step == 20:
            src, dst, used = kvpages.compact(refs, table)
            kvpages.copy(cache, src, dst)
            assert int(used) == n // block + answers * (-(-(n + 21) // block) - n // block)
        assert not missing.any()
        for c, t in ((cache, table), (own, own_table)):
            kv.write(c, x[:, hq:hq + heads], x[:, hq + heads:], t, lens)
        lens = lens + 1
        q = x[:, :hq]
        a, la = kv.attention(q, cache, table, lens, shared=shared, return_lse=True)
        b, lb = kv.attention(q, own, own_table, lens, return_lse=True)
        assert float((la - lb).abs().max()) <= 2.0 ** -17 * (1 + float(lb.abs().max()))
        assert float((a.double() - b.double()).abs().max()) <= 2.0 ** -8 * float(b.abs().max()) + 2.0 ** -14
        u = torch.rand((answers,), generator=g, device="cuda")
        token = sampling.sample(b.reshape(answers, -1).float() @ out_w.t(), u, temperature=0.9, top_k=100, top_p=0.95)
        assert int(token.min()) >= 0
        seen.append(token.tolist())
    assert len({tuple(s[b] for s in seen) for b in range(answers)}) == answers
    kvpages.free(refs, table)
    assert not refs.any()


def test_graph_replays(kv):  # noqa: F811
    """Common pages in splits with their join, changed scores and masks in one graph, with new contents."""
    rng = np.random.default_rng(12)
    lens = [2300, 2200, 2100, 2050]
    c, o, table = _filled_cache(kv, rng, lens, 1, 64, 16)
    table[1:, :128] = table[0, :128]
    t, held, shared, first = _i32(table), _i32(lens), _i32([128]), _i32([0, 5, 9, 1000])
    q = torch.from_numpy(rng.standard_normal((4, 4, 64))).to(torch.bfloat16).cuda()
    many = torch.from_numpy(rng.standard_normal((2400, 4, 64))).to(torch.bfloat16).cuda()
    _many(c, [600] * 4, 4, table)
    off, slopes = _i32([0, 600, 1200, 1800, 2400]), torch.tensor(_slopes(4), device="cuda")

    def step():
        return (*kv.attention(q, c, t, held, shared=shared, return_lse=True),
                *kv.attention(many, c, t, held, off, shared=shared, softcap=20.0, return_lse=True),
                kv.attention(q, c, t, held, first=first, slopes=slopes),
                kv.attention(many, c, t, held, off, prefix=held))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        got = [y.clone() for y in outs]
        for a, b in zip(got, step()):
            assert torch.equal(a, b), i
        q.copy_(torch.from_numpy(rng.standard_normal(q.shape)))
        many.copy_(torch.from_numpy(rng.standard_normal(many.shape)))
        held.sub_(40)
        shared.sub_(30)
        first.add_(100)


def test_refusals(kv, monkeypatch):  # noqa: F811
    c = kv.new(4, 2, 64, 16)
    q = torch.zeros((4, 4, 64), dtype=torch.bfloat16, device="cuda")
    t, n = _i32([[0], [1], [2], [3]]), _i32([16] * 4)
    ok = torch.ones(4, device="cuda")
    for bad in (dict(softcap=-1.0), dict(softcap=float("nan")), dict(softcap=float("inf")), dict(slopes=ok[:2]),
                dict(slopes=ok.double()), dict(slopes=[1.0] * 4), dict(slopes=ok.cpu()), dict(first=n[:3]),
                dict(prefix=n[:3]), dict(shared=n[:3]), dict(shared=n[:0]), dict(shared=3), dict(first=n.cpu())):
        with pytest.raises(ValueError):
            kv.attention(q, c, t, n, **bad)
    for bad in (dict(first=n.long()), dict(prefix=ok), dict(shared=t)):
        with pytest.raises(IndexError):
            kv.attention(q, c, t, n, **bad)
    y = q.clone().requires_grad_()
    with pytest.raises(NotImplementedError):
        kv.attention(y, c, t, n, softcap=3.0).sum().backward()
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    with pytest.raises(ValueError, match="current device"):
        kv.attention(q, c, t, n, softcap=3.0)
