"""The pages of a cache, forked, grown, copied, given back and compacted: every number and every
code as the oracle's, which keeps the books one page at a time."""
import numpy as np
import pytest
import torch

from oracle import pages_oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mods():
    from perm_amd import kvcache, kvpages
    return kvcache, kvpages


def _i32(v, shape=None):
    a = np.asarray(v, np.int32)
    return torch.tensor(a if shape is None else a.reshape(shape), dtype=torch.int32, device="cuda")


def _same(o, refs, table):
    assert np.array_equal(refs.cpu().numpy(), np.asarray(o.refs)), "refs"
    assert np.array_equal(table.cpu().numpy(), np.asarray(o.table).reshape(tuple(table.shape))), "table"


def _books(rng, pages, batch, max_pages, lens, block, spread=True):
    """Rows that hold lens[b] tokens on pages anywhere."""
    order = rng.permutation(pages) if spread else np.arange(pages)
    table, refs, at = np.full((batch, max_pages), -1), np.zeros(pages, int), 0
    for b in range(batch):
        n = -(-int(lens[b]) // block)
        table[b, :n] = order[at:at + n]
        at += n
    refs[table[table >= 0]] = 1
    return refs, table


@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("pages,batch,cap", [(40, 6, 4), (2000, 40, 12), (5000, 300, 9), (70001, 33, 300)])
def test_a_life_of_many_answers(mods, pages, batch, cap, block):
    """Random forks, growths, ends and compactions, with pages running short at times."""
    _, kp = mods
    print(f"life {pages} {batch} {cap} {block}", flush=True)
    rng = np.random.default_rng(pages + block)
    refs, table = kp.new(pages), torch.full((batch, cap), -1, dtype=torch.int32, device="cuda")
    o = O.Books([0] * pages, [[-1] * cap] * batch, block)
    lens = np.zeros(batch, int)
    alive = np.zeros(batch, bool)
    short = 0
    for step in range(30):
        what = step % 4
        if what == 0:
            begin = np.flatnonzero(~alive)[: batch // 3 + 1]
            alive[begin] = True
            lens[begin] = 0
            new = np.where(np.isin(np.arange(batch), begin), rng.integers(0, cap * block + 1, batch), 0)
        elif what == 1:
            mums = np.flatnonzero(alive)
            kids = np.flatnonzero(~alive)[: batch // 4]
            if mums.size and kids.size:
                mums = rng.choice(mums, kids.size)
                kp.fork(refs, table, _i32(lens), _i32(mums), _i32(kids), block)
                o.fork(lens, mums, kids)
                lens[kids] = lens[mums]
                alive[kids] = True
                _same(o, refs, table)
            new = np.where(alive, rng.integers(0, 3, batch), 0)
        else:
            new = np.where(alive, rng.integers(-1, 2 * block, batch), 0)
        src, dst, missing = kp.grow(refs, table, _i32(lens), _i32(new), block)
        want = o.grow(lens, new)
        for got, w, name in zip((src, dst, missing), want, ("src", "dst", "missing")):
            assert got.cpu().tolist() == w, (step, name)
        _same(o, refs, table)
        done = np.asarray(want[2]) == 0
        short += int((~done).sum())
        lens = lens + np.where(done, np.maximum(new, 0), 0)
        end = np.flatnonzero(alive & ((rng.random(batch) < 0.3) | ~done))
        kp.free(refs, table, _i32(end))
        o.free(end.tolist())
        alive[end] = False
        _same(o, refs, table)
        if what == 3:
            src, dst, used = kp.compact(refs, table)
            want = o.compact()
            assert src.cpu().tolist() == want[0] and dst.cpu().tolist() == want[1]
            assert used.cpu().tolist() == [want[2]]
            _same(o, refs, table)
    assert short or pages > 60000
    kp.free(refs, table)
    assert not refs.any() and bool((table == -1).all())


def test_last_pages_become_their_own(mods):
    """A prompt forked three ways and continued by all four: what each reads back is its own."""
    kv, kp = mods
    g = torch.Generator(device="cuda").manual_seed(0)
    heads, d, block, n = 2, 64, 16, 37
    cache = kv.new(40, heads, d, block)
    refs, table = kp.new(40), torch.full((4, 6), -1, dtype=torch.int32, device="cuda")
    lens = _i32([n, 0, 0, 0])
    first = torch.randn((n, heads, d), generator=g, device="cuda").to(torch.bfloat16)
    src, dst, missing = kp.grow(refs, table, _i32([0] * 4), lens, block)
    assert not missing.any() and bool((src == -1).all())
    kv.write(cache, first, first, table, _i32([0] * 4), _i32([0, n, n, n, n]))
    kp.fork(refs, table, lens, _i32([0, 0, 0]), _i32([1, 2, 3]), block)
    lens = _i32([n] * 4)
    kept = kv.read(cache, table[:1], _i32([0, n]), n, torch.float32)
    for step in range(20):
        src, dst, missing = kp.grow(refs, table, lens, 1, block)
        assert not missing.any()
        assert int((src >= 0).sum()) == (4 if step == 0 else 0)
        kp.copy(cache, src, dst)
        x = torch.randn((4, heads, d), generator=g, device="cuda").to(torch.bfloat16)
        kv.write(cache, x, x, table, lens)
        lens += 1
    assert int(refs.sum()) == int((table >= 0).sum())
    m = n + 20
    k, v = kv.read(cache, table, _i32([0, m, 2 * m, 3 * m, 4 * m]), 4 * m, torch.float32)
    # whole pages are shared still, the last one of the prompt is each one's own
    assert torch.equal(table[:, :2], table[:1, :2].expand(4, 2))
    assert len(set(table[:, 2:4].flatten().tolist())) == 8
    for b in range(4):
        for got, want in ((k, kept[0]), (v, kept[1])):
            # 32 tokens on pages nobody wrote to since; those of the third may have moved to a larger scale
            assert torch.equal(got[b * m:b * m + 32], want[:32])
            # a code moved to a scale s is rounded once more, by half a step: 2^-4 of itself, or of
            # the least normal 2^-6 s; s is at most 2^3 times as large here
            assert bool(((got[b * m + 32:b * m + n] - want[32:]).abs()
                         <= 2.0 ** -4 * want[32:].abs() + 2.0 ** -10).all())
    assert not torch.equal(k[m + n:2 * m], k[2 * m + n:3 * m])


@pytest.mark.parametrize("heads,d,block", [(1, 16, 16), (2, 80, 32), (8, 128, 16), (3, 256, 128), (5, 64, 64)])
def test_copy(mods, heads, d, block):
    """Within a cache, into another one, pairs that name no page."""
    kv, kp = mods
    print(f"copy {heads} {d} {block}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(d)

    def filled(pages):
        c = kv.new(pages, heads, d, block)
        for t in (c.k, c.v):
            t.copy_(torch.randint(0, 256, t.shape, generator=g, device="cuda", dtype=torch.uint8))
        for t in (c.k_scale, c.v_scale):
            t.copy_(torch.rand(t.shape, generator=g, device="cuda"))
        return c
    c, other = filled(9), filled(4)
    was, was_other = [t.clone() for t in c], [t.clone() for t in other]
    kp.copy(c, _i32([0, -1, 8, 3, 9, 2, 1 << 30]), _i32([5, 6, 7, -1, 1, 9, 4]))
    for t, w in zip(c, was):
        w[5], w[7] = w[0], w[8]
        assert torch.equal(t, w)
    kp.copy(c, _i32([8, 0, 1]), _i32([0, 3, 4]), into=other)
    for t, w, a in zip(other, was_other, was):
        w[0], w[3] = a[8], a[0]
        assert torch.equal(t, w)
    kp.copy(c, _i32([]), _i32([]))
    for t, w in zip(c, was):
        assert torch.equal(t, w)


@pytest.mark.parametrize("pages", [1, 2, 3, 63, 1023, 1024, 1025, 2048, 40000])
def test_compact_of_every_kind(mods, pages):
    _, kp = mods
    rng = np.random.default_rng(pages)
    for used in sorted({0, 1, pages // 2, pages - 1, pages}):
        for spread in (True, False):
            refs, table = _books(rng, pages, 3, max(1, used), [16 * used, 0, 0], 16, spread)
            table[2, : used // 2] = table[0, : used // 2]
            refs[table[2][table[2] >= 0]] += 1
            o = O.Books(refs, table, 16)
            r, t = _i32(refs), _i32(table)
            src, dst, n = kp.compact(r, t)
            want = o.compact()
            assert src.cpu().tolist() == want[0] and dst.cpu().tolist() == want[1] and n.item() == want[2]
            _same(o, r, t)


def test_entries_that_are_no_page(mods):
    """Books with numbers outside the cache: nothing outside is touched."""
    _, kp = mods
    refs = _i32([2, 1, 0, 0, 1])
    table = _i32([[0, 9, -7, 1], [0, 1 << 30, -1, 4], [-1, -1, -1, -1], [-1, -1, -1, -1]])
    lens = _i32([64, 20, -5, 0])
    o = O.Books(refs.tolist(), table.tolist(), 16)
    a, b = [0, 1, 7, -1, 3], [2, 3, 0, 1, 3]
    kp.fork(refs, table, lens, _i32(a), _i32(b), 16)
    o.fork(lens.tolist(), a, b)
    _same(o, refs, table)
    filled, new = [30, 0, 100, 5], [40, 33, 1, 20]
    got = kp.grow(refs, table, _i32(filled), _i32(new), 16)
    assert [t.cpu().tolist() for t in got] == list(o.grow(filled, new))
    _same(o, refs, table)
    kp.free(refs, table, _i32([3, 3, -1, 4, 0, 3]))
    o.free([3, -1, 4, 0])
    _same(o, refs, table)
    got = kp.grow(refs, table, _i32([0, 2 ** 31 - 1, 2 ** 31 - 20, -9]), 2 ** 31 - 1, 16)
    want = o.grow([0, 2 ** 31 - 1, 2 ** 31 - 20, -9], [2 ** 31 - 1] * 4)
    assert [t.cpu().tolist() for t in got] == list(want)
    _same(o, refs, table)


def test_graph_replays(mods):
    kv, kp = mods
    cache = kv.new(64, 2, 64, 16)
    refs, table = kp.new(64), torch.full((6, 8), -1, dtype=torch.int32, device="cuda")
    zero, lens = _i32([0] * 6), _i32([50, 50, 0, 0, 0, 0])
    kp.grow(refs, table, zero, lens, 16)
    mums, kids, held, new = _i32([0, 0, 1, 1]), _i32([2, 3, 4, 5]), _i32([50] * 6), _i32([0, 0, 1, 20, 1, 1])

    def step():
        kp.free(refs, table, kids)
        kp.fork(refs, table, lens, mums, kids, 16)
        src, dst, missing = kp.grow(refs, table, held, new, 16)
        kp.copy(cache, src, dst)
        return src, dst, missing
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
        got = [t.clone() for t in (*outs, refs, table)]
        eager = [*step(), refs, table]
        for a, b in zip(got, eager):
            assert torch.equal(a, b), i
        lens[:2] += 1
        held += 1
        new[2] += 3


def test_books_on_two_streams(mods):
    """Two pairs of books at once, each on a stream of its own."""
    _, kp = mods
    rng = np.random.default_rng(4)
    streams, runs = [torch.cuda.Stream() for _ in range(2)], []
    inputs = [[_i32(rng.integers(0, 300, 40)) for _ in range(6)] for _ in streams]
    rows = [_i32(rng.permutation(40)[:9]) for _ in range(6)]
    torch.cuda.synchronize()

    def run(new):
        refs, table = kp.new(3000), torch.full((40, 130), -1, dtype=torch.int32, device="cuda")
        lens, outs = torch.zeros(40, dtype=torch.int32, device="cuda"), []
        for n, r in zip(new, rows):
            outs += kp.grow(refs, table, lens, n, 16)
            lens = lens + n
            kp.free(refs, table, r)
            lens.index_fill_(0, r.long(), 0)
            outs += kp.compact(refs, table)
        return [refs, table, *outs]
    for s, new in zip(streams, inputs):
        with torch.cuda.stream(s):
            runs.append([run(new) for _ in range(2)])
    torch.cuda.synchronize()
    for got, new in zip(runs, inputs):
        for want, *both in zip(run(new), *got):
            assert all(torch.equal(want, t) for t in both)


def test_refusals(mods, monkeypatch):
    kv, kp = mods
    refs, table = kp.new(8), torch.full((2, 4), -1, dtype=torch.int32, device="cuda")
    lens, rows = _i32([0, 0]), _i32([0])
    with pytest.raises(ValueError):
        kp.new(0)
    for bad in (refs.cpu(), refs[::2], None):
        with pytest.raises(ValueError):
            kp.compact(bad, table)
    for bad in (table.cpu(), table.t(), table[:, ::2]):
        with pytest.raises(ValueError):
            kp.free(refs, bad)
    for bad in (refs.long(), table):
        with pytest.raises(IndexError):
            kp.compact(bad, table)
    with pytest.raises(IndexError):
        kp.free(refs, table.long())
    with pytest.raises(ValueError):
        kp.compact(refs, table[:, :0])
    for call in (lambda: kp.fork(refs, table, lens, rows, rows, 8), lambda: kp.grow(refs, table, lens, 1, 48),
                 lambda: kp.fork(refs, table, lens[:1], rows, rows, 16),
                 lambda: kp.fork(refs, table, lens, rows, lens, 16),
                 lambda: kp.grow(refs, table, rows, 1, 16), lambda: kp.grow(refs, table, lens, rows, 16),
                 lambda: kp.grow(refs, table, lens, -1, 16), lambda: kp.grow(refs, table, lens, 2 ** 31, 16)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        kp.grow(refs, table, lens, 1.5, 16)
    a, b = kv.new(4, 2, 64, 16), kv.new(4, 2, 64, 32)
    with pytest.raises(ValueError):
        kp.copy(a, rows, rows, into=b)
    with pytest.raises(ValueError):
        kp.copy(a, rows, lens)
    with pytest.raises(IndexError):
        kp.copy(a, rows.long(), rows.long())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    for call in (lambda: kp.free(refs, table), lambda: kp.copy(a, rows, rows)):
        with pytest.raises(ValueError, match="current device"):
            call()
