"""The operators for several answers at the edges of what their calls allow."""
import numpy as np
import pytest
import torch

from test_gpu_kvcache import _filled_cache, _i32, kv  # noqa: F401
from test_gpu_kvcache_padding import _dirty
from test_gpu_kvcache_tiles import _long
from test_gpu_kvpages import _books, _same
from test_gpu_sampling import DTYPES, _logits
from test_gpu_sampling import _check as _check_tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads", [4, 8])
def test_slopes_that_want_a_gradient(kv, heads):  # noqa: F811
    """Attention depends on its slopes: a backward pass to them alone raises, of results and log-sums."""
    c = kv.new(4, 2, 64, 16)
    t, n = _i32([[0], [1], [2]]), _i32([16] * 3)
    q = torch.ones((3, heads, 64), dtype=torch.bfloat16, device="cuda")
    slopes = torch.ones(heads, device="cuda").requires_grad_()
    plain = kv.attention(q, c, t, n, slopes=slopes.detach(), return_lse=True)
    for want, got in zip(plain, kv.attention(q, c, t, n, slopes=slopes, return_lse=True)):
        assert not want.requires_grad and got.requires_grad and torch.equal(want, got)
        with pytest.raises(NotImplementedError, match="attention"):
            got.float().sum().backward()
    with torch.no_grad():
        assert not kv.attention(q, c, t, n, slopes=slopes).requires_grad


@pytest.mark.parametrize("rows", [0, 3])
@pytest.mark.parametrize("apart", [None, True], ids=["rule", "apart"])
def test_common_pages_of_an_empty_batch(kv, monkeypatch, apart, rows):  # noqa: F811
    """A step without sequences, of any number of groups: what the call without common pages gives."""
    if apart:
        monkeypatch.setattr(kv, "_front_pays", lambda *a: True)
    c = kv.new(4, 2, 64, 16)
    q = torch.ones((rows, 8, 64), dtype=torch.bfloat16, device="cuda")
    table, lens = torch.empty((0, 5), dtype=torch.int32, device="cuda"), _i32([])
    for offsets in (_i32([0]), None) if rows == 0 else (_i32([0]),):
        for groups in (0, 1, 3):
            for more in (dict(), dict(softcap=5.0), dict(window=9)):
                out, lse = kv.attention(q, c, table, lens, offsets, return_lse=True, shared=_i32([1] * groups), **more)
                assert out.shape == q.shape and not out.any() and lse.shape == (rows, 8) and torch.isneginf(lse).all()
    # sequences, but no rows of theirs
    out = kv.attention(q[:0], c, _i32([[0], [1]]), _i32([9, 9]), _i32([0, 0, 0]), shared=_i32([1]))
    assert out.shape == (0, 8, 64)
    with pytest.raises(ValueError, match="groups"):
        kv.attention(q[:0], c, _i32([[0], [1]]), _i32([9, 9]), _i32([0, 0, 0]), shared=_i32([]))


@pytest.mark.parametrize("pages", [1, 2, 3, 2000])
@pytest.mark.parametrize("width", [1, 5])
def test_compaction_under_a_table_of_no_rows(pages, width):
    """Holders that no table names (another's, or none): pages in use move all the same."""
    from perm_amd import kvpages
    table = torch.empty((0, width), dtype=torch.int32, device="cuda")
    for held in ([], [pages - 1], list(range(0, pages, 2))):
        refs = kvpages.new(pages)
        refs[held] = 1
        src, dst, used = kvpages.compact(refs, table)
        n = len(held)
        assert used.tolist() == [n] and refs.tolist() == [1] * n + [0] * (pages - n)
        moved, free = [p for p in held if p >= n], [p for p in range(n) if p not in held]
        assert src.tolist() == moved + [-1] * (pages // 2 - len(moved))
        assert dst.tolist() == free + [-1] * (pages // 2 - len(moved))


@pytest.mark.parametrize("dtype", DTYPES)
def test_sampling_of_more_rows_than_a_batch_of_launches(dtype):
    """1500 rows of their own, part of a wider tensor, all four settings and a number for each."""
    from perm_amd import sampling
    rows, vocab = 1500, 500
    x, u = _logits(21, rows, vocab + 13, dtype)
    rng = np.random.default_rng(21)
    settings = dict(temperature=rng.choice([0.0, 0.3, 0.7, 1.0, 1.5], rows), top_k=rng.choice([0, 0, 1, 20, 50, 499], rows),
                    top_p=rng.choice([1.0, 1.0, 0.5, 0.9, 0.95], rows), min_p=rng.choice([0.0, 0.0, 0.02, 0.1], rows))
    for y, v in ((x[:, 5:5 + vocab], u), (x[:, :vocab], u.double())):
        assert y.stride(0) > vocab
        _check_tokens(sampling, y, v, **settings)


@pytest.mark.parametrize("dtype,vocab", [(torch.float32, 5000011), (torch.bfloat16, 1 << 24)])
def test_sampling_of_the_largest_vocabularies(dtype, vocab):
    """Pieces of a row of more than 1024 units of 16 bytes, one to four steps each: nothing left out, a share, long lists,
    and (bfloat16) thousands of equal logits at every border. Weights are multiples of 2^-39 and 2^-38 of the
    largest here and what a row keeps sums to more than 2^6 of it: they err by under 2^-21 of the whole in all."""
    from perm_amd import sampling
    print(f"sample {vocab} {dtype}", flush=True)
    x, _ = _logits(22, 1, vocab, dtype)
    kinds = [dict(), dict(top_p=0.9), dict(top_k=1500), dict(top_k=3000000, min_p=1e-4), dict(top_k=40, top_p=0.95)]
    numbers = [[0.03, 0.41, 0.77], [0.999], [0.5], [0.86], [0.2]]
    for kind, us in zip(kinds, numbers):
        _check_tokens(sampling, x.expand(len(us), vocab), torch.tensor(us, dtype=torch.float64, device="cuda"), **kind)


def test_growth_of_thousands_of_sequences():
    """2100 of them, of one entry to wave-wide ranges, some past the table's end: pages run short behind the first 1024."""
    from oracle import pages_oracle as O
    from perm_amd import kvpages
    rng = np.random.default_rng(23)
    batch, cap, block = 2100, 12, 16
    lens = rng.integers(0, 60, batch)
    lens[5::40] = 0
    new = rng.choice([0, 1, 1, 1, 20, 110], batch)
    new[[300, 1400]] = 300  # more than the table's row holds
    need = -(-(lens + new) // block) + (-lens // block)
    for short in (1030, 1500, None):
        pages = int((-(-lens // block)).sum() + need[:short].sum()) + (0 if short else 2000)
        refs, table = _books(rng, pages, batch, cap, lens, block)
        o = O.Books(refs, table, block)
        refs, table = _i32(refs), _i32(table)
        want = o.grow(lens, new)
        unserved = [b for b in np.flatnonzero(want[2]) if b not in (300, 1400)]
        assert len(unserved) > 100 and unserved[0] >= short if short else not unserved
        got = kvpages.grow(refs, table, _i32(lens), _i32(new), block)
        for g, w, name in zip(got, want, ("src", "dst", "missing")):
            assert g.tolist() == w, (short, name)
        _same(o, refs, table)


# first rows of three sequences among 40 rows, some of which are no rows of the call
OUTSIDE = [[-1000, 5, 9, 40], [-3, -2, 0, 40], [-90000, -500, 12, 30], [7, 20, 10 ** 6, 10 ** 6], [7, 10 ** 6, 10 ** 6, 10 ** 6],
           [-5, 10 ** 6, 10 ** 6, 10 ** 6], [-2 ** 31, 11, 25, 2 ** 31 - 1], [-2 ** 31, -2 ** 31, 2 ** 31 - 1, 2 ** 31 - 1],
           [50, 60, 70, 80], [-9, -8, -7, -6], [40, 40, 40, 41], [3, 3, 40, 41]]


@pytest.mark.parametrize("tiles", [False, True], ids=["few", "tiles"])
@pytest.mark.parametrize("offsets", OUTSIDE, ids=str)
def test_attention_of_sequences_with_rows_outside_the_call(kv, monkeypatch, offsets, tiles):  # noqa: F811
    """They have no results, the rows of no sequence neither, and the others theirs, whatever memory held."""
    monkeypatch.setattr(kv, "_front_pays", lambda *a: True)
    print(f"outside {offsets} {tiles}", flush=True)
    rng = np.random.default_rng(31)
    rows, hq, lens = 40, 32, [70, 90, 60]
    c, o, table = _filled_cache(kv, rng, lens, 1, 64, 16)
    table[:, 0] = table[0, 0]
    t = _i32(_long(table, rows, hq, 16) if tiles else table)
    q = torch.from_numpy(rng.standard_normal((rows, hq, 64))).to(torch.bfloat16).cuda()
    whole = [b for b in range(3) if 0 <= offsets[b] < offsets[b + 1] <= rows]
    for more in (dict(), dict(softcap=20.0), dict(slopes=torch.full((hq,), 0.1, device="cuda")), dict(shared=_i32([1, 1, 1])),
                 dict(shared=_i32([1]))):
        results = [] if len(more.get("shared", "___")) == 1 and not 0 <= offsets[0] <= offsets[3] <= rows else whole
        _dirty(((rows, hq, 64), torch.bfloat16), ((rows, hq), torch.float32), ((rows * hq * 64 * 16,), torch.float32))
        out, lse = kv.attention(q, c, t, _i32(lens), _i32(offsets), return_lse=True, **more)
        left = torch.ones(rows, dtype=torch.bool, device="cuda")
        for b in results:
            at = slice(offsets[b], offsets[b + 1])
            left[at] = False
            alone = {k: v[b:b + 1] if k == "shared" else v for k, v in more.items()}
            want, wl = kv.attention(q[at], c, t[b:b + 1], _i32(lens[b:b + 1]), _i32([0, offsets[b + 1] - offsets[b]]),
                                    return_lse=True, **alone)
            # the same to the order of float32 sums, which moves a result by one rounding to 16 bits at most
            assert float((out[at].float() - want.float()).abs().max()) <= 2.0 ** -7 * float(want.float().abs().max())
            assert float((lse[at] - wl).abs().max()) <= 1e-4
        assert not out[left].any() and bool((lse[left] == float("-inf")).all())


@pytest.mark.parametrize("offsets", OUTSIDE, ids=str)
def test_rows_outside_the_call_written_and_read(kv, offsets):  # noqa: F811
    """A sequence that begins before row 0 is neither written nor read (0); one that passes the last row is read as
    far as there are rows."""
    rng = np.random.default_rng(32)
    rows, lens = 40, [70, 90, 60]
    c, o, table = _filled_cache(kv, rng, lens, 2, 48, 16)
    for dtype in (torch.bfloat16, torch.float32):
        _dirty(((rows, 2, 48), dtype))
        k, v = kv.read(c, _i32(table), _i32(offsets), rows, dtype)
        left = torch.ones(rows, dtype=torch.bool, device="cuda")
        for b in range(3):
            n = min(offsets[b + 1], rows) - offsets[b]
            if offsets[b] < 0 or n <= 0:
                continue
            at = slice(offsets[b], offsets[b] + n)
            left[at] = False
            want = kv.read(c, _i32(table[b:b + 1]), _i32([0, n]), n, dtype)
            assert torch.equal(k[at], want[0]) and torch.equal(v[at], want[1])
        assert not k[left].any() and not v[left].any()
    # written: whole pages of rows that there are
    x = torch.from_numpy(rng.standard_normal((rows, 2, 48))).to(torch.bfloat16).cuda()
    a, b = kv.new(*_geometry(c)), kv.new(*_geometry(c))
    kv.write(a, x, x, _i32(table), _i32([0, 0, 0]), _i32(offsets))
    for s in range(3):
        n = offsets[s + 1] - offsets[s]
        if offsets[s] < 0 or n <= 0 or offsets[s] >= rows:
            continue
        n = n if offsets[s + 1] <= rows else (rows - offsets[s]) // 16 * 16
        kv.write(b, x[offsets[s]:offsets[s] + n], x[offsets[s]:offsets[s] + n], _i32(table[s:s + 1]), _i32([0]), _i32([0, n]))
    assert all(torch.equal(y, z) for y, z in zip(a, b))


def _geometry(c):
    pages, heads, block, d = c.k.shape
    return pages, heads, d, block


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("many", [False, True])
def test_small_caps_of_large_keys(kv, many, dtype):  # noqa: F811
    """Keys under the largest scale and caps down to the least: scores are at most the cap, 2^-60 or less of one, so
    every row is the mean of the values it sees. Queries of 0 among them, whose scores are 0 under any cap."""
    rng = np.random.default_rng(41)
    n, rows = (2500, 700) if many else (100, 9)
    c, o, table = _filled_cache(kv, rng, [n], 1, 64, 16)
    c.k_scale.fill_(2.0 ** 60)
    q = torch.from_numpy(rng.standard_normal((rows, 12, 64))).to(dtype).cuda()
    q[1], q[5, 3:] = 0, 0
    assert not many or rows * 12 * table.shape[1] * 16 > 1 << 24
    v = kv.read(c, _i32(table), _i32([0, n]), n, torch.float32)[1][:, 0].double()
    want = (v.cumsum(0)[n - rows:] / torch.arange(n - rows + 1, n + 1, device="cuda")[:, None])[:, None]
    # one rounding to 16 bits and one of each weight: 2^-11 at most, of values up to max |v|
    tol = 2.0 ** -8 * want.abs() + 2.0 ** -11 * v.abs().max()
    for cap in (1e-30, 1e-25, 1e-20):
        out = kv.attention(q, c, _i32(table), _i32([n]), _i32([0, rows]), softcap=cap)
        assert bool(((out.double() - want).abs() <= tol).all()), cap


@pytest.mark.parametrize("counts", [[1] * 6, [0, 30, 30, 0, 1, 30]], ids=["tokens", "rows"])
@pytest.mark.parametrize("ended", [[0], [0, 1, 3], [0, 1, 2, 3, 4], [0, 1, 2, 4]], ids=str)
def test_common_pages_of_a_group_whose_first_sequences_have_ended(kv, monkeypatch, ended, counts):  # noqa: F811
    """Rows given back hold no pages: the others' front is looked up in one that does. Groups of six and of three."""
    from perm_amd import kvpages
    rng = np.random.default_rng(51)
    front, block, own = 40, 16, [20, 33, 50, 7, 1, 64]
    lens = [front * block + n for n in own]
    c, o, table = _filled_cache(kv, rng, lens, 2, 64, block)
    for g in (1, 2):
        t = table.copy()
        for b in range(6):
            t[b, :front] = t[b - b % (6 // g), :front]
        refs = np.zeros(c.k.shape[0], int)
        np.add.at(refs, t[t >= 0], 1)
        refs, t = _i32(refs), _i32(t)
        kvpages.free(refs, t, _i32(ended))
        held = _i32([0 if b in ended else n for b, n in enumerate(lens)])
        n = [0 if b in ended else x for b, x in enumerate(counts)] if max(counts) > 1 else counts
        offsets = None if max(counts) == 1 else _i32(np.concatenate([[0], np.cumsum(n)]))
        q = torch.from_numpy(rng.standard_normal((sum(n), 8, 64))).to(torch.bfloat16).cuda()
        for more in (dict(), dict(softcap=9.0), dict(window=500)):
            want, wl = kv.attention(q, c, t, held, offsets, return_lse=True, **more)
            monkeypatch.setattr(kv, "_front_pays", lambda *a: True)
            got, gl = kv.attention(q, c, t, held, offsets, return_lse=True, shared=_i32([front] * g), **more)
            monkeypatch.undo()
            # the same but for the order of float32 sums and one rounding to bfloat16
            assert float((got.float() - want.float()).abs().max()) <= 2.0 ** -7 * float(want.float().abs().max()) + 1e-30
            some = torch.isfinite(wl)
            assert torch.equal(some, torch.isfinite(gl)) and bool(((gl - wl).abs()[some] <= 1e-4).all())
