"""Attention whose weights span many binades: rows that put nearly all of their weight on one
token whose values are 0, pages whose V scales are far apart, wide scores. The bound is the
other tests': 2^-11 of each token's own share, whatever the share is."""
import numpy as np
import pytest
import torch

from oracle import mx_oracle as O
from test_gpu_kvcache import _check_attention, _i32, _offsets, kv  # noqa: F401
from test_gpu_kvcache_tiles import _long

pytestmark = pytest.mark.gpu


def _cache_of(kv, rng, lens, heads, d, block, change):
    """Caches holding normal rows of every sequence as ``change(k, v, n)`` leaves them."""
    cap = max(lens) // block + 1
    pages = len(lens) * cap
    c, o = kv.new(pages, heads, d, block), O.Cache(pages, heads, d, block)
    table = rng.permutation(pages).reshape(len(lens), cap)
    ks, vs = [], []
    for n in lens:
        k, v = rng.standard_normal((n, heads, d)), rng.standard_normal((n, heads, d))
        change(k, v, n)
        ks.append(k)
        vs.append(v)
    k, v = (torch.from_numpy(np.concatenate(x)).to(torch.bfloat16).cuda() for x in (ks, vs))
    zero = np.zeros(len(lens), int)
    kv.write(c, k, v, _i32(table), _i32(zero), _offsets(lens))
    o.write(k.double().cpu().numpy(), v.double().cpu().numpy(), table, zero, lens)
    return c, o, table


def _check(kv, rng, c, o, table, lens, counts, hq, dtype, tiles, head0=None, spread=1.0):
    rows = int(np.sum(counts))
    q = rng.standard_normal((rows, hq, o.k.shape[3])) * spread
    if head0 is not None:
        q[..., 0] = head0
    t = _long(table, rows, hq, o.block) if tiles else table
    _check_attention(kv, o, c, t, lens, counts, hq, dtype, rng, q=torch.from_numpy(q).to(dtype).cuda())


@pytest.mark.parametrize("lead", [10.0, 16.6, 19.0, 25.0, 60.0])
@pytest.mark.parametrize("tiles", [False, True], ids=["few", "tiles"])
@pytest.mark.parametrize("d,block,dtype", [(64, 16, torch.bfloat16), (128, 32, torch.float16), (256, 16, torch.bfloat16)])
def test_a_first_token_without_values(kv, d, block, dtype, tiles, lead):  # noqa: F811
    print(f"first token {d} {block} {tiles} {lead} {dtype}", flush=True)
    rng = np.random.default_rng(int(lead) + d)

    def sink(k, v, n):
        k[:, :, 0] = 0
        k[0], v[0] = 0, 0
        k[0, :, 0] = lead / 16 * d ** 0.5
    lens, counts = ([900, 21], [70, 21]) if tiles else ([2048, 21, 70], [1, 5, 9])
    c, o, table = _cache_of(kv, rng, lens, 1, d, block, sink)
    _check(kv, rng, c, o, table, lens, counts, 4, dtype, tiles, head0=16.0)


@pytest.mark.parametrize("e", [8, 14, 20, 22, 26, 60, 100])
@pytest.mark.parametrize("tiles", [False, True], ids=["few", "tiles"])
def test_values_raised_by_an_unseen_token(kv, tiles, e):  # noqa: F811
    """Token 25's values are 2^e times the others': its page's scale grows, and rows before
    it see the page but not the token."""
    rng = np.random.default_rng(e)

    def raise25(k, v, n):
        if n > 25:
            v[25] *= 2.0 ** e
    lens = [60, 200]
    c, o, table = _cache_of(kv, rng, lens, 2, 64, 16, raise25)
    for counts in ([60, 200],) if tiles else ([36, 30], [1, 1]):
        _check(kv, rng, c, o, table, lens, counts, 4, torch.bfloat16, tiles)
    # one column alone is large, so the others' codes are 0 on that page
    def column(k, v, n):
        v[::40, :, 3] *= 2.0 ** e
    c, o, table = _cache_of(kv, rng, lens, 2, 64, 16, column)
    _check(kv, rng, c, o, table, lens, [60, 200] if tiles else [3, 20], 4, torch.bfloat16, tiles)


@pytest.mark.parametrize("lead", [-100.0, -30.0, 0.0, 5.0, 12.0, 30.0, 60.0])
@pytest.mark.parametrize("tiles", [False, True], ids=["few", "tiles"])
def test_the_scales_both_ends(kv, tiles, lead):  # noqa: F811
    """Pages at 2^60 beside pages at 2^-60 whose scores are ``lead`` above theirs."""
    rng = np.random.default_rng(int(lead) + 200)

    def ends(k, v, n):
        small = np.arange(n) // 16 % 3 == 1
        k[:, :, 0] = np.where(small, lead / 2, 0)[:, None]
        v *= np.where(small, 2.0 ** -58, 2.0 ** 66)[:, None, None]
    lens = [16, 40, 130]
    c, o, table = _cache_of(kv, rng, lens, 1, 64, 16, ends)
    assert o.vs.max() == 2.0 ** 60 and o.vs.min() <= 2.0 ** -60
    counts = lens if tiles else [1, 8, 20]
    _check(kv, rng, c, o, table, lens, counts, 4, torch.bfloat16, tiles, head0=16.0)


@pytest.mark.parametrize("spread", [3.0, 10.0, 40.0])
@pytest.mark.parametrize("tiles", [False, True], ids=["few", "tiles"])
def test_wide_scores(kv, tiles, spread):  # noqa: F811
    """Scores whose standard deviation is ``spread``, in prompts with a window's edge."""
    rng = np.random.default_rng(int(spread))
    lens, counts = [500, 77], ([90, 77] if tiles else [4, 9])
    c, o, table = _cache_of(kv, rng, lens, 2, 64, 16, lambda k, v, n: None)
    _check(kv, rng, c, o, table, lens, counts, 4, torch.bfloat16, tiles, spread=spread)
    _check(kv, rng, c, o, table, lens, counts, 4, torch.float16, tiles, spread=spread)


@pytest.mark.parametrize("d,block,heads", [(64, 16, 2), (80, 32, 1), (128, 64, 2), (256, 16, 1)])
@pytest.mark.parametrize("tiles", [False, True], ids=["few", "tiles"])
def test_waves_of_both_kinds(kv, tiles, d, block, heads):  # noqa: F811
    """Flat and peaked rows in turn, 8, 32 or 128 of a kind: waves of a workgroup that change
    at different tiles, or never."""
    rng = np.random.default_rng(d)
    lens = [700, 300]
    c, o, table = _cache_of(kv, rng, lens, heads, d, block, lambda k, v, n: None)
    for run in (8, 32, 128):
        counts = [260, 300] if tiles else [20, 7]
        kind = np.arange(sum(counts)) // max(1, run // 4) % 2  # four heads share a cache head
        q = rng.standard_normal((sum(counts), 4 * heads, d)) * np.where(kind, 30.0, 0.3)[:, None, None]
        t = _long(table, sum(counts), 4 * heads, block) if tiles else table
        _check_attention(kv, o, c, t, lens, counts, 4 * heads, torch.bfloat16, rng,
                         q=torch.from_numpy(q).to(torch.bfloat16).cuda())


@pytest.mark.parametrize("tiles", [False, True], ids=["few", "tiles"])
@pytest.mark.parametrize("d", [64, 112, 256])
def test_unseen_tokens_beside_wide_scores(kv, tiles, d):  # noqa: F811
    """NaN in tokens that a row does not see, where weights take two terms."""
    rng = np.random.default_rng(d + 1)
    lens = [37, 100]
    c, o, table = _cache_of(kv, rng, lens, 2, d, 16, lambda k, v, n: None)
    for buf in (o.k, o.v):
        buf[table[0][2], :, 37 % 16:] = 127
        buf[table[1][6], :, 100 % 16:] = 127
    o.v[table[1][5], 0, 85 % 16, 7] = 127
    o.v[table[1][2], 1, 5, d - 1] = 255
    o.k[table[1][5], 0, 90 % 16, 3] = 127
    c.k.copy_(torch.from_numpy(o.k))
    c.v.copy_(torch.from_numpy(o.v.swapaxes(2, 3).copy()))
    for counts in ([37, 100],) if tiles else ([1, 1], [10, 30]):
        _check(kv, rng, c, o, table, lens, counts, 8, torch.bfloat16, tiles, spread=40.0)
