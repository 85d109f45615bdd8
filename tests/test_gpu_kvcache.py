"""The paged 8-bit cache and attention over it, against the float64 oracle: codes and scales
exactly, attention within the bounds of float16 weights, float32 scores and one rounding."""
import numpy as np
import pytest
import torch

from oracle import mx_oracle as O

pytestmark = pytest.mark.gpu
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16)}


@pytest.fixture(scope="module")
def kv():
    from perm_amd import kvcache
    return kvcache


def _i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def _offsets(counts):
    return _i32(np.concatenate([[0], np.cumsum(counts)]))


def _tables(rng, batch, max_pages, pages):
    return rng.permutation(pages)[: batch * max_pages].reshape(batch, max_pages)


def _same_cache(c, o):
    assert np.array_equal(c.k_scale.cpu().numpy(), o.ks.astype(np.float32))
    assert np.array_equal(c.v_scale.cpu().numpy(), o.vs.astype(np.float32))
    for got, want in ((c.k.cpu().numpy(), o.k), (c.v.cpu().numpy().swapaxes(2, 3), o.v)):
        nan = (want & 127) == 127
        assert np.array_equal((got & 127) == 127, nan)
        assert np.array_equal(np.where(nan, 0, got), np.where(nan, 0, want))


def _append(kv, rng, c, o, table, filled, counts, dtype, grow=1.0, offsets=True):
    heads, d = o.k.shape[1], o.k.shape[3]
    rows = int(np.sum(counts))
    k, v = (torch.from_numpy(rng.standard_normal((rows, heads, d)) * grow).to(dtype).cuda()
            for _ in range(2))
    kv.write(c, k, v, _i32(table), _i32(filled), _offsets(counts) if offsets else None)
    o.write(k.double().cpu().numpy(), v.double().cpu().numpy(), table, filled, counts)
    _same_cache(c, o)
    return k, v


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("block,heads,d", [(16, 2, 64), (32, 1, 16), (64, 3, 80), (128, 2, 128), (16, 1, 256)])
def test_write_and_read(kv, block, heads, d, dtype):
    """A ragged prompt, single tokens, a few tokens across a page's end, with growing rows."""
    print(f"cache {block} {heads} {d} {dtype}", flush=True)
    rng = np.random.default_rng(block + d)
    cap = 300 // block + 2
    c, o = kv.new(5 * cap, heads, d, block), O.Cache(5 * cap, heads, d, block)
    table = _tables(rng, 4, cap, 5 * cap)
    counts = np.array([block + 3, 0, 1, 150])
    filled = np.zeros(4, int)
    _append(kv, rng, c, o, table, filled, counts, dtype)
    filled += counts
    for n, grow in ((1, 1.0), (1, 3.0), (5, 0.1), (17, 40.0)):
        new = np.full(4, n)
        _append(kv, rng, c, o, table, filled, new, dtype, grow, offsets=n != 1)
        filled += new
    for out in (torch.float32, torch.bfloat16, torch.float16):
        k, v = kv.read(c, _i32(table), _offsets(filled), int(filled.sum()), out)
        want = [o.tokens(table[b], filled[b]) for b in range(4)]
        for got, i in ((k, 0), (v, 1)):
            w = torch.from_numpy(np.concatenate([t[i] for t in want]))
            assert torch.equal(got.cpu(), w.to(torch.float32).to(out))


def test_a_page_written_again_is_its_own(kv):
    """A reused page takes the scale of its new rows, and slots not written keep their codes."""
    rng = np.random.default_rng(1)
    c, o = kv.new(3, 2, 32, 16), O.Cache(3, 2, 32, 16)
    table = np.array([[2, 0]])
    _append(kv, rng, c, o, table, [0], [32], torch.bfloat16, 100.0)
    _append(kv, rng, c, o, table, [0], [7], torch.bfloat16, 0.01)
    _append(kv, rng, c, o, table, [3], [2], torch.bfloat16, 0.02)  # taken back to three tokens


def test_nan_infinity_and_extremes(kv):
    c, o = kv.new(4, 1, 32, 16), O.Cache(4, 1, 32, 16)
    x = torch.randn((40, 1, 32), generator=torch.Generator().manual_seed(2))
    x[3, 0, 5], x[4, 0, 6], x[5, 0, 7] = float("nan"), float("inf"), -float("inf")
    x[16:32] = 0
    x[33, 0, 0] = 3e38  # past the largest scale
    y = x.clone()
    y[:16] *= 1e-30     # below the least
    y[35] = float("nan")
    for dtype in (torch.float32, torch.bfloat16):
        k, v = x.to(dtype).cuda(), y.to(dtype).cuda()
        kv.write(c, k, v, _i32([[1, 3, 0]]), _i32([0]), _i32([0, 40]))
        o.write(k.double().cpu().numpy(), v.double().cpu().numpy(), [[1, 3, 0]], [0], [40])
        _same_cache(c, o)


def test_every_bf16_value_is_coded(kv):
    b = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    b = b[torch.isfinite(b)]
    b = b[: b.numel() // 32 * 32].view(-1, 1, 32)
    pages = -(-b.shape[0] // 16)
    c, o = kv.new(pages, 1, 32, 16), O.Cache(pages, 1, 32, 16)
    table = np.arange(pages)[None, :]
    kv.write(c, b.cuda(), b.cuda(), _i32(table), _i32([0]), _i32([0, b.shape[0]]))
    o.write(b.double().numpy(), b.double().numpy(), table, [0], [b.shape[0]])
    _same_cache(c, o)


def test_pages_outside_the_cache_and_past_the_table(kv):
    rng = np.random.default_rng(4)
    c, o = kv.new(4, 2, 32, 16), O.Cache(4, 2, 32, 16)
    table = np.array([[1, -1, 2], [4, 3, 1 << 30]])
    _append(kv, rng, c, o, table, [0, 0], [60, 40], torch.bfloat16)
    k, v = kv.read(c, _i32(table), _i32([0, 50, 90]), 90, torch.float32)
    want = [o.tokens(table[b], n) for b, n in ((0, 50), (1, 40))]
    assert np.array_equal(k.cpu().numpy(), np.concatenate([w[0] for w in want]).astype(np.float32))
    assert np.array_equal(v.cpu().numpy(), np.concatenate([w[1] for w in want]).astype(np.float32))
    assert not k[16:32].any()


def test_strides_of_a_joint_projection(kv):
    """q, k and v as views of one projection's output; a view that is not aligned."""
    rng = np.random.default_rng(5)
    c, o = kv.new(4, 2, 64, 16), O.Cache(4, 2, 64, 16)
    qkv = torch.from_numpy(rng.standard_normal((20, 8, 64))).to(torch.bfloat16).cuda()
    k, v = qkv[:, 4:6], qkv[:, 6:8]
    kv.write(c, k, v, _i32([[0, 2]]), _i32([0]), _i32([0, 20]))
    o.write(k.double().cpu().numpy(), v.double().cpu().numpy(), [[0, 2]], [0], [20])
    _same_cache(c, o)
    want = kv.attention(qkv[:, :4].contiguous(), c, _i32([[0, 2]]), _i32([20]), _i32([0, 20]))
    assert torch.equal(kv.attention(qkv[:, :4], c, _i32([[0, 2]]), _i32([20]), _i32([0, 20])), want)
    odd = torch.zeros((20 * 8 * 64 + 1), dtype=torch.bfloat16, device="cuda")[1:].view(20, 8, 64)
    odd.copy_(qkv)
    kv.write(c, odd[:, 4:6], odd[:, 6:8], _i32([[3, 1]]), _i32([0]), _i32([0, 20]))
    assert torch.equal(c.k[3], c.k[0]) and torch.equal(c.v[1][..., :4], c.v[2][..., :4])
    heads_first = qkv[:, :4].transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(kv.attention(heads_first, c, _i32([[0, 2]]), _i32([20]), _i32([0, 20])), want)


def _filled_cache(kv, rng, lens, heads, d, block, dtype=torch.bfloat16, grow=1.0, extra=3):
    cap = -(-max(max(lens), 1) // block) + 1
    pages = len(lens) * cap + extra
    c, o = kv.new(pages, heads, d, block), O.Cache(pages, heads, d, block)
    table = _tables(rng, len(lens), cap, pages)
    rows = int(np.sum(lens))
    k, v = (torch.from_numpy(rng.standard_normal((rows, heads, d)) * grow).to(dtype).cuda() for _ in range(2))
    # a channel far above the rest, and pages of their own size
    k[..., 0] *= 8
    if rows:
        kv.write(c, k, v, _i32(table), _i32(np.zeros(len(lens))), _offsets(lens))
        o.write(k.double().cpu().numpy(), v.double().cpu().numpy(), table, np.zeros(len(lens), int), lens)
    return c, o, table


def _check_attention(kv, o, c, table, lens, counts, hq, dtype, rng, causal=True, window=0, scale=None,
                     offsets=True, q=None):
    heads, d = o.k.shape[1], o.k.shape[3]
    rows = int(np.sum(counts))
    if q is None:
        q = torch.from_numpy(rng.standard_normal((rows, hq, d))).to(dtype).cuda()
    out, lse = kv.attention(q, c, _i32(table), _i32(lens), _offsets(counts) if offsets else None,
                            causal=causal, window=window, scale=scale, return_lse=True)
    assert torch.equal(kv.attention(q, c, _i32(table), _i32(lens), _offsets(counts) if offsets else None,
                                    causal=causal, window=window, scale=scale).view(torch.int16),
                       out.view(torch.int16))
    r = 0
    for b, n in enumerate(counts):
        k, v, have = o.tokens(table[b], min(lens[b], len(table[b]) * o.block))
        qd = q[r:r + n].double().cpu().numpy()
        want, wl, bound = O.attention(qd, k, v, have, causal, window, d ** -0.5 if scale is None else scale)
        got, gl = out[r:r + n].double().cpu().numpy(), lse[r:r + n].double().cpu().numpy()
        nan = np.isnan(want)
        assert np.array_equal(np.isnan(got), nan)
        err = np.abs(np.where(nan, 0, got - np.where(nan, 0, want)))
        limit = np.nan_to_num(bound) + HALF_ULP[dtype] * np.abs(np.nan_to_num(want)) * 1.01 + 2.0 ** -24
        assert (err <= limit).all(), (b, (err / limit).max())
        fin = np.isfinite(wl)
        assert np.array_equal(np.isfinite(gl), fin)
        assert (np.abs(gl[fin] - wl[fin]) <= 2.0 ** -17 * (1 + np.abs(wl[fin]))).all()
        r += n


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("block,heads,d,group", [(16, 2, 128, 2), (32, 1, 64, 4), (64, 2, 80, 1), (128, 1, 256, 8),
                                                 (16, 1, 16, 3), (32, 2, 96, 20)])
def test_single_tokens(kv, block, heads, d, group, dtype):
    print(f"attend token {block} {heads} {d} {group} {dtype}", flush=True)
    rng = np.random.default_rng(d + group)
    lens = [1, 0, 15, 16, 17, 63, 64, 65, 130, 700]
    c, o, table = _filled_cache(kv, rng, lens, heads, d, block)
    ones = np.ones(len(lens), int)
    _check_attention(kv, o, c, table, lens, ones, heads * group, dtype, rng, offsets=False)
    _check_attention(kv, o, c, table, lens, ones, heads * group, dtype, rng, window=33)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 40), (False, 0), (False, 25), (True, 1)])
@pytest.mark.parametrize("block,heads,d,group", [(16, 2, 128, 2), (64, 1, 64, 4), (32, 1, 112, 1)])
def test_ragged_prompts(kv, block, heads, d, group, causal, window, dtype):
    """Prompts of no rows, one, many, and more rows than tokens (the first ones see nothing)."""
    print(f"attend prompt {block} {heads} {d} {group} {causal} {window} {dtype}", flush=True)
    rng = np.random.default_rng(block + group + window)
    lens, counts = [150, 70, 5, 33, 0, 200], [150, 1, 9, 0, 3, 77]
    c, o, table = _filled_cache(kv, rng, lens, heads, d, block)
    _check_attention(kv, o, c, table, lens, counts, heads * group, dtype, rng, causal, window)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_long_prompt_and_long_cache(kv, dtype):
    rng = np.random.default_rng(6)
    c, o, table = _filled_cache(kv, rng, [1500, 40], 1, 64, 16)
    _check_attention(kv, o, c, table, [1500, 40], [300, 2], 4, dtype, rng)
    _check_attention(kv, o, c, table, [1500, 40], [1, 1], 4, dtype, rng, offsets=False)
    _check_attention(kv, o, c, table, [1500, 40], [5, 2], 4, dtype, rng, window=200)


def test_scale_and_large_scores(kv):
    """Scores of hundreds, a softmax of one token, and scales of every size."""
    rng = np.random.default_rng(7)
    c, o, table = _filled_cache(kv, rng, [90, 200], 1, 64, 16, grow=30.0)
    _check_attention(kv, o, c, table, [90, 200], [90, 3], 2, torch.bfloat16, rng, scale=1.0)
    _check_attention(kv, o, c, table, [90, 200], [90, 3], 2, torch.float16, rng, scale=1e-4)
    for p in range(o.vs.shape[0]):  # V scales of their own: from 2^-30 to 2^7
        o.vs[p] = c.v_scale[p] = 2.0 ** int(rng.integers(-30, 8))
    _check_attention(kv, o, c, table, [90, 200], [40, 3], 2, torch.bfloat16, rng)


def test_unseen_tokens_do_not_reach_a_row(kv):
    """NaN in slots past the length, in later tokens of a prompt, before the window, and on
    pages of other sequences; a NaN that a row sees makes it NaN."""
    rng = np.random.default_rng(8)
    lens = [37, 100]
    c, o, table = _filled_cache(kv, rng, lens, 2, 64, 16)
    for buf in (o.k, o.v):
        page, slot = table[0][37 // 16], 37 % 16
        buf[page, :, slot:] = 127
        buf[table[0][3]] = 255
        buf[table[1][100 // 16], :, 100 % 16:] = 127
    spots = [(table[1][85 // 16], 85 % 16), (table[1][2], 5)]
    o.v[spots[0][0], 0, spots[0][1], 7] = 127   # token 85: rows before it do not see it
    o.v[spots[1][0], 1, spots[1][1], 9] = 255   # token 37
    o.k[table[1][90 // 16], 0, 90 % 16, 3] = 127
    c.k.copy_(torch.from_numpy(o.k))
    c.v.copy_(torch.from_numpy(o.v.swapaxes(2, 3).copy()))
    for window in (0, 20):
        for counts in ([1, 1], [10, 30], [37, 100]):
            _check_attention(kv, o, c, table, lens, counts, 4, torch.bfloat16, rng, window=window)
    _check_attention(kv, o, c, table, lens, [3, 60], 4, torch.float16, rng, causal=False)


def test_missing_pages(kv):
    rng = np.random.default_rng(9)
    c, o, table = _filled_cache(kv, rng, [120, 64, 40], 2, 64, 16)
    table = table.copy()
    table[0][1], table[0][4], table[1][:] = -1, o.k.shape[0], -5
    _check_attention(kv, o, c, table, [120, 64, 40], [120, 3, 1], 4, torch.bfloat16, rng)
    # lengths past the table's end see what the table holds
    _check_attention(kv, o, c, table, [16 * table.shape[1], 64, 40], [1, 1, 1], 4, torch.bfloat16, rng,
                     offsets=False)


def test_offsets_past_32_bits(kv):
    """A cache of 4.3 GB each of K and V whose last pages are used."""
    pages, heads, d, block = 264000, 8, 128, 16
    c = kv.new(pages, heads, d, block)
    rng = np.random.default_rng(10)
    small, o = kv.new(8, heads, d, block), O.Cache(8, heads, d, block)
    table = rng.permutation(8)[None, :]
    k, v = (torch.from_numpy(rng.standard_normal((120, heads, d))).to(torch.bfloat16).cuda() for _ in range(2))
    kv.write(small, k, v, _i32(table), _i32([0]), _i32([0, 120]))
    kv.write(c, k, v, _i32(table + pages - 8), _i32([0]), _i32([0, 120]))
    assert torch.equal(c.k[-8:], small.k) and torch.equal(c.v[-8:], small.v) and not c.k[:64].any()
    for n in (1, 50):
        q = torch.from_numpy(rng.standard_normal((n, 16, d))).to(torch.bfloat16).cuda()
        off = _i32([0, n])
        assert torch.equal(kv.attention(q, c, _i32(table + pages - 8), _i32([120]), off),
                           kv.attention(q, small, _i32(table), _i32([120]), off))
    a = kv.read(c, _i32(table + pages - 8), _i32([0, 120]), 120)
    b = kv.read(small, _i32(table), _i32([0, 120]), 120)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_other_stream_and_empty_batches(kv):
    rng = np.random.default_rng(11)
    c, o, table = _filled_cache(kv, rng, [300, 20], 2, 64, 16)
    q = torch.from_numpy(rng.standard_normal((2, 4, 64))).to(torch.bfloat16).cuda()
    args = (q, c, _i32(table), _i32([300, 20]))
    want = kv.attention(*args)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [kv.attention(*args) for _ in range(4)]
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(g, want) for g in got)
    none = torch.empty((0, 4, 64), dtype=torch.bfloat16, device="cuda")
    assert kv.attention(none, c, _i32(table), _i32([300, 20]), _i32([0, 0, 0])).shape == (0, 4, 64)
    kv.write(c, none[:, :2], none[:, :2], _i32(table), _i32([300, 20]), _i32([0, 0, 0]))
    assert kv.read(c, _i32(table), _i32([0, 0, 0]), 0)[0].shape == (0, 2, 64)
    _same_cache(c, o)


def test_a_graph_replays(kv):
    """One decoding step (write, attend) captured; replayed with new rows and lengths."""
    rng = np.random.default_rng(12)
    c, o, table = _filled_cache(kv, rng, [30, 50], 2, 64, 16)
    filled, lens = _i32([30, 50]), _i32([31, 51])
    x = torch.from_numpy(rng.standard_normal((2, 8, 64))).to(torch.bfloat16).cuda()
    t = _i32(table)

    def step():
        kv.write(c, x[:, 4:6], x[:, 6:], t, filled, None)
        return kv.attention(x[:, :4], c, t, lens)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for i in range(4):
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, step()), i
        x.copy_(torch.from_numpy(rng.standard_normal((2, 8, 64))))
        filled.add_(1)
        lens.add_(1)


def test_refusals(kv):
    c = kv.new(4, 2, 64, 16)
    k = torch.zeros((2, 2, 64), dtype=torch.bfloat16, device="cuda")
    t, n = _i32([[0], [1]]), _i32([0, 0])
    with pytest.raises(ValueError):
        kv.new(4, 2, 72, 16)
    with pytest.raises(ValueError):
        kv.new(4, 2, 64, 24)
    with pytest.raises(TypeError):
        kv.write(c, k, k.float(), t, n)
    with pytest.raises(ValueError):
        kv.write(c, k[:, :1], k, t, n)
    with pytest.raises(ValueError):
        kv.write(c, k[:1], k[:1], t, n)
    with pytest.raises(ValueError):
        kv.write(c, k.cpu(), k.cpu(), t, n)
    with pytest.raises(IndexError):
        kv.write(c, k, k, t.long(), n)
    with pytest.raises(ValueError):
        kv.write(c, k, k, t, n[:1])
    with pytest.raises(ValueError):
        kv.write(c, k, k, t, n, _i32([0, 2]))
    with pytest.raises(ValueError):
        kv.attention(k[:, :1].expand(2, 3, 64), c, t, n)
    with pytest.raises(TypeError):
        kv.attention(k.float(), c, t, n)
    with pytest.raises(ValueError):
        kv.attention(k, c, t, n, window=-1)
    with pytest.raises(ValueError):
        kv.read(c, t, None, 2)
    with pytest.raises(TypeError):
        kv.read(c, t, _i32([0, 1, 2]), 2, torch.int8)
    with pytest.raises(ValueError):
        kv.write(kv.KvCache(c.k, c.v[:2], c.k_scale, c.v_scale), k, k, t, n)
    with pytest.raises(TypeError):
        kv.write(kv.KvCache(c.k, c.v, c.k_scale.double(), c.v_scale), k, k, t, n)
