"""NaN codes that a row does not see, at every head size and page size, in the columns where a
kernel's bookkeeping changes: the first, the last, past 64 and past 128."""
import numpy as np
import pytest
import torch

from test_gpu_kvcache import _check_attention, _filled_cache, kv  # noqa: F401
from test_gpu_kvcache_tiles import _long

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tiles", [False, True], ids=["few", "tiles"])
@pytest.mark.parametrize("block", [16, 64, 128])
@pytest.mark.parametrize("d", [16, 80, 112, 128, 192, 256])
def test_unseen_tokens(kv, d, block, tiles):  # noqa: F811
    print(f"nan {d} {block} {tiles}", flush=True)
    rng = np.random.default_rng(d + block)
    lens = [37, 200]
    c, o, table = _filled_cache(kv, rng, lens, 2, d, block)
    columns = sorted({0, 15, d // 2, d - 1} | {x for x in (63, 64, 127, 128, 200) if x < d})
    for buf in (o.k, o.v):  # slots past the sequences' ends, and a page past the first's
        buf[table[0][37 // block], :, 37 % block:] = 127
        buf[table[1][200 // block], :, 200 % block:] = 255
        buf[table[0][37 // block + 1]] = 127
    # tokens that later rows see and earlier ones do not, a column each
    for i, x in enumerate(columns):
        p = 130 + 5 * i
        o.v[table[1][p // block], i % 2, p % block, x] = 127 + 128 * (i % 2)
    o.k[table[1][185 // block], 1, 185 % block, d - 1] = 255
    # before every window: rows that see it all the same are NaN in that column
    o.v[table[1][2 // block], 0, 2 % block, d - 1] = 127
    c.k.copy_(torch.from_numpy(o.k))
    c.v.copy_(torch.from_numpy(o.v.swapaxes(2, 3).copy()))
    for counts in ([37, 200],) if tiles else ([1, 1], [9, 90]):
        t = _long(table, sum(counts), 8, block) if tiles else table
        _check_attention(kv, o, c, t, lens, counts, 8, torch.bfloat16, rng)
        _check_attention(kv, o, c, t, lens, counts, 8, torch.float16, rng, causal=False)
    if not tiles:
        _check_attention(kv, o, c, table, lens, [9, 90], 8, torch.bfloat16, rng, window=20)


def test_unseen_tokens_before_a_window(kv):  # noqa: F811
    """The same in tiles of 128 rows, which with a window take more rows."""
    rng = np.random.default_rng(5)
    n, window, d = 1400, 300, 192
    c, o, table = _filled_cache(kv, rng, [n], 1, d, 32)
    for p, x in ((700, 0), (701, 191), (1000, 130), (3, 64)):
        o.v[table[0][p // 32], 0, p % 32, x] = 127
    c.v.copy_(torch.from_numpy(o.v.swapaxes(2, 3).copy()))
    q = torch.from_numpy(rng.standard_normal((n, 32, d))).to(torch.bfloat16).cuda()
    from test_gpu_kvcache import _i32, _offsets
    out = kv.attention(q, c, _i32(table), _i32([n]), _offsets([n]), window=window)
    bad = out.isnan()
    want = torch.zeros((n, d), dtype=torch.bool, device="cuda")
    for p, x in ((700, 0), (701, 191), (1000, 130), (3, 64)):
        want[p:p + window, x] = True
    assert torch.equal(bad, want[:, None].expand_as(bad))
