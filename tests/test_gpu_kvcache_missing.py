"""Tokens without a page beside a first page whose buffers hold no cache yet: nothing of it
reaches a row."""
import numpy as np
import pytest
import torch

from test_gpu_kvcache import _check_attention, _filled_cache, kv  # noqa: F401
from test_gpu_kvcache_tiles import _long

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), 0.0, -1.0])
@pytest.mark.parametrize("tiles", [False, True], ids=["few", "tiles"])
@pytest.mark.parametrize("d,block", [(64, 16), (112, 32)])
def test_the_first_page_is_not_in_use(kv, d, block, tiles, scale):  # noqa: F811
    rng = np.random.default_rng(d)
    lens = [120, 64, 40]
    c, o, table = _filled_cache(kv, rng, lens, 2, d, block)
    table = table.copy()
    table[table == 0] = -1  # one sequence's page, or none's
    table[0][1], table[1][0] = -1, o.k.shape[0] + 3
    for x in (c.k_scale, c.v_scale):
        x[0] = scale
    for x, y in ((c.k, o.k), (c.v, o.v)):
        x[0], y[0] = 127, 127
    counts = [120, 64, 40] if tiles else [9, 1, 2]
    t = _long(table, sum(counts), 4, block) if tiles else table
    for spread in (1.0, 30.0):
        q = rng.standard_normal((sum(counts), 4, d)) * spread
        _check_attention(kv, o, c, t, lens, counts, 4, torch.bfloat16, rng,
                         q=torch.from_numpy(q).to(torch.bfloat16).cuda())
