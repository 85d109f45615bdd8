"""Windows past 32 bits: none of them hides a token."""
import numpy as np
import pytest
import torch

from test_gpu_kvcache import _filled_cache, _i32, _offsets, kv  # noqa: F401
from test_gpu_kvcache_tiles import _long

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 5, 2 ** 40])
@pytest.mark.parametrize("tiles", [False, True], ids=["few", "tiles"])
def test_no_window_is_this_wide(kv, tiles, window):  # noqa: F811
    rng = np.random.default_rng(31)
    c, o, table = _filled_cache(kv, rng, [150, 40], 1, 64, 16)
    counts = [150, 40] if tiles else [3, 1]
    t = _i32(_long(table, sum(counts), 4, 16) if tiles else table)
    q = torch.from_numpy(rng.standard_normal((sum(counts), 4, 64))).to(torch.bfloat16).cuda()
    args = (q, c, t, _i32([150, 40]), _offsets(counts))
    for causal in (True, False):
        assert torch.equal(kv.attention(*args, causal=causal, window=window), kv.attention(*args, causal=causal))
