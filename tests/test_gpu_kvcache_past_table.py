"""Sequences longer than their table: rows keep their positions, tokens past the table have no
page."""
import numpy as np
import pytest
import torch

from oracle import mx_oracle as O
from test_gpu_kvcache import HALF_ULP, _filled_cache, _i32, _offsets, kv  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("causal,window", [(True, 0), (True, 60), (True, 130), (False, 0), (False, 70)])
@pytest.mark.parametrize("tiles", [False, True], ids=["few", "tiles"])
def test_positions(kv, tiles, causal, window):  # noqa: F811
    rng = np.random.default_rng(window)
    c, o, table = _filled_cache(kv, rng, [192, 64, 64, 192], 1, 64, 16)
    table = table[:, :12]  # 192 tokens at most
    table[1:3, 4:] = -1
    lens, hq = [200, 400, 70, 2 ** 31 - 1], 4
    # tiles of 128 rows are taken above 2^24 rows x heads x tokens
    counts = [2 ** 24 // (hq * 150), 3, 33, 1] if tiles else [10, 3, 12, 1]
    q = torch.from_numpy(rng.standard_normal((sum(counts), hq, 64))).to(torch.bfloat16).cuda()
    out, lse = kv.attention(q, c, _i32(table), _i32(lens), _offsets(counts), causal=causal, window=window,
                            return_lse=True)
    r = 0
    for b, n in enumerate(counts):
        length = min(lens[b], 1000)  # the longest ends past every window either way
        k, v, have = o.tokens(table[b], length)
        last = min(n, 170)
        got, gl = (x[r + n - last:r + n].double().cpu().numpy() for x in (out, lse))
        want, wl, bound = O.attention(q[r + n - last:r + n].double().cpu().numpy(), k, v, have, causal, window, 0.125)
        err = np.abs(got - want)
        assert (err <= bound + HALF_ULP[torch.bfloat16] * np.abs(want) * 1.01 + 2.0 ** -24).all(), (b, err.max())
        assert np.array_equal(np.isfinite(gl), np.isfinite(wl)), b
        r += n
