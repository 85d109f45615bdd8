"""The low-bit oracle's number formats against their definitions: e2m1 and e4m3 rounding by
exhaustive search, torch's own e4m3 conversion, and the block scales' two rules."""
import numpy as np
import pytest
import torch

from oracle import mx_oracle as O


def _by_search(x, grid):
    best = np.abs(np.abs(x)[:, None] - grid[None, :])
    near = best == best.min(1, keepdims=True)
    idx = np.where(near, np.arange(len(grid)), -1)
    hi = idx.max(1)
    lo = np.where(near, np.arange(len(grid)), len(grid)).min(1)
    return np.where(hi == lo, lo, np.where(lo % 2 == 0, lo, hi))


@pytest.mark.parametrize("grid", [O.E2M1, O.E4M3[:127]], ids=["e2m1", "e4m3"])
def test_nearest_is_the_nearest(grid):
    rng = np.random.default_rng(1)
    mids = (grid[1:] + grid[:-1]) / 2
    x = np.concatenate([grid, mids, np.nextafter(mids, 0), np.nextafter(mids, 1e9),
                        rng.uniform(0, grid[-1], 2000), grid[-1] * np.array([1.01, 2, 100])])
    assert np.array_equal(O.nearest(x, grid), _by_search(x, grid))


def test_e4m3_matches_torch():
    b = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).float()
    b = b[torch.isfinite(b) & (b.abs() <= 448)]
    want = b.to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(O.e4m3_encode(b.numpy()), want)
    codes = torch.arange(256, dtype=torch.int32).to(torch.uint8).view(torch.float8_e4m3fn)
    assert np.array_equal(O.E4M3, codes.double().numpy(), equal_nan=True)


@pytest.mark.parametrize("a", [0.0, 1e-30, 1.0, 3.999, 4.0, 6.0, 7.9, 448.0, 3e38, 1e-45])
def test_block_exponent(a):
    x = np.zeros((1, 32))
    x[0, 5] = a = float(np.float32(a))
    codes, s = O.mx_quantize(x)
    e = int(s[0, 0]) - 127
    if a == 0:
        assert e == -127 and not codes.any()
    elif a > 2.0 ** -125:  # the scaled maximum lies in [4, 8)
        assert 4 <= a * 2.0 ** -e < 8
    assert O.mx_values(codes, s)[0, 5] == pytest.approx(min(a, 6 * 2.0 ** e), rel=0.26)


def test_cache_scale_is_the_least():
    for a in (0.0, 1e-30, 447.0, 448.0, 449.0, 1.0, 1e30):
        s = O.kv_scale(a)
        assert a <= 448 * s or s == 2.0 ** 60
        assert s == 2.0 ** -60 or a > 448 * s / 2


def test_a_grown_scale_moves_codes_exactly():
    """Three appends of growing rows to one page: codes that stay normal are unharmed."""
    c = O.Cache(1, 1, 16, 16)
    rng = np.random.default_rng(2)
    rows = [rng.uniform(1, 2, (1, 1, 16)) * 4.0 ** i for i in range(3)]
    for i, r in enumerate(rows):
        c.write(r, r, [[0]], [i], [1])
    k, _, _ = c.tokens([0], 3)
    alone = O.E4M3[O.e4m3_encode(rows[0] / O.kv_scale(rows[0].max()))] * O.kv_scale(rows[0].max())
    assert np.array_equal(k[0], alone[0])


def test_attention_matches_torch():
    rng = np.random.default_rng(3)
    q, k, v = rng.standard_normal((5, 4, 16)), rng.standard_normal((9, 2, 16)), rng.standard_normal((9, 2, 16))
    out, lse, _ = O.attention(q, k, v, np.ones(9, bool), True, 3, 0.25)
    tq, tk, tv = (torch.from_numpy(a) for a in (q, k, v))
    s = torch.einsum("nhd,lhd->hnl", tq, tk.repeat_interleave(2, 1)) * 0.25
    pos, j = torch.arange(4, 9)[:, None], torch.arange(9)
    s = s.masked_fill((j > pos) | (j <= pos - 3), -torch.inf)
    want = torch.einsum("hnl,lhd->nhd", torch.softmax(s, -1), tv.repeat_interleave(2, 1))
    assert np.allclose(out, want.numpy(), atol=1e-13)
    assert np.allclose(lse, torch.logsumexp(s, -1).t().numpy(), atol=1e-13)
    out, lse, _ = O.attention(q, k[:3], v[:3], np.ones(3, bool), True, 0, 0.25)
    assert not out[:2].any() and np.isneginf(lse[:2]).all() and out[2:].any()
