"""Rows that no sequence has (a padded batch): 0 with a log-sum of -inf, whatever memory held."""
import numpy as np
import pytest
import torch

from test_gpu_kvcache import _check_attention, _filled_cache, _i32, _offsets, kv  # noqa: F401
from test_gpu_kvcache_tiles import _long

pytestmark = pytest.mark.gpu


def _dirty(*shapes):
    """Leaves the allocator blocks of these sizes that hold NaN."""
    held = [torch.full(s, float("nan"), dtype=t, device="cuda") for s, t in shapes for _ in range(4)]
    torch.cuda.synchronize()
    del held


@pytest.mark.parametrize("tiles,top", [(False, 60), (False, 5000), (True, 200)], ids=["few", "split", "tiles"])
@pytest.mark.parametrize("before,after", [(0, 1), (0, 300), (7, 0), (33, 90)])
def test_attention(kv, tiles, top, before, after):  # noqa: F811
    print(f"padding {tiles} {top} {before} {after}", flush=True)
    rng = np.random.default_rng(before + after + top)
    heads, d, hq = 2, 80, 6
    lens = [top, 41, 9]
    counts = [top, 41, 9] if tiles else [1, 0, 9]
    c, o, table = _filled_cache(kv, rng, lens, heads, d, 16)
    n = sum(counts)
    rows = before + n + after
    t = _i32(_long(table, rows, hq, 16) if tiles else table)
    q = torch.from_numpy(rng.standard_normal((rows, hq, d))).to(torch.bfloat16).cuda()
    want, wlse = kv.attention(q[before:before + n].contiguous(), c, t, _i32(lens), _offsets(counts), return_lse=True)
    _dirty(((rows, hq, d), torch.bfloat16), ((rows, hq), torch.float32), ((rows * hq * d * 16,), torch.float32))
    out, lse = kv.attention(q, c, t, _i32(lens), _offsets(counts) + before, return_lse=True)
    none = torch.ones(rows, dtype=torch.bool, device="cuda")
    none[before:before + n] = False
    assert not out[none].any() and torch.isneginf(lse[none]).all()
    assert torch.allclose(out[~none].float(), want.float(), atol=0.02, rtol=0.02)
    assert torch.allclose(lse[~none], wlse, atol=1e-3)


def test_a_batch_of_padding_alone(kv):  # noqa: F811
    rng = np.random.default_rng(3)
    c, o, table = _filled_cache(kv, rng, [40, 20], 2, 64, 16)
    for rows in (1, 50, 3000):
        q = torch.from_numpy(rng.standard_normal((rows, 4, 64))).to(torch.float16).cuda()
        _dirty(((rows, 4, 64), torch.float16), ((rows, 4), torch.float32))
        for t, lens, off in ((table, [40, 20], [0, 0, 0]), (table[:0], [], [0])):
            out, lse = kv.attention(q, c, _i32(t), _i32(lens), _i32(off), return_lse=True)
            assert not out.any() and torch.isneginf(lse).all()
            k, v = kv.read(c, _i32(t), _i32(off), rows)
            assert not k.any() and not v.any()


def test_a_sequence_that_passes_the_rows(kv):  # noqa: F811
    """Its rows are 0 in attention; reading gives those that there are."""
    rng = np.random.default_rng(4)
    c, o, table = _filled_cache(kv, rng, [40, 90], 2, 64, 16)
    q = torch.from_numpy(rng.standard_normal((30, 4, 64))).to(torch.bfloat16).cuda()
    for t in (table, _long(table, 30, 4, 16)):
        _dirty(((30, 4, 64), torch.bfloat16), ((30, 4), torch.float32))
        out, lse = kv.attention(q, c, _i32(t), _i32([40, 90]), _i32([0, 10, 60]), return_lse=True)
        assert out[:10].any(2).all() and not out[10:].any() and torch.isneginf(lse[10:]).all()
    k0, v0 = kv.read(c, _i32(table), _i32([0, 40, 130]), 130)
    _dirty(((57, 2, 64), torch.bfloat16))
    k, v = kv.read(c, _i32(table), _i32([0, 40, 130]), 57)
    assert torch.equal(k, k0[:57]) and torch.equal(v, v0[:57])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("before,after", [(0, 1), (0, 1000), (19, 0), (5, 40)])
def test_read(kv, before, after, dtype):  # noqa: F811
    rng = np.random.default_rng(before + after)
    lens = [37, 0, 100]
    c, o, table = _filled_cache(kv, rng, lens, 3, 48, 32)
    want = kv.read(c, _i32(table), _offsets(lens), 137, dtype)
    total = before + 137 + after
    _dirty(((total, 3, 48), dtype))
    got = kv.read(c, _i32(table), _offsets(lens) + before, total, dtype)
    for g, w in zip(got, want):
        assert torch.equal(g[before:before + 137], w)
        assert not g[:before].any() and not g[before + 137:].any()
