"""Attention in tiles of 128 rows, which calls of many rows over long tables take: the cases
and bounds of the short tables' tests, with tables that go on, without pages, until rows x
query heads x tokens pass the 2^24 above which these tiles are used."""
import numpy as np
import pytest
import torch

from oracle import mx_oracle as O
from test_gpu_kvcache import (HALF_ULP, _check_attention, _filled_cache, _i32, _offsets, kv)  # noqa: F401

pytestmark = pytest.mark.gpu


def _long(table, rows, hq, block):
    more = 2 ** 24 // (rows * hq * block) + 1
    return np.concatenate([table, np.full((table.shape[0], more), -1)], axis=1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("block,heads,d,group", [(16, 2, 128, 2), (64, 1, 64, 4), (32, 1, 112, 3), (128, 1, 256, 8),
                                                 (16, 1, 16, 5), (32, 4, 80, 4)])
def test_ragged_prompts(kv, block, heads, d, group, causal, dtype):  # noqa: F811
    print(f"attend tiles {block} {heads} {d} {group} {causal} {dtype}", flush=True)
    rng = np.random.default_rng(block + group)
    lens, counts = [150, 70, 5, 33, 0, 200], [150, 1, 9, 0, 3, 77]
    c, o, table = _filled_cache(kv, rng, lens, heads, d, block)
    _check_attention(kv, o, c, _long(table, sum(counts), heads * group, block), lens, counts, heads * group, dtype,
                     rng, causal)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_split_and_whole(kv, dtype):  # noqa: F811
    """The tokens split (few row tiles), and whole (more row tiles than the CUs hold)."""
    rng = np.random.default_rng(21)
    c, o, table = _filled_cache(kv, rng, [1500, 40], 1, 64, 16)
    _check_attention(kv, o, c, _long(table, 303, 4, 16), [1500, 40], [300, 3], 4, dtype, rng)
    c, o, table = _filled_cache(kv, rng, [700], 8, 64, 64)
    q = torch.from_numpy(rng.standard_normal((700, 64, 64))).to(dtype).cuda()
    out = kv.attention(q, c, _i32(table), _i32([700]), _offsets([700]))  # 700 x 64 x 704 > 2^24
    k, v, have = o.tokens(table[0], 700)
    for h in (0, 37, 63):
        want, _, bound = O.attention(q[:, h:h + 1].double().cpu().numpy(), k[:, h // 8:h // 8 + 1],
                                     v[:, h // 8:h // 8 + 1], have, True, 0, 0.125)
        err = np.abs(out[:, h:h + 1].double().cpu().numpy() - want)
        assert (err <= bound + HALF_ULP[dtype] * np.abs(want) * 1.01 + 2.0 ** -24).all(), h


@pytest.mark.parametrize("causal", [True, False])
def test_windows(kv, causal):  # noqa: F811
    """2048 rows of 16 heads, each seeing 400 tokens (not causal: and those after it)."""
    rng = np.random.default_rng(22)
    n, window = 2048, 400
    c, o, table = _filled_cache(kv, rng, [n + 50], 1, 64, 32)
    q = torch.from_numpy(rng.standard_normal((n, 16, 64))).to(torch.bfloat16).cuda()
    out = kv.attention(q, c, _i32(table), _i32([n + 50]), _offsets([n]), causal=causal, window=window)
    k, v, have = o.tokens(table[0], n + 50)
    for h in (0, 11):
        want, _, bound = O.attention(q[:, h:h + 1].double().cpu().numpy(), k, v, have, causal, window, 0.125)
        err = np.abs(out[:, h:h + 1].double().cpu().numpy() - want)
        assert (err <= bound + HALF_ULP[torch.bfloat16] * np.abs(want) * 1.01 + 2.0 ** -24).all(), h


def test_scale_and_large_scores(kv):  # noqa: F811
    rng = np.random.default_rng(23)
    c, o, table = _filled_cache(kv, rng, [90, 200], 1, 64, 16, grow=30.0)
    t = _long(table, 93, 2, 16)
    _check_attention(kv, o, c, t, [90, 200], [90, 3], 2, torch.bfloat16, rng, scale=1.0)
    _check_attention(kv, o, c, t, [90, 200], [90, 3], 2, torch.float16, rng, scale=1e-4)
    for p in range(o.vs.shape[0]):
        o.vs[p] = c.v_scale[p] = 2.0 ** int(rng.integers(-30, 8))
    _check_attention(kv, o, c, t, [90, 200], [90, 50], 2, torch.bfloat16, rng)


def test_unseen_tokens_do_not_reach_a_row(kv):  # noqa: F811
    rng = np.random.default_rng(24)
    lens = [37, 100]
    c, o, table = _filled_cache(kv, rng, lens, 2, 64, 16)
    for buf in (o.k, o.v):
        page, slot = table[0][37 // 16], 37 % 16
        buf[page, :, slot:] = 127
        buf[table[0][3]] = 255
        buf[table[1][100 // 16], :, 100 % 16:] = 127
    o.v[table[1][85 // 16], 0, 85 % 16, 7] = 127   # rows before token 85 do not see it
    o.v[table[1][2], 1, 5, 9] = 255                # token 37
    o.k[table[1][90 // 16], 0, 90 % 16, 3] = 127
    c.k.copy_(torch.from_numpy(o.k))
    c.v.copy_(torch.from_numpy(o.v.swapaxes(2, 3).copy()))
    for causal, dtype in ((True, torch.bfloat16), (False, torch.float16)):
        _check_attention(kv, o, c, _long(table, 137, 8, 16), lens, [37, 100], 8, dtype, rng, causal=causal)


def test_missing_pages(kv):  # noqa: F811
    rng = np.random.default_rng(25)
    c, o, table = _filled_cache(kv, rng, [120, 64, 40], 2, 64, 16)
    table = table.copy()
    table[0][1], table[0][4], table[1][:] = -1, o.k.shape[0], -5
    _check_attention(kv, o, c, _long(table, 200, 4, 16), [120, 64, 40], [120, 40, 40], 4, torch.bfloat16, rng)


def test_offsets_past_32_bits(kv):  # noqa: F811
    """Pages at the end of a cache of 4.3 GB each of K and V."""
    pages, heads, d, block = 264000, 8, 128, 16
    rng = np.random.default_rng(26)
    c, small = kv.new(pages, heads, d, block), kv.new(8, heads, d, block)
    table = rng.permutation(8)[None, :]
    k, v = (torch.from_numpy(rng.standard_normal((120, heads, d))).to(torch.bfloat16).cuda() for _ in range(2))
    kv.write(small, k, v, _i32(table), _i32([0]), _i32([0, 120]))
    kv.write(c, k, v, _i32(table + pages - 8), _i32([0]), _i32([0, 120]))
    q = torch.from_numpy(rng.standard_normal((100, 16, d))).to(torch.bfloat16).cuda()
    assert torch.equal(kv.attention(q, c, _i32(_long(table + pages - 8, 100, 16, block)), _i32([120]), _i32([0, 100])),
                       kv.attention(q, small, _i32(_long(table, 100, 16, block)), _i32([120]), _i32([0, 100])))
