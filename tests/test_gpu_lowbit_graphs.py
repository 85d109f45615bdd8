"""The low-bit operators in a captured graph where they use workspaces: a product in splits, rows
quantized ahead of it, attention in splits with its join. Replayed with new contents, every
replay against the eager calls."""
import numpy as np
import pytest
import torch

from test_gpu_kvcache import _filled_cache, _i32, kv  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 40])
def test_a_step_replays(kv, rows):  # noqa: F811
    from perm_amd import _lib, mxfp4
    rng = np.random.default_rng(rows)
    heads, d, hq, k = 2, 64, 8, 14336
    lens = [3000, 900]
    c, _, table = _filled_cache(kv, rng, lens, heads, d, 16)
    cap = table.shape[1]
    g = torch.Generator(device="cuda").manual_seed(rows)
    w = mxfp4.quantize(torch.randn((hq * d, k), generator=g, device="cuda") * 0.02)
    x = torch.randn((2 * rows, k), generator=g, device="cuda").to(torch.bfloat16)
    kvs = torch.randn((2 * rows, 2 * heads, d), generator=g, device="cuda").to(torch.bfloat16)
    filled, held, off = _i32([2900 - rows, 800 - rows]), _i32([2900, 800]), _i32([0, rows, 2 * rows])
    t = _i32(table)
    assert _lib.load().cp_mx4_linear_ws_bytes(2 * rows, hq * d, k) > 0
    assert rows == 1 or _lib.load().cp_mx4_matmul_ws_bytes(2 * rows, hq * d, k) > 0
    desc = kv._desc(c)
    import ctypes
    assert _lib.load().cp_kv_attention_ws_bytes(ctypes.byref(desc), 2 * rows, hq, 2, cap, 1, 0) > 0

    def step():
        q = mxfp4.linear(x, w).view(2 * rows, hq, d)
        kv.write(c, kvs[:, :heads], kvs[:, heads:], t, filled, off)
        out, lse = kv.attention(q, c, t, held, off, return_lse=True)
        k16, v16 = kv.read(c, t, off, 2 * rows)
        return q, out, lse, k16, v16, mxfp4.roundtrip(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        got = [y.clone() for y in outs]
        eager = step()
        for a, b in zip(got, eager):
            assert torch.equal(a, b), i
        assert torch.isfinite(got[1]).all() and got[1].any()
        x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        kvs.copy_(torch.randn(kvs.shape, generator=g, device="cuda"))
        filled.add_(1)
        held.add_(1)
        if i == 1:
            off.copy_(_i32([0, 0, rows]))  # fewer rows: the rest has no sequence
