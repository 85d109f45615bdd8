"""Every block of a product, exactly. With all scales equal, products of e2m1 codes are multiples
of 1/4 below 2^24 / 4 in sum, so float32 holds every sum in any order; with one block of a row
not zero, the same holds under any scales. No tolerance: a block that is lost, taken twice or scaled
by another's exponent changes bits."""
import numpy as np
import pytest
import torch

from oracle import mx_oracle as O

pytestmark = pytest.mark.gpu


def _packed(codes, by_row):
    """MxTensor of one code an entry [rows, k] and scale bytes [rows, k / 32] (numpy)."""
    from perm_amd import mxfp4
    rows, k = codes.shape
    full = np.zeros((-(-rows // 64) * 64, 4 * -(-k // 128)), np.uint8)
    full[:rows, : k // 32] = by_row
    s = full.reshape(-1, 4, 16, full.shape[1] // 4, 4).transpose(3, 0, 4, 2, 1)
    return mxfp4.MxTensor(torch.from_numpy(codes[:, ::2] | codes[:, 1::2] << 4).cuda(),
                          torch.from_numpy(np.ascontiguousarray(s)).cuda())


def _product(a, b):
    return (torch.from_numpy(a).cuda() @ torch.from_numpy(b).cuda().t()).cpu().numpy()


# few rows with one and two tiles of either operand, then tiles of 64, 128 and 256, whole and in splits
SHAPES = [(1, 48, 32768), (16, 40, 24608), (9, 8200, 4128), (17, 40, 32768), (31, 9001, 2080), (32, 8192, 4096),
          (33, 100, 14336), (64, 70, 32768), (130, 66, 8224), (128, 4096, 14336), (300, 1100, 1056), (1030, 12400, 160),
          (520, 2100, 6176)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_all_blocks_count(m, n, k):
    from perm_amd import mxfp4
    print(f"all blocks {m} x {n} x {k}", flush=True)
    rng = np.random.default_rng(m + n)
    ca, cb = (rng.integers(0, 16, (r, k)).astype(np.uint8) for r in (m, n))
    one = [np.full((r, k // 32), 127, np.uint8) for r in (m, n)]
    a, b = _packed(ca, one[0]), _packed(cb, one[1])
    want = _product(O.mx_values(ca, one[0]), O.mx_values(cb, one[1]))
    assert np.abs(want).max() < 2 ** 22 and k * 36 < 2 ** 22
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        got = mxfp4.matmul(a, b, dtype)
        assert torch.equal(got.cpu(), torch.from_numpy(want).to(torch.float32).to(dtype))


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_one_block_a_row(m, n, k):
    from perm_amd import mxfp4
    print(f"one block {m} x {n} x {k}", flush=True)
    rng = np.random.default_rng(m + k)
    blocks = k // 32
    cb = rng.integers(0, 16, (n, k)).astype(np.uint8)
    sb, sa = rng.integers(110, 140, (n, blocks)).astype(np.uint8), rng.integers(110, 140, (m, blocks)).astype(np.uint8)
    b, vb = _packed(cb, sb), torch.from_numpy(O.mx_values(cb, sb)).cuda().view(n, blocks, 32)
    code = rng.integers(1, 16, (m, 32)).astype(np.uint8)
    # every block in turn, spread over the rows
    for first in range(0, blocks, m):
        at = (first + np.arange(m)) % blocks
        ca = np.zeros((m, blocks, 32), np.uint8)
        ca[np.arange(m), at] = code
        ca = ca.reshape(m, k)
        va = torch.from_numpy(O.mx_values(ca, sa)).cuda().view(m, blocks, 32)[torch.arange(m), torch.from_numpy(at)]
        got = mxfp4.matmul(_packed(ca, sa), b, torch.float32)
        want = torch.stack([vb[:, x] @ va[i] for i, x in enumerate(at)])
        assert torch.equal(got, want.to(torch.float32)), first


# (fused: whether the rows are quantized inside the product)
LINEAR = [(1, 48, 24576, True), (2, 40, 12288, True), (5, 2000, 1024, True), (16, 1000, 1536, True), (17, 1000, 1056, True),
          (24, 77, 1024, True), (32, 130, 768, True), (31, 333, 768, True), (1, 16, 32768, False), (32, 1000, 1024, False),
          (17, 50, 1472, False), (31, 9001, 288, True), (2, 8200, 4096, True), (3, 14336, 8192, False)]


@pytest.mark.parametrize("m,n,k,fused", LINEAR)
def test_rows_quantized_on_the_way(m, n, k, fused):
    """linear() on values that MXFP4 holds exactly: each block's largest is 4 or 6."""
    from perm_amd import _lib, mxfp4
    print(f"linear blocks {m} x {n} x {k} {fused}", flush=True)
    assert (_lib.load().cp_mx4_linear_ws_bytes(m, n, k) == 0) == fused
    rng = np.random.default_rng(m * n)
    ca, cb = (rng.integers(0, 16, (r, k)).astype(np.uint8) for r in (m, n))
    ca[:, ::32] = 6 + rng.integers(0, 2, (m, k // 32))
    one = [np.full((r, k // 32), 127, np.uint8) for r in (m, n)]
    x = O.mx_values(ca, one[0])
    want = torch.from_numpy(_product(x, O.mx_values(cb, one[1])))
    w = _packed(cb, one[1])
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        got = mxfp4.linear(torch.from_numpy(x).to(dtype).cuda(), w, torch.float32)
        assert torch.equal(got.cpu(), want.to(torch.float32)), dtype
    # one block of each row, under scales of its own
    sb = rng.integers(110, 140, (n, k // 32)).astype(np.uint8)
    w, vb = _packed(cb, sb), torch.from_numpy(O.mx_values(cb, sb)).cuda().view(n, -1, 32)
    blocks = k // 32
    for first in range(0, blocks, m):
        at = (first + np.arange(m)) % blocks
        y = np.zeros((m, blocks, 32))
        y[np.arange(m), at] = x.reshape(m, blocks, 32)[np.arange(m), at] * 2.0 ** rng.integers(-20, 20, (m, 1))
        got = mxfp4.linear(torch.from_numpy(y.reshape(m, k)).to(torch.bfloat16).cuda(), w, torch.float32)
        yd = torch.from_numpy(y[np.arange(m), at]).cuda()
        want = torch.stack([vb[:, b] @ yd[i] for i, b in enumerate(at)])
        assert torch.equal(got, want.to(torch.float32)), first


@pytest.mark.parametrize("m,n,k", [(17, 8200, 1056), (31, 9001, 288), (32, 14336, 4096), (18, 8193, 160), (16, 8206, 416)])
def test_few_rows_and_many_columns(m, n, k):
    """Two tiles of rows times two of columns a wave, a NaN scale in a row of each tile."""
    from perm_amd import mxfp4
    print(f"two by two {m} x {n} x {k}", flush=True)
    rng = np.random.default_rng(n)
    ca, cb = (rng.integers(0, 16, (r, k)).astype(np.uint8) for r in (m, n))
    sa, sb = np.full((m, k // 32), 126, np.uint8), np.full((n, k // 32), 128, np.uint8)
    va, vb = O.mx_values(ca, sa), O.mx_values(cb, sb)
    want = torch.from_numpy(_product(va, vb)).to(torch.float32)
    nan = torch.zeros((m, n), dtype=torch.bool)
    for r, block in ((3, 0), (m - 1, k // 32 - 1)):
        sa[r, block] = 255
        nan[r] = True
    for r, block in ((0, k // 32 - 1), (n // 32 * 32 - 16, 1), (n - 1, 0)):
        sb[r, block] = 255
        nan[:, r] = True
    a, b = _packed(ca, sa), _packed(cb, sb)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        got = mxfp4.matmul(a, b, dtype).cpu()
        assert torch.equal(got.isnan(), nan)
        assert torch.equal(torch.where(nan, 0, got), torch.where(nan, 0, want).to(dtype))
