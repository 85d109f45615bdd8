"""MXFP4 on the GPU against the float64 oracle: codes and scale bytes exactly, products
within the bounds of float32 sums and one final rounding."""
import numpy as np
import pytest
import torch

from oracle import mx_oracle as O

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
# half a unit in the last place of one rounding to the output type (its epsilon is a whole one)
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in DTYPES}


@pytest.fixture(scope="module")
def mx():
    from perm_amd import mxfp4
    return mxfp4


def _rows(rows, k, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, k), generator=g) * torch.exp(torch.randn((k,), generator=g)) * scale
    return x.to(dtype)


def _check_quantized(mx, q, x):
    codes, scales = O.mx_quantize(x.double().cpu().numpy())
    got_s = mx.block_scales(q).cpu().numpy()
    assert np.array_equal(got_s, scales)
    got_c = O.mx_unpack(q.codes.cpu().numpy())
    bad = np.repeat(scales == 255, 32, axis=1)
    assert np.array_equal(np.where(bad, 0, got_c), np.where(bad, 0, codes))
    return O.mx_values(codes, scales)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k", [(1, 32), (1, 1024), (3, 96), (16, 128), (65, 160), (64, 4096),
                                    (130, 352), (257, 32)])
def test_quantize_and_decode(mx, rows, k, dtype):
    print(f"mx quantize [{rows}, {k}] {dtype}", flush=True)
    x = _rows(rows, k, dtype, rows + k).cuda()
    q = mx.quantize(x)
    want = _check_quantized(mx, q, x)
    # blocks past the end of a row are read by the product and must not be NaN
    tail = k // 32 % 4
    if tail:
        assert not (q.scales[-1, :, tail:] == 255).any()
    for out in DTYPES:
        got = mx.dequantize(q, out)
        exact = torch.from_numpy(want).cuda()
        assert torch.equal(got, exact.to(torch.float32).to(out))
    assert torch.equal(mx.roundtrip(x), mx.dequantize(q, dtype))


def test_every_bf16_value(mx):
    """Every finite bf16 as the largest of its block, with ties and tiny values beside it."""
    b = torch.arange(32768, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    b = b[torch.isfinite(b)].double()
    ratio = torch.tensor([1.0, -1.0] + [s * r for r in (0.0625, 0.125, 0.1875, 0.25, 0.3125, 0.375, 0.4375,
                                                       0.625, 0.875, 1e-4, 0.03125, 0.05, 0.2, 0.7, 0.99)
                                        for s in (1, -1)], dtype=torch.float64)
    x = (b[:, None] * ratio[None, :]).to(torch.float32).cuda()
    _check_quantized(mx, mx.quantize(x), x)
    xb = x.to(torch.bfloat16)
    _check_quantized(mx, mx.quantize(xb), xb)


@pytest.mark.parametrize("dtype", DTYPES)
def test_zeros_nan_and_infinity(mx, dtype):
    x = _rows(6, 128, dtype, 5)
    x[0] = 0
    x[1, 5] = float("nan")
    x[2, 40] = float("inf")
    x[3, 127] = -float("inf")
    x[4, 32:64] = -0.0
    tiny = torch.finfo(dtype).smallest_normal / 8
    x[5, 64:96] = tiny
    x = x.cuda()
    q = mx.quantize(x)
    want = _check_quantized(mx, q, x)
    got = mx.dequantize(q).cpu().numpy()
    assert np.array_equal(got, want.astype(np.float32), equal_nan=True)
    assert np.isnan(got[1, :32]).all() and np.isnan(got[2, 32:64]).all() and np.isnan(got[3, 96:]).all()
    assert np.isfinite(got).sum() == 6 * 128 - 96


def test_float32_extremes(mx):
    x = torch.zeros((4, 64))
    x[0, :4] = torch.tensor([3.4e38, -3.4e38, 1.0, 2.0 ** 126])
    x[1, :4] = torch.tensor([2.0 ** -149, 2.0 ** -127, -2.0 ** -126, 2.0 ** -125])
    x[2, 0], x[2, 33] = 2.0 ** -149, 1.9 * 2.0 ** -126
    x = x.cuda()
    q = mx.quantize(x)
    want = _check_quantized(mx, q, x)
    assert np.array_equal(mx.dequantize(q).cpu().numpy(), want.astype(np.float32))


def test_strides_alignment_and_dimensions(mx):
    base = _rows(40, 512, torch.bfloat16, 9).cuda()
    for x in (base[:, 64:192], base[::3, :96], base[5:, 8:136], base.t()[:96, :32],
              base.reshape(-1)[3:3 + 7 * 64].view(7, 64), base[:, 1:33], base[:1].expand(5, 512),
              base.view(4, 10, 512)[:, ::2, :160]):
        q = mx.quantize(x)
        flat = x.reshape(-1, x.shape[-1])
        _check_quantized(mx, q, flat)
        assert mx.roundtrip(x).shape == x.shape


def test_host_input_and_no_rows(mx):
    x = _rows(5, 64, torch.float32, 3)
    q = mx.quantize(x.numpy())
    _check_quantized(mx, q, x)
    assert isinstance(mx.roundtrip(x.numpy()), np.ndarray)
    e = mx.quantize(torch.empty((0, 64), device="cuda"))
    assert e.shape == (0, 64) and mx.dequantize(e).shape == (0, 64)
    assert mx.matmul(e, q).shape == (0, 5) and mx.matmul(q, e).shape == (5, 0)
    assert mx.linear(torch.empty((2, 0, 64), device="cuda"), q).shape == (2, 0, 5)


def _check_product(y, a, b, k, dtype):
    """|error| <= k 2^-23 sum |a b| (float32 sums in any order, twice over) + one rounding."""
    a, b = torch.from_numpy(a).cuda(), torch.from_numpy(b).cuda()
    want, mass = a @ b.t(), a.abs() @ b.abs().t()
    err = (y.double() - want).abs()
    u = HALF_ULP[dtype]
    small = 2.0 ** -25 if dtype == torch.float16 else 0.0  # below float16's normal range
    assert (err <= k * 2.0 ** -23 * mass * (1 + u) + u * want.abs() * 1.001 + small).all(), \
        (err / want.abs().clamp(min=1e-30)).max()


SHAPES = [(1, 1, 32), (1, 64, 128), (1, 1000, 1056), (2, 48, 4096), (3, 17, 96), (5, 130, 14336),
          (8, 256, 512), (15, 33, 160), (16, 16, 128), (17, 1000, 1056), (31, 257, 288),
          (33, 64, 4096), (64, 512, 1024), (65, 130, 352), (100, 96, 2080), (128, 128, 128),
          (129, 255, 544), (200, 1030, 256), (256, 256, 256), (257, 300, 1184), (520, 130, 640),
          (1030, 515, 416)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_matmul_and_linear(mx, m, n, k):
    print(f"mx product {m} x {n} x {k}", flush=True)
    x = _rows(m, k, torch.bfloat16, m + n).cuda()
    w = _rows(n, k, torch.float32, n + k, 0.02).cuda()
    qx, qw = mx.quantize(x), mx.quantize(w)
    a = O.mx_values(*O.mx_quantize(x.double().cpu().numpy()))
    b = O.mx_values(*O.mx_quantize(w.double().cpu().numpy()))
    for dtype in DTYPES:
        _check_product(mx.matmul(qx, qw, dtype), a, b, k, dtype)
    _check_product(mx.linear(x, qw), a, b, k, torch.bfloat16)
    _check_product(mx.linear(x, qw, torch.float32), a, b, k, torch.float32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [1, 7, 20, 300])
def test_linear_types(mx, m, dtype):
    x = _rows(m, 1120, dtype, m).cuda()
    w = mx.quantize(_rows(200, 1120, torch.float32, 77, 0.02).cuda())
    a = O.mx_values(*O.mx_quantize(x.double().cpu().numpy()))
    b = O.mx_values(O.mx_unpack(w.codes.cpu().numpy()), mx.block_scales(w).cpu().numpy())
    y = mx.linear(x, w)
    assert y.dtype == dtype
    _check_product(y, a, b, 1120, dtype)
    # rows of a wider tensor, and leading dimensions
    wide = torch.zeros((m, 2048), dtype=dtype, device="cuda")
    wide[:, 512:1632] = x
    assert torch.equal(mx.linear(wide[:, 512:1632], w), y)
    assert torch.equal(mx.linear(x.view(1, m, 1120), w), y[None])


@pytest.mark.parametrize("m", [1, 9, 40, 260])
def test_scales_over_the_whole_range(mx, m):
    """Random codes under any exponent: products of 2^(ea + eb) inside float32's range, and a
    NaN scale that reaches its own row or column and nothing else."""
    g = torch.Generator().manual_seed(m)
    n, k = 100, 416
    ts, vals = [], []
    for rows, lo, hi in ((m, 60, 190), (n, 100, 150)):
        codes = torch.randint(0, 256, (rows, k // 2), generator=g).to(torch.uint8)
        by_row = torch.randint(lo, hi, (rows, k // 32), generator=g).to(torch.uint8)
        by_row[rows // 2, 3] = 255
        full = torch.zeros((-(-rows // 64) * 64, 4 * -(-k // 128)), dtype=torch.uint8)
        full[:rows, : k // 32] = by_row
        s = full.view(-1, 4, 16, -(-k // 128), 4).permute(3, 0, 4, 2, 1).contiguous()
        ts.append(mx.MxTensor(codes.cuda(), s.cuda()))
        assert torch.equal(mx.block_scales(ts[-1]).cpu(), by_row)
        vals.append(O.mx_values(O.mx_unpack(codes.numpy()), by_row.numpy()))
    y = mx.matmul(*ts, torch.float32)
    nan = torch.zeros((m, n), dtype=torch.bool)
    nan[m // 2], nan[:, n // 2] = True, True
    assert torch.equal(y.isnan().cpu(), nan)
    a, b = (np.nan_to_num(v) for v in vals)
    y = torch.where(y.isnan(), torch.from_numpy(a).cuda() @ torch.from_numpy(b).cuda().t(), y.double())
    _check_product(y, a, b, k, torch.float32)


def test_offsets_past_32_bits(mx):
    """3.2e9 values: the last rows' codes lie past 2^30 and their inputs past 2^32 bytes."""
    rows, k = 99000, 32768
    x = torch.zeros((rows, k), dtype=torch.bfloat16, device="cuda")
    tail = _rows(40, k, torch.bfloat16, 4).cuda()
    x[-40:] = tail
    q = mx.quantize(x)
    del x
    y = mx.dequantize(q, torch.bfloat16)
    assert torch.equal(y[-40:], mx.roundtrip(tail)) and not y[:64].any()
    del y
    w = mx.quantize(tail[:3])
    got = mx.matmul(w, q)
    assert torch.equal(got[:, -40:], mx.matmul(w, mx.quantize(tail))) and not got[:, :64].any()


def test_other_stream_and_repeat(mx):
    x = _rows(300, 1024, torch.bfloat16, 1).cuda()
    w = mx.quantize(_rows(500, 1024, torch.float32, 2, 0.02).cuda())
    want = mx.linear(x, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [mx.linear(x, w) for _ in range(4)]
    torch.cuda.current_stream().wait_stream(s)
    for y in got:
        assert torch.equal(y, want)


def test_refusals(mx):
    x = _rows(4, 64, torch.bfloat16, 1).cuda()
    q = mx.quantize(x)
    with pytest.raises(ValueError):
        mx.quantize(x[:, :48])
    with pytest.raises(ValueError):
        mx.quantize(x[:, :0])
    with pytest.raises(TypeError):
        mx.quantize(x.double())
    with pytest.raises(TypeError):
        mx.dequantize(q, torch.int32)
    with pytest.raises(ValueError):
        mx.linear(x[:, :32], q)
    with pytest.raises(ValueError):
        mx.linear(x.cpu(), q)
    with pytest.raises(TypeError):
        mx.linear(x, q, torch.int8)
    with pytest.raises(ValueError):
        mx.matmul(q, mx.quantize(x[:, :32]))
    with pytest.raises(ValueError):
        mx.matmul(q, mx.MxTensor(q.codes, q.scales[:, :, :3].contiguous()))
    with pytest.raises(TypeError):
        mx.matmul(q, mx.MxTensor(q.codes.float(), q.scales))
    with pytest.raises(ValueError):
        mx.matmul(q, mx.MxTensor(q.codes.t(), q.scales))


@pytest.mark.parametrize("m,n,k", [(33, 100, 14336), (64, 70, 6144), (70, 4100, 3104), (130, 66, 8224),
                                   (300, 1100, 1056), (600, 4097, 288), (1030, 12400, 160), (257, 15000, 128)])
def test_tiles_and_splits(mx, m, n, k):
    """Sizes that take each tile of the product, columns split in several parts among them."""
    x = _rows(m, k, torch.bfloat16, m).cuda()
    w = _rows(n, k, torch.float32, n, 0.02).cuda()
    qx, qw = mx.quantize(x), mx.quantize(w)
    a = mx.dequantize(qx).double().cpu().numpy()
    b = mx.dequantize(qw).double().cpu().numpy()
    for dtype in DTYPES:
        y = mx.matmul(qx, qw, dtype)
        _check_product(y, a, b, k, dtype)
        assert torch.equal(y, mx.matmul(qx, qw, dtype))
    assert torch.equal(mx.linear(x, qw), mx.matmul(qx, qw))


@pytest.mark.parametrize("m,n,k", [(1, 16, 32768), (31, 40, 1056), (32, 1000, 1024), (17, 50, 96), (2, 8200, 4096)])
def test_rows_quantized_in_the_product(mx, m, n, k):
    """Few rows: the codes made inside the product are those of quantize()."""
    x = _rows(m, k, torch.bfloat16, m + k).cuda()
    x[m // 2, 5] = float("nan")
    w = mx.quantize(_rows(n, k, torch.float32, n, 0.02).cuda())
    y = mx.linear(x, w)
    want = mx.matmul(mx.quantize(x), w)
    assert y[m // 2].isnan().all() and y.isnan().sum() == n
    a = np.nan_to_num(mx.dequantize(mx.quantize(x)).double().cpu().numpy())
    b = mx.dequantize(w).double().cpu().numpy()
    a[m // 2] = 0
    _check_product(torch.where(y.isnan(), 0, y), a, b, k, torch.bfloat16)
    _check_product(torch.where(want.isnan(), 0, want), a, b, k, torch.bfloat16)


@pytest.mark.parametrize("m,n,k", [(1, 48, 24576), (9, 333, 1024), (16, 1000, 1536), (23, 77, 1056), (32, 130, 768),
                                   (5, 24000, 1024)])
def test_rows_quantized_by_more_waves(mx, m, n, k):
    """The largest shares that are quantized inside the product, by eight and sixteen waves."""
    test_rows_quantized_in_the_product(mx, m, n, k)
