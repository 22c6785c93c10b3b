"""GPU: microscaled 4-bit quantisation and products against the 64-bit statements of mxfp4_reference.py.  Quantisation
and its inverse are bit-exact; products of one exponent are exact in f32, others within the bound of an f32 sum."""
import threading

import numpy as np
import pytest
import torch

import mxfp4_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def B():
    import bsir
    bsir.lib()
    yield bsir
    assert bsir.device_error() == 0


def _values(rows, cols, dtype, seed):
    """Normal values over many exponents, with zeros, ties, tiny and huge blocks, a NaN and infinities."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp2(torch.randint(-6, 7, (rows, cols), generator=g).float())
    x[torch.rand(rows, cols, generator=g) < 0.05] = 0.0
    pick = lambda: (int(torch.randint(0, rows, (1,), generator=g)), int(torch.randint(0, cols, (1,), generator=g)))
    x[pick()] = float("nan")
    x[pick()] = float("inf")
    x[pick()] = -float("inf")
    r = pick()[0]
    x[r] = 0.0
    r = pick()[0]
    x[r] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0]).repeat(cols // 8 + 1)[:cols]      # ties
    if dtype == torch.float32:
        r = pick()[0]
        x[r] = torch.randn(cols, generator=g) * 2.0 ** -126
        r = pick()[0]
        x[r] = torch.randn(cols, generator=g).clamp(-1.9, 1.9) * 2.0 ** 127
    if dtype == torch.float16:
        r = pick()[0]
        x[r] = torch.randint(-9, 10, (cols,), generator=g) * 2.0 ** -24
    return x.to(dtype)


def _same(got, want_values):
    got = got.cpu().double().numpy()
    assert np.array_equal(got, want_values, equal_nan=True), np.argwhere(~((got == want_values) | (np.isnan(got) & np.isnan(want_values))))[:5]


SHAPES = [(1, 1), (1, 32), (3, 31), (5, 33), (33, 5), (2, 64), (64, 64), (7, 1000), (257, 70), (130, 520), (31, 4097)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quant_rows(B, rows, cols, dtype):
    x = _values(rows, cols, dtype, rows * 1000 + cols)
    wq, ws, wv = R.quant(x)
    q, s = B.quant_mxfp4(x.cuda())
    assert np.array_equal(s.cpu().numpy(), ws)
    _same(torch.from_numpy(R.decode(q, s, cols)), wv)
    # the signs of zeros too, and the unused half byte
    nan = np.repeat(ws == 255, 32, axis=1)[:, :cols]
    got = np.stack((q.cpu().numpy() & 15, q.cpu().numpy() >> 4), -1).reshape(rows, -1)
    want = np.stack((wq & 15, wq >> 4), -1).reshape(rows, -1)
    assert np.array_equal(got[:, :cols], np.where(nan, 0, want[:, :cols])) and (got[:, cols:] == 0).all()
    _same(B.dequant_mxfp4(q, s, dtype, cols=cols), wv)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quant_columns_and_both(B, rows, cols, dtype):
    x = _values(rows, cols, dtype, rows * 1000 + cols + 7)
    _, ws, wv = R.quant(x)
    _, wst, wvt = R.quant(x.t())
    q, s = B.quant_mxfp4(x.cuda(), axis=0)
    assert tuple(q.shape) == (cols, (rows + 1) // 2) and np.array_equal(s.cpu().numpy(), wst)
    _same(torch.from_numpy(R.decode(q, s, rows)), wvt)
    if rows % 2:
        assert (q[:, -1] >> 4 == 0).all()
    q2, s2, qt, st = B.quant_mxfp4_both(x.cuda())
    assert torch.equal(qt, q) and torch.equal(st, s)
    assert np.array_equal(s2.cpu().numpy(), ws)
    _same(torch.from_numpy(R.decode(q2, s2, cols)), wv)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_quant_ends_of_the_range(B, dtype):
    """Blocks at every exponent of the type, subnormals and the largest values among them, both ways."""
    g = torch.Generator().manual_seed(0)
    lo, hi = (-24, 15) if dtype == torch.float16 else (-140, 127)
    e = torch.arange(lo, hi + 1).double()
    x = torch.ldexp(torch.rand(len(e), 32, generator=g).double() * 1.98 - 0.99, e[:, None]).to(dtype)
    _, ws, wv = R.quant(x)
    q, s = B.quant_mxfp4(x.cuda())
    assert np.array_equal(s.cpu().numpy(), ws)
    _same(torch.from_numpy(R.decode(q, s, 32)), wv)
    _same(B.dequant_mxfp4(q, s, dtype), wv)
    qt, st = B.quant_mxfp4(x.t().contiguous().cuda(), axis=0)
    assert torch.equal(qt, q) and torch.equal(st, s)


def test_quant_beyond_32_bits(B):
    """9.7e9 elements: element numbers, byte offsets and the launch's own indices pass 2^31 and 2^32."""
    rows, cols = 9, 1 << 30
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    spots = [(0, 5), (3, cols - 1), (8, 7), (8, cols - 33), (8, cols - 1)]
    for i, (r, c) in enumerate(spots):
        x[r, c] = i + 1.0
    q, s = B.quant_mxfp4(x)
    for i, (r, c) in enumerate(spots):
        _, byte, v = R.quant(x[r:r + 1, c // 32 * 32:c // 32 * 32 + 32])
        assert s[r, c // 32].item() == byte[0, 0]
        assert R.decode(q[r:r + 1, c // 32 * 16:c // 32 * 16 + 16], s[r:r + 1, c // 32:c // 32 + 1], 32)[0, c % 32] == v[0, c % 32]
    assert sum(int((q[r] != 0).sum()) for r in range(rows)) == len(spots)
    y = B.dequant_mxfp4(q, s, torch.bfloat16)
    assert all(y[r, c].item() == {1: 1, 2: 2, 3: 3, 4: 4, 5: 4}[i + 1] for i, (r, c) in enumerate(spots))


@pytest.mark.parametrize("offset,pitch", [(0, 0), (1, 3), (8, 8), (2, 0)])
def test_quant_strides_and_alignment(B, offset, pitch):
    rows, cols = 9, 96
    buf = _values(rows, cols + offset + pitch, torch.bfloat16, 3).cuda()
    x = buf[:, offset:offset + cols]
    _, ws, wv = R.quant(x)
    codes = torch.full((rows, 61), 0xee, dtype=torch.uint8, device="cuda")
    exps = torch.full((rows, 5), 0xee, dtype=torch.uint8, device="cuda")
    q, s = B.quant_mxfp4(x, q=codes[:, 3:51], scale=exps[:, 1:4])
    assert np.array_equal(s.cpu().numpy(), ws)
    _same(torch.from_numpy(R.decode(q, s, cols)), wv)
    assert (codes[:, :3] == 0xee).all() and (codes[:, 51:] == 0xee).all() and (exps[:, 0] == 0xee).all() and (exps[:, 4] == 0xee).all()
    out = torch.zeros(rows, cols + 5, dtype=torch.float16, device="cuda")
    B.dequant_mxfp4(q, s, out=out[:, 5:])
    with np.errstate(over="ignore"):
        _same(out[:, 5:], wv.astype(np.float16).astype(np.float64))
    assert (out[:, :5] == 0).all()
    qt, st = B.quant_mxfp4(x, axis=0, q=torch.zeros(cols, 7, dtype=torch.uint8, device="cuda")[:, 1:6])
    assert np.array_equal(R.decode(qt, st, rows), R.quant(x.t())[2], equal_nan=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,cols,odd", [(130, 69, 1), (128, 64, 0), (128, 64, 4), (97, 129, 0), (300, 200, 2), (1, 8, 0), (257, 33, 16)])
def test_quant_both_from_aligned_rows(B, rows, cols, odd, dtype):
    """Source rows start 16-byte aligned, results wherever the caller has them."""
    x = torch.full((rows, (cols + 15) // 16 * 16), 1e4, device="cuda", dtype=dtype)[:, :cols]
    x.copy_(_values(rows, cols, dtype, rows))
    outs = []
    for r, c in ((rows, cols), (cols, rows)):
        for n in ((c + 1) // 2, (c + 31) // 32):
            outs.append(torch.full((r, n + 2 * odd), 7, dtype=torch.uint8, device="cuda")[:, odd:odd + n])
    B.quant_mxfp4_both(x, *outs)
    want = (*B.quant_mxfp4(x.contiguous()), *B.quant_mxfp4(x.T.contiguous()))
    for got, ref in zip(outs, want):
        assert torch.equal(got, ref)
        if odd:
            whole = got.as_strided((got.shape[0], got.shape[1] + 2 * odd), (got.stride(0), 1), got.storage_offset() - odd)
            assert (whole[:, :odd] == 7).all() and (whole[:, odd + got.shape[1]:] == 7).all()


def test_dequant_every_code_and_exponent(B):
    q = torch.arange(256, dtype=torch.uint8).repeat(256, 1)[:, :256].contiguous()
    s = torch.arange(256, dtype=torch.uint8)[:, None].repeat(1, 16)
    want = R.decode(q, s, 512)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        got = B.dequant_mxfp4(q.cuda(), s.cuda(), dtype)
        ref = torch.from_numpy(want).to(torch.float32).to(dtype).double().numpy()      # f32 holds every value or overflows
        _same(got, ref)


PRODUCTS = [(1, 1, 1), (1, 128, 256), (1, 300, 4096), (2, 64, 31), (5, 17, 33), (16, 129, 512), (17, 256, 768), (48, 100, 2900), (64, 640, 1024),
            (65, 128, 256), (100, 5, 2016), (128, 128, 8192), (129, 257, 640), (200, 1111, 3333), (333, 384, 14336), (700, 512, 512), (1100, 1300, 1536)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product_exact_with_one_exponent(B, m, n, k):
    a, sa = R.random_codes(m, k, seed=m + n, lo=127, hi=127)
    b, sb = R.random_codes(n, k, seed=k, lo=125, hi=125)
    ref = R.decode(a, sa, k) @ R.decode(b, sb, k).T
    got = B.matmul_mxfp4(a, sa, b, sb, out_dtype=torch.float32)
    assert np.array_equal(got.cpu().double().numpy(), ref)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product(B, m, n, k, dtype):
    a, sa = R.random_codes(m, k, seed=2 * m + n, lo=118, hi=128)
    b, sb = R.random_codes(n, k, seed=2 * k, lo=118, hi=128)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(1)).cuda()
    av, bv = R.decode(a, sa, k), R.decode(b, sb, k)
    tol = R.product_tolerance(av, bv, k, dtype)
    ref = av @ bv.T
    got = B.matmul_mxfp4(a, sa, b, sb, out_dtype=dtype).cpu().double().numpy()
    assert (np.abs(got - ref) <= tol(ref)).all()
    ref = ref + bias.cpu().double().numpy()
    got = B.matmul_mxfp4(a, sa, b, sb, bias=bias, out_dtype=dtype).cpu().double().numpy()
    assert (np.abs(got - ref) <= tol(ref) + 2.0 ** -23 * np.abs(ref)).all()


@pytest.mark.parametrize("m", [3, 100, 400])
def test_product_nan_rows_strides_and_bias_types(B, m):
    n, k = 200, 1000
    a, sa = R.random_codes(m, k, seed=5)
    b, sb = R.random_codes(n, k, seed=6)
    sa[m - 1, 30] = 255
    sb[7, 0] = 255
    sb[9] = 0                                                     # 2^-127: the products vanish next to the others
    out = torch.full((m + 1, n + 9), -7.0, device="cuda")
    bias = torch.randn(n, device="cuda").to(torch.bfloat16)
    B.matmul_mxfp4(a, sa, b, sb, bias=bias, out=out[:m, 3:3 + n])
    av, bv = R.decode(a, sa, k), R.decode(b, sb, k)
    ref = av @ bv.T + bias.cpu().double().numpy()
    got = out[:m, 3:3 + n].cpu().double().numpy()
    assert np.isnan(got[m - 1]).all() and np.isnan(got[:, 7]).all()
    ok = ~np.isnan(ref)
    tol = R.product_tolerance(np.nan_to_num(av), np.nan_to_num(bv), k, torch.float32)(np.nan_to_num(ref))
    assert np.array_equal(np.isnan(got), ~ok) and (np.abs(got - ref)[ok] <= (tol + 2.0 ** -23 * np.abs(ref))[ok]).all()
    assert (out[m] == -7).all() and (out[:, :3] == -7).all() and (out[:, 3 + n:] == -7).all()


GROUPS = [([3], 40, 256), ([0, 1, 0, 5, 16, 0], 130, 512), ([17, 0, 33], 128, 768), ([130, 1, 0, 257, 128], 300, 1024), ([0, 0, 0], 64, 256),
          ([2] * 70, 200, 544), ([300, 20, 500, 1], 516, 2048), ([1500, 0, 700], 1300, 640)]


@pytest.mark.parametrize("tail", [0, 5])
@pytest.mark.parametrize("sizes,n,k", GROUPS)
def test_grouped_product(B, sizes, n, k, tail):
    lead = 2 if tail else 0                                       # rows ahead of the first group belong to none either
    m, e = lead + sum(sizes) + tail, len(sizes)
    if m == 0:
        m = 1
    a, sa = R.random_codes(m, k, seed=m, lo=127, hi=127)
    a_nan = sa.clone()
    if tail:
        sa[m - 1] = 255                                           # a row of no group: must not reach any result
    b, sb = R.random_codes(e * n, k, seed=n, lo=126, hi=126)
    b3 = b.as_strided((e, n, b.shape[1]), (n * b.stride(0), b.stride(0), 1))
    sb3 = sb.as_strided((e, n, sb.shape[1]), (n * sb.stride(0), sb.stride(0), 1))
    offs = np.concatenate(([lead], lead + np.cumsum(sizes))).astype(np.int32)
    off = torch.from_numpy(offs).cuda()
    out = torch.full((m, n), 123.0, device="cuda")
    B.matmul_mxfp4(a, sa, b3, sb3, offsets=off, out=out)
    av, bv = R.decode(a, a_nan, k), R.decode(b, sb, k).reshape(e, n, k)
    ref = np.full((m, n), 123.0)
    for g in range(e):
        ref[offs[g]:offs[g + 1]] = av[offs[g]:offs[g + 1]] @ bv[g].T
    assert np.array_equal(out.cpu().double().numpy(), ref)
    bias = torch.randint(-8, 9, (e, n), generator=torch.Generator().manual_seed(2)).float().cuda()
    out.fill_(123.0)
    B.matmul_mxfp4(a, sa, b3, sb3, offsets=off, bias=bias, out=out)
    for g in range(e):
        ref[offs[g]:offs[g + 1]] += bias[g].cpu().double().numpy()
    assert np.array_equal(out.cpu().double().numpy(), ref)


def test_grouped_product_bad_offsets_stay_inside(B):
    m, n, k, e = 40, 64, 256, 4
    a, sa = R.random_codes(m, k, seed=1, lo=127, hi=127)
    b, sb = R.random_codes(e * n, k, seed=2, lo=127, hi=127)
    b3, sb3 = b.reshape(e, n, -1), sb.as_strided((e, n, sb.shape[1]), (n * sb.stride(0), sb.stride(0), 1))
    av, bv = R.decode(a, sa, k), R.decode(b, sb, k).reshape(e, n, k)
    guard = torch.full((m + 8, n), 5.0, device="cuda")
    off = torch.tensor([-9, 10, 4, 2000, 3], dtype=torch.int32, device="cuda")      # groups: 0..10, none, 10..40, none
    B.matmul_mxfp4(a, sa, b3, sb3, offsets=off, out=guard[:m])
    ref = np.concatenate((av[:10] @ bv[0].T, av[10:] @ bv[2].T))
    assert np.array_equal(guard[:m].cpu().double().numpy(), ref) and (guard[m:] == 5).all()


def test_linear_backward_and_gradient_by_differences(B):
    """dX = dY W and dW = dY^T X with operands quantised along what each product contracts, equal to the formula's; and the
    gradient of a scalar of the product's result equals differences of it (the product is linear in its decoded A)."""
    m, n, k = 96, 160, 224
    g = torch.Generator().manual_seed(0)
    dy, x, w = (torch.randn(s, generator=g).to(torch.bfloat16).cuda() for s in ((m, n), (m, k), (n, k)))
    q, s, qt, st = B.quant_mxfp4_both(dy)
    wq, ws = B.quant_mxfp4(w, axis=0)
    xq, xs = B.quant_mxfp4(x, axis=0)
    dx = B.matmul_mxfp4(q, s, wq, ws, out_dtype=torch.float32).cpu().double().numpy()
    dw = B.matmul_mxfp4(qt, st, xq, xs, out_dtype=torch.float32).cpu().double().numpy()
    dyr, dyc, wc, xc = R.quant(dy)[2], R.quant(dy.t())[2], R.quant(w.t())[2], R.quant(x.t())[2]
    for got, a, b, kk in ((dx, dyr, wc, n), (dw, dyc, xc, m)):
        ref = a @ b.T
        assert (np.abs(got - ref) <= R.product_tolerance(a, b, kk, torch.float32)(ref)).all()
    # f(A) = <C, G>, C = A B^T with one exponent everywhere: df/dA = G B, by differences of one code each
    a, sa = R.random_codes(4, 64, 1, 127, 127)
    b, sb = R.random_codes(32, 64, 2, 127, 127)
    gmat = torch.randint(-3, 4, (4, 32), generator=g).double()
    grad = gmat.numpy() @ R.decode(b, sb, 64)
    f = lambda: (B.matmul_mxfp4(a, sa, b, sb, out_dtype=torch.float32).cpu().double() * gmat).sum().item()
    for r, c in ((0, 0), (1, 31), (3, 62)):
        keep = int(a[r, c // 2])
        vals = []
        for code in (2, 10):                                       # +1 and -1
            a[r, c // 2] = (keep & 0xf0) | code if c % 2 == 0 else (keep & 0x0f) | (code << 4)
            vals.append(f())
        a[r, c // 2] = keep
        assert (vals[0] - vals[1]) / 2 == grad[r, c]


# few tiles and a long K: a cluster shares a tile's K, in tiles of 16, 32, 64 and 128 rows
SHARED_K = [(1, 1920, 8192), (9, 130, 9000), (16, 2048, 8192), (31, 2100, 2500), (33, 300, 8192), (64, 1000, 4100), (100, 1000, 8192),
            (120, 4096, 5000), (200, 3900, 14000), (256, 700, 8100)]


@pytest.mark.parametrize("m,n,k", SHARED_K)
def test_product_with_shared_k(B, m, n, k):
    """Sums of multiples of 1/4 under 2^20: f32 holds them in any order, so results are exact."""
    a, sa = R.random_codes(m, k, seed=m + n, lo=127, hi=127)
    b, sb = R.random_codes(n, k, seed=k, lo=127, hi=127)
    bias = torch.randint(-8, 9, (n,), generator=torch.Generator().manual_seed(2)).float().cuda()
    ref = R.decode(a, sa, k) @ R.decode(b, sb, k).T
    wide = torch.full((m + 1, n + 3), -7.0, device="cuda")       # rows that vector stores cannot take
    B.matmul_mxfp4(a, sa, b, sb, bias=bias, out=wide[:m, 1:n + 1])
    assert np.array_equal(wide[:m, 1:n + 1].cpu().double().numpy(), ref + bias.cpu().double().numpy())
    assert (wide[m] == -7).all() and (wide[:, 0] == -7).all() and (wide[:, n + 1:] == -7).all()
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        got = B.matmul_mxfp4(a, sa, b, sb, out_dtype=dtype)
        assert torch.equal(got.cpu(), torch.from_numpy(ref).float().to(dtype)), dtype
    assert B.device_error() == 0


@pytest.mark.parametrize("sizes,n,k", [([3, 0, 20], 260, 8192), ([40, 0, 33, 64], 200, 8192), ([130, 0, 100], 390, 6000), ([0, 90], 100, 4096),
                                       ([20, 1, 70], 250, 5000)])
def test_grouped_product_with_shared_k(B, sizes, n, k):
    m, e = sum(sizes) + 2, len(sizes)
    a, sa = R.random_codes(m, k, seed=m, lo=127, hi=127)
    b, sb = R.random_codes(e * n, k, seed=n, lo=127, hi=127)
    b3 = b.as_strided((e, n, b.shape[1]), (n * b.stride(0), b.stride(0), 1))
    sb3 = sb.as_strided((e, n, sb.shape[1]), (n * sb.stride(0), sb.stride(0), 1))
    offs = np.concatenate(([1], 1 + np.cumsum(sizes))).astype(np.int32)
    bias = torch.randint(-8, 9, (e, n), generator=torch.Generator().manual_seed(2)).float().cuda()
    out = torch.full((m, n), 123.0, device="cuda")
    B.matmul_mxfp4(a, sa, b3, sb3, offsets=torch.from_numpy(offs).cuda(), bias=bias, out=out)
    av, bv = R.decode(a, sa, k), R.decode(b, sb, k).reshape(e, n, k)
    ref = np.full((m, n), 123.0)
    for g in range(e):
        ref[offs[g]:offs[g + 1]] = av[offs[g]:offs[g + 1]] @ bv[g].T + bias[g].cpu().double().numpy()
    assert np.array_equal(out.cpu().double().numpy(), ref)


@pytest.mark.parametrize("m", [20, 60, 300])
def test_product_into_rows_far_apart(B, m):
    """Rows of C 2^26 elements apart: their offsets pass 2^31."""
    n, k, pitch = 128, 512, 1 << 26
    a, sa = R.random_codes(m, k, 1, 127, 127)
    b, sb = R.random_codes(n, k, 2, 127, 127)
    out = torch.empty(m * pitch, dtype=torch.bfloat16, device="cuda").as_strided((m, n), (pitch, 1))
    B.matmul_mxfp4(a, sa, b, sb, out=out)
    assert torch.equal(out.contiguous(), B.matmul_mxfp4(a, sa, b, sb))
    want = torch.from_numpy(R.decode(a, sa, k) @ R.decode(b, sb, k).T).float().to(torch.bfloat16)
    assert torch.equal(out.cpu(), want)


def test_capture_streams_and_repeats(B):
    """Captured into a graph and replayed on new contents; on a side stream; the same bits every time."""
    m, n, k, e = 24, 256, 1024, 3
    a, sa = R.random_codes(m, k, 1, 120, 130)
    b, sb = R.random_codes(e * n, k, 2, 120, 130)
    b3, sb3 = b.reshape(e, n, -1), sb.as_strided((e, n, sb.shape[1]), (n * sb.stride(0), sb.stride(0), 1))
    off = torch.tensor([0, 5, 5, 24], dtype=torch.int32, device="cuda")
    x = torch.randn(m, k, device="cuda").to(torch.bfloat16)
    out = torch.zeros(m, n, device="cuda", dtype=torch.bfloat16)

    def step():
        q, s = B.quant_mxfp4(x, q=a, scale=sa)
        B.matmul_mxfp4(q, s, b3, sb3, offsets=off, out=out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    first = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)
    x.copy_(torch.randn(m, k, device="cuda"))
    off.copy_(torch.tensor([0, 0, 20, 22], dtype=torch.int32))
    out.zero_()
    graph.replay()
    replay = out.clone()
    out.zero_()
    step()
    assert torch.equal(out, replay) and (out[22:] == 0).all() and out[:22].abs().sum() > 0


def test_two_threads_on_two_streams(B):
    """Clusters that share K, from two threads at once: the same bits as alone."""
    a, sa = R.random_codes(64, 8192, 1)
    b, sb = R.random_codes(1000, 8192, 2)
    alone = B.matmul_mxfp4(a, sa, b, sb, out_dtype=torch.float32)
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got[i].append(B.matmul_mxfp4(a, sa, b, sb, out_dtype=torch.float32))
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(y, alone) for ys in got for y in ys) and len(got[0]) == len(got[1]) == 20
    assert B.device_error() == 0


def test_python_refusals(B):
    x = torch.zeros(4, 64, device="cuda")
    with pytest.raises(B.BsirError):
        B.quant_mxfp4(torch.zeros(4, 64))                            # not on the device
    with pytest.raises(B.BsirError):
        B.quant_mxfp4(x, axis=2)
    with pytest.raises(B.BsirError):
        B.quant_mxfp4(x.t())                                         # columns contiguous
    with pytest.raises(B.BsirError):
        B.quant_mxfp4(x.to(torch.int8))
    q, s = B.quant_mxfp4(x)
    with pytest.raises(B.BsirError):
        B.dequant_mxfp4(q, s, cols=63 + 3)
    with pytest.raises(B.BsirError):
        B.matmul_mxfp4(q, s, q, s[:, :1])
    with pytest.raises(B.BsirError):
        B.matmul_mxfp4(q, s, q.contiguous(), s.contiguous())          # exponents 2 bytes apart: rows not 16-byte aligned
    with pytest.raises(B.BsirError):
        B.matmul_mxfp4(q, s, q, s, out=torch.zeros(4, 5, device="cuda"))
    with pytest.raises(B.BsirError):
        B.matmul_mxfp4(q, s, q[None], s[None], offsets=torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(B.BsirError):
        B.matmul_mxfp4(q, s, q, s, bias=torch.zeros(3, device="cuda"))
    assert tuple(B.matmul_mxfp4(q[:0], s[:0], q, s).shape) == (0, 4)
