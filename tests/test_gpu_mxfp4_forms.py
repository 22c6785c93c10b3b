"""GPU: every form of the 4-bit product and of the quantiser at sizes where its loops come round: CTA pairs over several
rounds of tiles, streamed weights over hundreds of tiles of several groups, columns quantised over thousands of tiles.
Products of one exponent are exact in f32 (multiples of 1/4 under 2^22), so that any order of adding gives the same bits;
the reference is a 64-bit product of the decoded operands."""
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


def _decoded(q, s, cols):
    return torch.from_numpy(R.decode(q, s, cols)).cuda()


def _guarded(m, n, dtype, odd):
    """An [m, n] view with a row behind it and columns around it that have to stay, 16-byte aligned rows unless `odd`."""
    lead, pitch = (1, n + 3 + n % 2) if odd else (16, (n + 47) // 16 * 16)
    whole = torch.full((m + 1, pitch), -7.0, dtype=dtype, device="cuda")
    return whole, whole[:m, lead:lead + n], lead


def _guards_stay(whole, m, lead, n):
    return bool((whole[m] == -7).all() and (whole[:, :lead] == -7).all() and (whole[:, lead + n:] == -7).all())


# the last: one row and one column in the last tiles, six stages
PAIRS = [(1500, 3001, 2100), (2100, 5001, 2100), (2305, 4865, 1540)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", PAIRS)
def test_pairs(B, m, n, k, dtype):
    assert B.matmul_mxfp4_form(m, n, k) == (256, 256, 2)
    a, sa = R.random_codes(m, k, seed=m, lo=127, hi=127)
    b, sb = R.random_codes(n, k, seed=n, lo=126, hi=126)
    bias = torch.randint(-8, 9, (n,), generator=torch.Generator().manual_seed(2)).float().cuda()
    ref = _decoded(a, sa, k) @ _decoded(b, sb, k).T
    for odd in (False, True):
        for add in (None, bias):
            want = (ref if add is None else ref + add.double()).float().to(dtype)
            for _ in range(2):
                whole, out, lead = _guarded(m, n, dtype, odd)
                B.matmul_mxfp4(a, sa, b, sb, bias=add, out=out)
                assert torch.equal(out, want) and _guards_stay(whole, m, lead, n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_pairs_with_exponents(B, dtype):
    """Every row's and block's own exponent reaches its products."""
    m, n, k = 1500, 3001, 2100
    a, sa = R.random_codes(m, k, seed=1, lo=118, hi=128)
    b, sb = R.random_codes(n, k, seed=2, lo=118, hi=128)
    av, bv = _decoded(a, sa, k), _decoded(b, sb, k)
    ref = av @ bv.T
    got = B.matmul_mxfp4(a, sa, b, sb, out_dtype=dtype).double()
    # additions each off by a step of at most the magnitudes' sum, then half a step of C
    tol = (k + 1) * 2.0 ** -23 * (av.abs() @ bv.abs().T) + torch.finfo(dtype).eps / 2 * ref.abs()
    assert ((got - ref).abs() <= tol).all()


def _groups(B, sizes, n, k, dtype, odd, with_bias, lead=0, tail=0):
    """The grouped product against a 64-bit one a group; rows of no group hold NaN exponents and must not be written."""
    m, e = lead + sum(sizes) + tail, len(sizes)
    a, sa = R.random_codes(m, k, seed=m, lo=127, hi=127)
    av = _decoded(a, sa, k)
    sa[:lead] = 255
    sa[m - tail:] = 255
    b, sb = R.random_codes(e * n, k, seed=n, lo=126, hi=126)
    cut = lambda t: t.as_strided((e, n, t.shape[1]), (n * t.stride(0), t.stride(0), 1))
    bv = _decoded(b, sb, k).view(e, n, k)
    offs = np.concatenate(([lead], lead + np.cumsum(sizes))).astype(np.int32)
    bias = torch.randint(-8, 9, (e, n), generator=torch.Generator().manual_seed(2)).float().cuda() if with_bias else None
    want = torch.full((m, n), -7.0, dtype=dtype, device="cuda")
    for g in range(e):
        lo, hi = int(offs[g]), int(offs[g + 1])
        v = av[lo:hi] @ bv[g].T
        want[lo:hi] = (v if bias is None else v + bias[g].double()).float().to(dtype)
    off = torch.from_numpy(offs).cuda()
    for _ in range(2):
        whole, out, first = _guarded(m, n, dtype, odd)
        B.matmul_mxfp4(a, sa, cut(b), cut(sb), bias=bias, offsets=off, out=out)
        assert torch.equal(out, want) and _guards_stay(whole, m, first, n)


@pytest.mark.parametrize("dtype,odd,with_bias", [(torch.float32, False, True), (torch.float32, True, False), (torch.bfloat16, False, False),
                                                 (torch.bfloat16, True, True), (torch.float16, True, False), (torch.float16, False, True)])
@pytest.mark.parametrize("sizes,n,k", [([2100, 0, 1000, 700], 2500, 1100), ([1500, 0, 700, 300], 4100, 2100), ([900, 129, 1, 257, 2000], 2049, 2100)])
def test_pairs_of_groups(B, sizes, n, k, dtype, odd, with_bias):
    assert B.matmul_mxfp4_form(3 + sum(sizes) + 5, n, k, len(sizes)) == (256, 256, 2)
    _groups(B, sizes, n, k, dtype, odd, with_bias, lead=3, tail=5)


# groups of about `mean` rows, some of none: hundreds of tiles on each form that streams the weights
STREAMED = [(16, 60, 10, 1200, 544), (32, 48, 18, 1300, 544), (64, 48, 33, 1300, 544), (128, 40, 90, 1700, 300)]


@pytest.mark.parametrize("dtype,odd,with_bias", [(torch.float32, True, True), (torch.bfloat16, False, True), (torch.float16, True, False)])
@pytest.mark.parametrize("rows,groups,mean,n,k", STREAMED)
def test_many_groups_of_few_rows(B, rows, groups, mean, n, k, dtype, odd, with_bias):
    g = torch.Generator().manual_seed(rows)
    sizes = torch.randint(0, 2 * mean + 1, (groups,), generator=g).tolist()
    sizes[0] = sizes[7] = sizes[groups - 1] = 0
    m = 2 + sum(sizes) + 1
    form = B.matmul_mxfp4_form(m, n, k, groups)
    assert form == (rows, 128, 1)
    tiles = sum(-(-s // rows) for s in sizes) * -(-n // 128)
    assert tiles > 2 * 148
    _groups(B, sizes, n, k, dtype, odd, with_bias, lead=2, tail=1)


@pytest.mark.parametrize("m,k,rows", [(9, 700, 16), (30, 700, 32), (40, 2100, 64), (120, 300, 128)])
def test_many_columns(B, m, k, rows):
    """One group, more than two rounds of tiles."""
    n = 40001
    assert B.matmul_mxfp4_form(m, n, k) == (rows, 128, 1)
    a, sa = R.random_codes(m, k, seed=m, lo=127, hi=127)
    b, sb = R.random_codes(n, k, seed=n, lo=126, hi=126)
    ref = _decoded(a, sa, k) @ _decoded(b, sb, k).T
    for dtype, odd in ((torch.float32, False), (torch.bfloat16, True)):
        whole, out, lead = _guarded(m, n, dtype, odd)
        B.matmul_mxfp4(a, sa, b, sb, out=out)
        assert torch.equal(out, ref.float().to(dtype)) and _guards_stay(whole, m, lead, n)


def _spread(rows, cols, dtype, seed):
    """Values over many exponents, made on the device, with a NaN, an infinity and a row of zeros."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, device="cuda") * torch.exp2(torch.randint(-6, 7, (rows, 1), generator=g, device="cuda").float())
    x[rows // 3, cols // 5] = float("nan")
    x[rows - 1, cols - 1] = -float("inf")
    x[rows // 2] = 0.0
    return x.to(dtype)


# tiles of 128 x 64, two to five CTAs an SM take them: 2607 and 1080 of them, ragged both ways, from 16-byte aligned rows
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(4100, 5000), (15300, 569)])
def test_columns_over_many_tiles(B, rows, cols, dtype):
    """Against the blocks along the rows of the transposed matrix, which have a kernel of their own."""
    x = torch.zeros(rows, (cols + 7) // 8 * 8, dtype=dtype, device="cuda")[:, :cols]
    x.copy_(_spread(rows, cols, dtype, rows))
    want_t = B.quant_mxfp4(x.t().contiguous())
    want = B.quant_mxfp4(x.contiguous())
    for _ in range(2):
        got = B.quant_mxfp4(x, axis=0)
        assert all(torch.equal(a, b) for a, b in zip(got, want_t))
        got = B.quant_mxfp4_both(x)
        assert all(torch.equal(a, b) for a, b in zip(got, (*want, *want_t)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_columns_of_more_rows_than_a_grid_has(B, dtype):
    """8.4e6 rows of any alignment: strips of 65535 x 128 rows."""
    rows, cols = 65535 * 128 + 300, 3
    x = _spread(rows, cols, dtype, 5)
    x[65535 * 128 + 40, 1] = 1000.0
    got = B.quant_mxfp4_both(x)
    want = (*B.quant_mxfp4(x), *B.quant_mxfp4(x.t().contiguous()))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_columns_beyond_32_bits(B):
    """2.2e9 elements: element numbers pass 2^31."""
    rows, cols = 66000, 33000
    x = torch.randn(rows, cols, device="cuda", generator=torch.Generator(device="cuda").manual_seed(0), dtype=torch.bfloat16)
    got = B.quant_mxfp4_both(x)
    want = (*B.quant_mxfp4(x), *B.quant_mxfp4(x.t().contiguous()))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
