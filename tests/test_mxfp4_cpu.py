"""CPU: the host-side checks of the microscaled 4-bit and expert-routing entry points refuse what the kernels could not
address, before anything is enqueued, and the reference the GPU tests use obeys the format's definition."""
import ctypes as C

import numpy as np
import pytest
import torch

import mxfp4_reference as R

P = C.c_void_p
I = C.c_int64
A0, A1, A2, A3, A4 = (0x10000000 * i for i in range(1, 6))      # addresses that are never touched


@pytest.fixture(scope="module")
def L():
    import bsir
    return bsir.lib()


def test_reference_rounds_to_nearest_with_ties_to_the_even_code():
    x = torch.zeros(1, 32)
    v = [6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -5.0, 7.9, -0.26, 0.2499]
    x[0, :len(v)] = torch.tensor(v)
    _, byte, got = R.quant(x)
    assert byte[0, 0] == 127
    assert got[0, :len(v)].tolist() == [6, 0, 1, 1, 2, 2, 4, 4, 0, -4, 6, -0.5, 0]


def test_reference_exponent_and_nan_blocks():
    x = torch.zeros(4, 64)
    x[0, :32] = 2.0 ** -140
    x[1, 3] = float("inf")
    x[2, 40] = float("nan")
    x[3, :32] = 3e38
    _, byte, got = R.quant(x)
    assert byte[:, 0].tolist() == [0, 255, 0, 252] and byte[2, 1] == 255
    assert np.isnan(got[1, :32]).all() and np.isnan(got[2, 32:]).all() and (got[2, :32] == 0).all()
    assert (got[0] == 0).all()                                   # 2^-140 * 2^127 rounds to zero


def _quant(L, dtype=2, rows=4, cols=64, x=A0, xs=64, q=A1, qs=32, s=A2, ss=2, qt=None, qts=0, st=None, sts=0):
    return L.bsir_quant_mxfp4(dtype, I(rows), I(cols), P(x), I(xs), P(q), I(qs), P(s), I(ss), P(qt), I(qts), P(st), I(sts), None)


def test_quant_refusals(L):
    assert _quant(L, dtype=3) == -4
    assert _quant(L, rows=-1) == -2 and _quant(L, cols=(1 << 31) + 1) == -2
    assert _quant(L, rows=0) == 0 and _quant(L, cols=0) == 0
    assert _quant(L, s=None) == -1 and _quant(L, q=None) == -1 and _quant(L, q=None, s=None) == -1 and _quant(L, x=None) == -1
    assert _quant(L, qt=A3, qts=2) == -1
    assert _quant(L, xs=63) == -3 and _quant(L, qs=31) == -3 and _quant(L, ss=1) == -3
    assert _quant(L, qt=A3, qts=1, st=A4, sts=1) == -3
    assert _quant(L, x=A0 + 1) == -6
    assert _quant(L, q=A0 + 16) == -11 and _quant(L, s=A0 + 3 * 128 + 127) == -11
    assert b"overlap" in L.bsir_last_error()


def _dequant(L, dtype=0, rows=4, cols=64, q=A0, qs=32, s=A1, ss=2, y=A2, ys=64):
    return L.bsir_dequant_mxfp4(dtype, I(rows), I(cols), P(q), I(qs), P(s), I(ss), P(y), I(ys), None)


def test_dequant_refusals(L):
    assert _dequant(L, dtype=7) == -4 and _dequant(L, cols=-1) == -2 and _dequant(L, rows=0) == 0
    assert _dequant(L, y=None) == -1 and _dequant(L, q=None) == -1
    assert _dequant(L, qs=31) == -3 and _dequant(L, ss=1) == -3 and _dequant(L, ys=63) == -3
    assert _dequant(L, y=A2 + 2) == -6 and _dequant(L, y=A1 - 128) == -11


def _product(L, **kw):
    import bsir
    d = bsir.MatmulMxfp4Desc()
    base = dict(out_dtype=2, bias_dtype=0, m=8, n=64, k=512, a=A0, lda=256, scale_a=A1, ldsa=16, b=A2, ldb=256, scale_b=A3, ldsb=16,
                batch_stride_b=64 * 256, batch_stride_sb=64 * 16, out=A4, ldo=64)
    base.update(kw)
    for name, v in base.items():
        setattr(d, name, v)
    return L.bsir_matmul_mxfp4(C.byref(d), None)


def test_product_refusals(L):
    assert L.bsir_matmul_mxfp4(None, None) == -1
    assert _product(L, out_dtype=3) == -4 and _product(L, bias=A4 + 0x1000000, bias_dtype=5) == -4
    assert _product(L, k=0) == -2 and _product(L, m=-1) == -2 and _product(L, n=(1 << 30) + 1) == -2
    assert _product(L, groups=2) == -2                                            # several groups want offsets
    assert _product(L, offsets=A4 + 0x1000000, groups=0) == -2 and _product(L, offsets=A4 + 0x1000000, groups=1025) == -2
    assert _product(L, m=0) == 0 and _product(L, n=0) == 0
    for name in ("a", "scale_a", "b", "scale_b", "out"):
        assert _product(L, **{name: None}) == -1
    assert _product(L, lda=240) == -3 and _product(L, lda=257) == -3 and _product(L, ldsa=8) == -3 and _product(L, ldsb=17) == -3
    off = dict(offsets=A4 + 0x1000000, groups=2)
    assert _product(L, batch_stride_b=64 * 256 - 16, **off) == -3 and _product(L, batch_stride_sb=1000, **off) == -3
    assert _product(L, a=A0 + 8) == -6 and _product(L, scale_b=A3 + 4) == -6 and _product(L, out=A4 + 1) == -6
    assert _product(L, ldo=63) == -3
    assert _product(L, bias=A4 + 0x1000000, bias_stride=-64, **off) == -3
    assert _product(L, out=A0 + 16) == -11 and _product(L, offsets=A4 + 64, groups=1) == -11


def _sort(L, dt=5, tokens=4, top_k=2, experts=8, ids=A0, offsets=A1, slots=A2):
    return L.bsir_expert_sort(dt, I(tokens), I(top_k), I(experts), P(ids), P(offsets), P(slots), None)


def test_expert_refusals(L):
    assert _sort(L, dt=4) == -4 and _sort(L, experts=0) == -2 and _sort(L, experts=1025) == -2 and _sort(L, tokens=-1) == -2
    assert _sort(L, tokens=1 << 30, top_k=4) == -2
    assert _sort(L, ids=None) == -1 and _sort(L, offsets=None) == -1 and _sort(L, slots=None) == -1
    assert _sort(L, ids=A0 + 2) == -6 and _sort(L, dt=6, ids=A0 + 4) == -6
    assert _sort(L, slots=A0 + 16) == -11

    def dispatch(dt=2, tokens=4, top_k=2, cols=8, x=A0, xs=8, slots=A1, rows=8, out=A2, os=8):
        return L.bsir_expert_dispatch(dt, I(tokens), I(top_k), I(cols), P(x), I(xs), P(slots), I(rows), P(out), I(os), None)
    assert dispatch(dt=99) == -4 and dispatch(cols=-1) == -2 and dispatch(tokens=0) == 0 and dispatch(top_k=0) == 0
    assert dispatch(x=None) == -1 and dispatch(slots=None) == -1 and dispatch(out=None) == -1
    assert dispatch(xs=7) == -3 and dispatch(os=7) == -3 and dispatch(x=A0 + 1) == -6 and dispatch(slots=A1 + 2) == -6
    assert dispatch(out=A0 + 16) == -11 and dispatch(out=A1) == -11

    def combine(dt=2, tokens=4, top_k=2, cols=8, rows=8, y=A0, ys=8, slots=A1, wdt=0, w=A2, out=A3, os=8):
        return L.bsir_expert_combine(dt, I(tokens), I(top_k), I(cols), I(rows), P(y), I(ys), P(slots), wdt, P(w), P(out), I(os), None)
    assert combine(dt=5) == -4 and combine(wdt=3) == -4 and combine(rows=-1) == -2 and combine(tokens=0) == 0 and combine(cols=0) == 0
    assert combine(y=None) == -1 and combine(slots=None) == -1 and combine(out=None) == -1
    assert combine(ys=7) == -3 and combine(os=7) == -3 and combine(w=A2 + 2) == -6 and combine(out=A0 + 16) == -11 and combine(out=A2) == -11

    def grad(dt=2, tokens=4, top_k=2, cols=8, rows=8, g=A0, gs=8, y=A1, ys=8, slots=A2, wdt=0, w=A3, dy=A4, dys=8, dw=A4 + 0x1000000):
        return L.bsir_expert_combine_grad(dt, I(tokens), I(top_k), I(cols), I(rows), P(g), I(gs), P(y), I(ys), P(slots), wdt, P(w), P(dy),
                                          I(dys), P(dw), None)
    assert grad(dt=3) == -4 and grad(wdt=6) == -4 and grad(cols=-1) == -2 and grad(tokens=0) == 0
    assert grad(g=None) == -1 and grad(y=None) == -1 and grad(slots=None) == -1 and grad(dy=None) == -1 and grad(dw=None) == -1
    assert grad(gs=7) == -3 and grad(ys=7) == -3 and grad(dys=7) == -3 and grad(dw=A4 + 2) == -6
    assert grad(dy=A1) == -11 and grad(dw=A2) == -11 and grad(dw=A4 + 16) == -11


# Results side by side in rows of one buffer are told from results that share bytes.
@pytest.mark.parametrize("kw", [
    dict(s=A1 + 31),                                             # the last byte of the first row of codes
    dict(s=A1 - 1, ss=2),                                        # the second exponent of the first row
    dict(qs=64, s=A1 + 63, ss=64),                               # wraps into the next row of codes
    dict(qs=48, s=A1 + 40, ss=40),                               # other pitches: row 2's exponents lie in row 2's codes
    dict(qt=A1 + 96, qts=2, st=A4, sts=1),                       # one direction with the other
    dict(qt=A3, qts=2, st=A2 + 7, sts=1),
    dict(qt=A3, qts=2, st=A3 + 127, sts=1),
    dict(q=None, s=None, qt=A3, qts=2, st=A3 + 1, sts=2),
    dict(rows=1, s=A1 + 31), dict(cols=1, qt=A3, qts=2, st=A3 + 1, sts=1),
])
def test_quant_results_that_share_bytes_are_refused(L, kw):
    assert _quant(L, **kw) == -11
    assert b"each other" in L.bsir_last_error()


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are made up, and the call gets as far as the launch")
@pytest.mark.parametrize("kw", [
    dict(s=A1 + 128), dict(s=A1 - 8),                            # behind and ahead
    dict(qs=48, s=A1 + 32, ss=48), dict(qs=48, s=A1 - 2, ss=48), # between the rows of codes
    dict(qs=34, s=A1 + 32, ss=34), dict(qs=64, s=A1 + 33, ss=128),
    dict(qs=64, ss=64, s=A1 + 32, qt=A3, qts=3, st=A3 + 2, sts=3),
    dict(rows=1, s=A1 + 32), dict(rows=1, qs=1, s=A1 + 32, ss=1),
])
def test_quant_results_side_by_side_are_not(L, kw):
    _quant(L, **kw)
    assert b"overlap" not in L.bsir_last_error()


@pytest.mark.parametrize("m,n,k,groups,form", [
    (1, 4096, 4096, 1, (16, 128)), (17, 4096, 512, 1, (32, 128)), (40, 40000, 512, 1, (128, 128)), (40, 40000, 2100, 1, (64, 128)), (400, 1000, 512, 1, (128, 128)),
    (1500, 3001, 2100, 1, (256, 256)), (2100, 5001, 2100, 1, (256, 256)), (4096, 4096, 4096, 1, (256, 256)),
    (3800, 2500, 1100, 4, (256, 256)), (2500, 4100, 2100, 4, (256, 256)),
    (600, 1200, 544, 60, (16, 128)), (900, 1300, 544, 48, (32, 128)), (1600, 1300, 544, 48, (64, 128)),
])
def test_product_form(L, m, n, k, groups, form):
    """The rows and columns of a tile go by the sizes alone (the CTAs that share one by the device too)."""
    import bsir
    assert bsir.matmul_mxfp4_form(m, n, k, groups)[:2] == form


def test_product_form_refusals(L):
    import bsir
    for bad in ((0, 1, 1, 1), (1, 0, 1, 1), (1, 1, 0, 1), ((1 << 30) + 1, 1, 1, 1), (1 << 30, 1 << 30, 1, 1), (1, 1, 1, 0), (1, 1, 1, 1025)):
        with pytest.raises(bsir.BsirError):
            bsir.matmul_mxfp4_form(*bad)
    assert L.bsir_matmul_mxfp4_form(I(1), I(1), I(1), I(1), None, None, None) == -1
