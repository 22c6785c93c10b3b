"""GPU: tokens sorted by expert and back, with weights and gradients, against plain loops in 64 bits; and a whole
mixture-of-experts layer made of the library's calls."""
import os
import subprocess
import sys

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


def _ids(tokens, top_k, experts, seed, masked=0.2, skew=False):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, experts, (tokens, top_k), generator=g)
    if skew:
        ids = torch.minimum(ids, torch.randint(0, experts, (tokens, top_k), generator=g) // 3)
    drop = torch.rand(tokens, top_k, generator=g)
    ids[drop < masked / 2] = -1
    ids[drop > 1 - masked / 2] = experts + 3                           # another rank's
    return ids


SORTS = [(1, 1, 1), (1, 8, 256), (7, 3, 5), (32, 4, 64), (512, 8, 8), (513, 8, 60), (1000, 5, 1024), (4096, 1, 2), (9001, 6, 128), (9000, 7, 127), (70000, 8, 33)]


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("tokens,top_k,experts", SORTS)
def test_sort(B, tokens, top_k, experts, wide):
    ids = _ids(tokens, top_k, experts, tokens, skew=tokens > 1000)
    wo, wsl = R.sort(ids.tolist(), experts)
    off, slots = B.expert_sort(ids.cuda() if wide else ids.int().cuda(), experts)
    assert np.array_equal(off.cpu().numpy(), wo) and np.array_equal(slots.cpu().numpy(), wsl)


@pytest.mark.parametrize("tokens,top_k,experts", [(2048, 8, 60), (2049, 8, 61), (16000, 8, 1024), (16385, 8, 128), (30001, 9, 500)])
def test_sort_of_many_choices(B, tokens, top_k, experts):
    """At the borders between the sizes of the cluster, and of what its warps keep in registers."""
    ids = _ids(tokens, top_k, experts, tokens, skew=True)
    wo, wsl = R.sort(ids.tolist(), experts)
    for _ in range(2):
        off, slots = B.expert_sort(ids.int().cuda(), experts)
        assert np.array_equal(off.cpu().numpy(), wo) and np.array_equal(slots.cpu().numpy(), wsl)


def test_sort_extremes(B):
    off, slots = B.expert_sort(torch.full((5000, 2), -1, dtype=torch.int64, device="cuda"), 4)
    assert (off == 0).all() and (slots == -1).all()
    off, slots = B.expert_sort(torch.full((5000, 2), 3, dtype=torch.int32, device="cuda"), 4)
    assert off.tolist() == [0, 0, 0, 0, 10000] and torch.equal(slots.flatten().cpu(), torch.arange(10000, dtype=torch.int32))
    off, slots = B.expert_sort(torch.zeros((0, 2), dtype=torch.int32, device="cuda"), 3)
    assert off.tolist() == [0, 0, 0, 0]
    big = torch.tensor([[1 << 40, -(1 << 40), 1]], dtype=torch.int64, device="cuda")      # must not wrap into an expert
    assert B.expert_sort(big, 2)[1].tolist() == [[-1, -1, 0]]


CASES = [(1, 1, 1, 1), (1, 2, 4, 8), (3, 2, 4, 33), (40, 4, 8, 4096), (17, 8, 16, 1000), (65, 6, 7, 514), (300, 9, 40, 72), (5, 16, 64, 12288), (4, 70, 100, 200)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16, torch.uint8, torch.int64])
@pytest.mark.parametrize("tokens,top_k,experts,cols", CASES)
def test_dispatch(B, tokens, top_k, experts, cols, dtype):
    _, slots = R.sort(_ids(tokens, top_k, experts, cols).tolist(), experts)
    x = torch.randint(0, 200, (tokens, cols), generator=torch.Generator().manual_seed(1)).to(dtype)
    rows = tokens * top_k
    out = torch.full((rows + 1, cols), 77, dtype=dtype, device="cuda")
    B.expert_dispatch(x.cuda(), torch.from_numpy(slots).cuda(), out=out)
    want = torch.full((rows + 1, cols), 77, dtype=dtype)
    for t in range(tokens):
        for j in range(top_k):
            if slots[t, j] >= 0:
                want[slots[t, j]] = x[t]
    assert torch.equal(out.cpu(), want)


def _layer(tokens, top_k, experts, cols, dtype, wdtype, seed):
    g = torch.Generator().manual_seed(seed)
    _, slots = R.sort(_ids(tokens, top_k, experts, seed).tolist(), experts)
    rows = tokens * top_k
    y = torch.randn(rows, cols, generator=g).to(dtype)
    used = set(slots[slots >= 0].tolist())
    for r in range(rows):
        if r not in used:
            y[r] = float("nan")                                        # nobody's rows are not read
    w = torch.randn(tokens, top_k, generator=g).to(wdtype)
    w[torch.from_numpy(slots) < 0] = float("nan")                     # nor masked choices' weights
    dout = torch.randn(tokens, cols, generator=g).to(dtype)
    return slots, y, w, dout


@pytest.mark.parametrize("wdtype", [torch.float32, torch.bfloat16, torch.float16, None])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens,top_k,experts,cols", CASES)
def test_combine_and_gradient(B, tokens, top_k, experts, cols, dtype, wdtype):
    slots, y, w, dout = _layer(tokens, top_k, experts, cols, dtype, wdtype or torch.float32, cols + top_k)
    rows = y.shape[0]
    yd, gd = y.double().numpy(), dout.double().numpy()
    wd = w.double().numpy() if wdtype else np.ones((tokens, top_k))
    out, mag = np.zeros((tokens, cols)), np.zeros((tokens, cols))
    dy, dw, dmag = np.full((rows, cols), 9.0), np.zeros((tokens, top_k)), np.zeros((tokens, top_k))
    for t in range(tokens):
        for j in range(top_k):
            s = slots[t, j]
            if s < 0:
                continue
            out[t] += wd[t, j] * yd[s]
            mag[t] += np.abs(wd[t, j] * yd[s])
            dy[s] = wd[t, j] * gd[t]
            dw[t, j] = (gd[t] * yd[s]).sum()
            dmag[t, j] = np.abs(gd[t] * yd[s]).sum()
    half = torch.finfo(dtype).eps / 2
    tiny = float(torch.finfo(dtype).smallest_normal)
    sl = torch.from_numpy(slots).cuda()
    wc = w.cuda() if wdtype else None
    got = B.expert_combine(y.cuda(), sl, wc).cpu().double().numpy()
    # one f32 rounding a term (2^-24 of a partial sum, at most the magnitudes' sum), then C's
    assert (np.abs(got - out) <= top_k * 2.0 ** -24 * mag * 1.01 + half * np.abs(out) * 1.001 + tiny * half).all()
    dy0 = torch.full((rows, cols), 9.0, dtype=dtype, device="cuda")
    gy, gw = B.expert_combine_grad(dout.cuda(), y.cuda(), sl, wc, out=dy0)
    # the f32 product's rounding, then dy's
    assert (np.abs(gy.cpu().double().numpy() - dy) <= (half + 2.0 ** -24) * 1.001 * np.abs(dy) + tiny * half).all()
    # a dot product of `cols` terms, each addition off by 2^-24 of at most the magnitudes' sum
    assert (np.abs(gw.cpu().double().numpy() - dw) <= cols * 2.0 ** -24 * 1.01 * dmag).all()
    assert (gw.cpu()[torch.from_numpy(slots) < 0] == 0).all()


def test_dispatch_gradient_is_combine_without_weights(B):
    """<dispatch(x), g> = <x, combine(g)> for integer data, hence by linearity its gradient; with differences of the former."""
    tokens, top_k, experts, cols = 20, 3, 5, 64
    _, slots = B.expert_sort(_ids(tokens, top_k, experts, 4).cuda(), experts)
    g = torch.Generator().manual_seed(0)
    x = torch.randint(-4, 5, (tokens, cols), generator=g).float().cuda()
    gr = torch.randint(-4, 5, (tokens * top_k, cols), generator=g).float().cuda()
    dx = B.expert_combine(gr, slots)
    f = lambda v: (B.expert_dispatch(v, slots) * gr).sum().item()
    assert f(x) == (x * dx).sum().item()
    for t, c in ((0, 0), (7, 63), (19, 5)):
        x1 = x.clone()
        x1[t, c] += 1
        assert f(x1) - f(x) == dx[t, c].item()


def test_strided_and_unaligned_rows(B):
    tokens, top_k, cols = 12, 2, 40
    _, slots = B.expert_sort(_ids(tokens, top_k, 4, 9).cuda(), 4)
    base = torch.randn(tokens, cols + 7, device="cuda").to(torch.bfloat16)
    x = base[:, 3:3 + cols]
    out = torch.zeros(tokens * top_k, cols + 5, dtype=torch.bfloat16, device="cuda")
    B.expert_dispatch(x, slots, out=out[:, 1:1 + cols])
    want = B.expert_dispatch(x.contiguous(), slots)
    assert torch.equal(out[:, 1:1 + cols], want) and (out[:, 0] == 0).all() and (out[:, 1 + cols:] == 0).all()
    w = torch.rand(tokens, top_k, device="cuda")
    comb = torch.zeros(tokens, cols + 3, dtype=torch.bfloat16, device="cuda")
    B.expert_combine(out[:, 1:1 + cols], slots, w, out=comb[:, 2:2 + cols])
    assert torch.equal(comb[:, 2:2 + cols], B.expert_combine(want, slots, w)) and (comb[:, :2] == 0).all()
    dy, dw = B.expert_combine_grad(x, out[:, 1:1 + cols], slots, w, out=torch.zeros_like(out)[:, 1:1 + cols])
    dy2, dw2 = B.expert_combine_grad(x.contiguous(), want, slots, w)
    assert torch.equal(dy, dy2)
    assert (dw - dw2).abs().max() <= 2 * cols * 2.0 ** -24 * (x.float().abs().amax() * want.float().abs().amax() * cols)


def test_rows_far_apart(B):
    """Rows 2^27 elements apart: offsets pass 2^31."""
    tokens, top_k, cols, pitch = 12, 2, 64, 1 << 27
    _, slots = B.expert_sort(_ids(tokens, top_k, 4, 9).cuda(), 4)
    x = torch.randn(tokens, cols, device="cuda").to(torch.bfloat16)
    w = torch.rand(tokens, top_k, device="cuda")
    far = torch.empty(24 * pitch, dtype=torch.bfloat16, device="cuda").as_strided((24, cols), (pitch, 1))
    far.zero_()
    B.expert_dispatch(x, slots, out=far)
    near = B.expert_dispatch(x, slots)
    assert torch.equal(far.contiguous(), near)
    assert torch.equal(B.expert_combine(far, slots, w), B.expert_combine(near, slots, w))
    dy, dw = B.expert_combine_grad(x, near, slots, w)
    far_dy, far_dw = B.expert_combine_grad(x, far, slots, w)
    assert torch.equal(dy, far_dy) and torch.equal(dw, far_dw)


def test_bad_slots_are_masked_and_reported(B):
    x = torch.ones(3, 8, device="cuda")
    slots = torch.tensor([[0, 99], [-5, 1], [2, -1]], dtype=torch.int32, device="cuda")
    out = B.expert_dispatch(x, slots, out=torch.zeros(4, 8, device="cuda"))
    assert out.sum(1).tolist() == [8, 8, 8, 0]
    assert B.device_error() == 0x100
    assert B.expert_combine(out, slots).sum(1).tolist() == [8, 8, 8]
    assert B.device_error() == 0x100
    dy, dw = B.expert_combine_grad(x, out, slots)
    assert dw.tolist() == [[8, 0], [0, 8], [8, 0]] and dy.sum(1).tolist() == [8, 8, 8, 0]
    assert B.device_error() == 0x100


def test_empty(B):
    e = lambda *s: torch.zeros(*s, device="cuda")
    no = torch.zeros(0, 2, dtype=torch.int32, device="cuda")
    assert tuple(B.expert_dispatch(e(0, 8), no).shape) == (0, 8)
    assert tuple(B.expert_combine(e(5, 8), no).shape) == (0, 8)
    none = torch.full((3, 2), -1, dtype=torch.int32, device="cuda")
    assert (B.expert_combine(e(0, 8), none) == 0).all()
    dy, dw = B.expert_combine_grad(e(3, 8) + 1, e(6, 8) + 1, none)
    assert (dy == 0).all() and (dw == 0).all()
    assert tuple(B.expert_combine(e(4, 8), torch.zeros(3, 0, dtype=torch.int32, device="cuda")).shape) == (3, 8)


def _moe(B, x, ids, w, w1, w2, experts, hidden):
    """A feed-forward layer of experts: sort, quantise once per token, dispatch codes and exponents, product, relu,
    quantise, product, combine."""
    off, slots = B.expert_sort(ids, experts)
    q, s = B.quant_mxfp4(x)
    rows = ids.numel()
    qr = torch.zeros(rows, q.stride(0), dtype=torch.uint8, device="cuda")[:, :q.shape[1]]
    sr = torch.zeros(rows, s.stride(0), dtype=torch.uint8, device="cuda")[:, :s.shape[1]]
    B.expert_dispatch(q, slots, out=qr)
    B.expert_dispatch(s, slots, out=sr)
    h = torch.zeros(rows, hidden, dtype=torch.bfloat16, device="cuda")
    B.matmul_mxfp4(qr, sr, *w1, offsets=off, out=h)
    h = B.elemwise_unary("relu", h)
    hq, hs = B.quant_mxfp4(h)
    y = torch.zeros(rows, x.shape[1], dtype=torch.bfloat16, device="cuda")
    B.matmul_mxfp4(hq, hs, *w2, offsets=off, out=y)
    return off, slots, qr, sr, h, y, B.expert_combine(y, slots, w)


def _expert_weights(B, experts, n, k, seed):
    g = torch.Generator().manual_seed(seed)
    flat = (torch.randn(experts * n, k, generator=g) * 0.05).to(torch.bfloat16).cuda()
    q, s = B.quant_mxfp4(flat)
    cut = lambda t: t.as_strided((experts, n, t.shape[1]), (n * t.stride(0), t.stride(0), 1))
    return flat, (cut(q), cut(s))


@pytest.mark.parametrize("tokens,top_k,experts,cols,hidden", [(3, 2, 4, 256, 320), (64, 4, 8, 512, 288), (600, 2, 4, 320, 1024)])
def test_layer(B, tokens, top_k, experts, cols, hidden):
    g = torch.Generator().manual_seed(tokens)
    x = torch.randn(tokens, cols, generator=g).to(torch.bfloat16).cuda()
    ids = _ids(tokens, top_k, experts, tokens + 1).cuda()
    w = torch.rand(tokens, top_k, generator=g).cuda()
    _, w1 = _expert_weights(B, experts, hidden, cols, 1)
    _, w2 = _expert_weights(B, experts, cols, hidden, 2)
    off, slots, qr, sr, h, y, out = _moe(B, x, ids, w, w1, w2, experts, hidden)
    wo, wsl = R.sort(ids.tolist(), experts)
    assert np.array_equal(off.cpu().numpy(), wo) and np.array_equal(slots.cpu().numpy(), wsl)
    xv = R.quant(x)[2]
    half = torch.finfo(torch.bfloat16).eps / 2
    for e in range(experts):
        w1v = R.decode(w1[0][e], w1[1][e], cols)
        w2v = R.decode(w2[0][e], w2[1][e], hidden)
        for t, j in np.argwhere(ids.cpu().numpy() == e)[:40]:
            r = wsl[t, j]
            ref = xv[t] @ w1v.T
            tol = R.product_tolerance(xv[t:t + 1], w1v, cols, torch.bfloat16)(ref[None])[0]
            got = h[r].cpu().double().numpy()
            assert (np.abs(got - np.maximum(ref, 0)) <= tol).all()
            hv = R.quant(h[r:r + 1])[2]                                # from the layer's own intermediate, as rounded there
            ref = hv @ w2v.T
            assert (np.abs(y[r].cpu().double().numpy() - ref) <= R.product_tolerance(hv, w2v, hidden, torch.bfloat16)(ref)).all()
    yd, wd = y.cpu().double().numpy(), w.cpu().double().numpy()
    for t in range(tokens):
        live = wsl[t] >= 0
        terms = wd[t][live, None] * yd[wsl[t][live]]
        ref = terms.sum(0)
        assert (np.abs(out[t].cpu().double().numpy() - ref) <= half * np.abs(ref) * 1.001 + top_k * 2.0 ** -23 * np.abs(terms).sum(0)).all()


def test_layer_captured_and_replayed(B):
    tokens, top_k, experts, cols, hidden = 16, 2, 4, 256, 256
    x = torch.randn(tokens, cols, device="cuda").to(torch.bfloat16)
    ids = _ids(tokens, top_k, experts, 3).cuda()
    w = torch.rand(tokens, top_k, device="cuda")
    _, w1 = _expert_weights(B, experts, hidden, cols, 1)
    _, w2 = _expert_weights(B, experts, cols, hidden, 2)
    _moe(B, x, ids, w, w1, w2, experts, hidden)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = _moe(B, x, ids, w, w1, w2, experts, hidden)
    for seed in (5, 6):
        ids.copy_(_ids(tokens, top_k, experts, seed))
        x.copy_(torch.randn(tokens, cols, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        got = [t.clone() for t in res]
        want = _moe(B, x, ids, w, w1, w2, experts, hidden)
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_two_streams_at_once(B):
    """Long sorts take scratch: each stream its own."""
    ids = [_ids(20000, 4, 64, s).cuda() for s in (1, 2)]
    want = [R.sort(i.tolist(), 64) for i in ids]
    streams = [torch.cuda.Stream() for _ in ids]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for st, i in zip(streams, ids):
            with torch.cuda.stream(st):
                got.append(B.expert_sort(i, 64))
        torch.cuda.synchronize()
        for (o, s), (wo, ws) in zip(got, want):
            assert np.array_equal(o.cpu().numpy(), wo) and np.array_equal(s.cpu().numpy(), ws)


@pytest.mark.parametrize("k", [96, 2900])
def test_dispatched_codes_go_into_a_product(B, k):
    """Rows of codes and exponents whose length is no multiple of 16 bytes, through dispatch's own result."""
    g = torch.Generator(device="cuda").manual_seed(k)
    x = torch.randn(40, k, device="cuda", generator=g)
    w = torch.randn(4 * 70, k, device="cuda", generator=g)
    ids = torch.randint(0, 4, (40, 2), device="cuda", generator=g)
    off, slots = B.expert_sort(ids, 4)
    q, s = B.quant_mxfp4(x)
    qw, sw = B.quant_mxfp4(w)
    qr, sr = B.expert_dispatch(q, slots), B.expert_dispatch(s, slots)
    cut = lambda t: t.as_strided((4, 70, t.shape[1]), (70 * t.stride(0), t.stride(0), 1))
    y = B.matmul_mxfp4(qr, sr, cut(qw), cut(sw), offsets=off, out_dtype=torch.float32)
    full = B.matmul_mxfp4(q, s, qw, sw, out_dtype=torch.float32)          # every token with every expert: the same sums up to order
    for t in range(40):
        for j in range(2):
            e = int(ids[t, j])
            ref = full[t, 70 * e:70 * e + 70].double()
            # sums of k products in f32, each order off by at most k / 2 ulps of the sum of magnitudes
            mags = B.dequant_mxfp4(q[t:t + 1], s[t:t + 1]).abs().double() @ B.dequant_mxfp4(qw, sw).abs().double()[70 * e:70 * e + 70].T
            assert ((y[int(slots[t, j])].double() - ref).abs() <= 2 * k * 2.0 ** -24 * mags[0]).all()


@pytest.mark.parametrize("tokens,top_k,experts,n", [(7, 2, 4, 96), (300, 2, 4, 1000)])
def test_grouped_product_makes_zeros_of_rows_without_a_group(B, tokens, top_k, experts, n):
    """Masked choices leave rows behind the last expert's; a result made by the call holds zeros there, whatever the
    memory held before."""
    k = 256
    g = torch.Generator().manual_seed(tokens)
    ids = _ids(tokens, top_k, experts, tokens, masked=0.5).cuda()
    off, slots = B.expert_sort(ids, experts)
    q, s = B.quant_mxfp4(torch.randn(tokens, k, generator=g).cuda())
    _, w = _expert_weights(B, experts, n, k, 1)
    qr, sr = B.expert_dispatch(q, slots), B.expert_dispatch(s, slots)
    want = B.matmul_mxfp4(qr, sr, *w, offsets=off, out=torch.zeros(tokens * top_k, n, dtype=torch.bfloat16, device="cuda"))
    torch.cuda.synchronize()
    held = int(off[-1])
    assert 0 < held < tokens * top_k
    torch.full((tokens * top_k, n), float("nan"), dtype=torch.bfloat16, device="cuda")     # freed at once, for the next call
    got = B.matmul_mxfp4(qr, sr, *w, offsets=off)
    assert (got[held:] == 0).all() and torch.equal(got, want)


FIRST_CALLS = """
import sys
sys.path.insert(0, sys.argv[1])
import torch
import bsir as B
g = torch.Generator(device="cuda").manual_seed(1)
x = torch.randn(96, 256, device="cuda", generator=g).bfloat16()
w = torch.randn(4 * 64, 256, device="cuda", generator=g).bfloat16()
ids = torch.randint(-1, 4, (96, 2), device="cuda", generator=g)
wt = torch.rand(96, 2, device="cuda", generator=g)
longer = torch.randn(16, 8192, device="cuda", generator=g).bfloat16()
wide = torch.randn(2048, 8192, device="cuda", generator=g).bfloat16()
many = torch.randint(-1, 60, (9000, 2), device="cuda", generator=g)        # the largest cluster

def step():
    off, slots = B.expert_sort(ids, 4)
    q, s, qt, st = B.quant_mxfp4_both(x)
    qw, sw = B.quant_mxfp4(w)
    cut = lambda t: t.as_strided((4, 64, t.shape[1]), (64 * t.stride(0), t.stride(0), 1))
    y = B.matmul_mxfp4(B.expert_dispatch(q, slots), B.expert_dispatch(s, slots), cut(qw), cut(sw), offsets=off)
    out = B.expert_combine(y, slots, wt)
    few = B.matmul_mxfp4(*B.quant_mxfp4(longer), *B.quant_mxfp4(wide), out_dtype=torch.float32)     # a cluster shares K
    return off, slots, B.dequant_mxfp4(qt, st), y, out, *B.expert_combine_grad(out, y, slots, wt), few, *B.expert_sort(many, 60)

graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, capture_error_mode=sys.argv[2]):
    got = step()
graph.replay()
torch.cuda.synchronize()
assert B.device_error() == 0
assert all(torch.equal(a, b) for a, b in zip(got, step()))
assert B.matmul_mxfp4_form(16, 2048, 8192)[2] > 1
print("same")
"""


@pytest.mark.parametrize("mode", ["global", "thread_local"])
def test_first_calls_inside_a_capture(mode):
    """A process whose first calls are captured: nothing has to run once before."""
    import bsir
    root = os.path.dirname(os.path.dirname(os.path.abspath(bsir.__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS, root, mode], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stdout + r.stderr


@pytest.mark.parametrize("tokens,top_k", [(20000, 4), (45000, 4)])
def test_long_sorts_on_two_streams(B, tokens, top_k):
    """Two clusters at work side by side; the longer sort's warps go over their choices twice."""
    ids = [_ids(tokens, top_k, 64, s).cuda() for s in (3, 4)]
    alone = [B.expert_sort(i, 64) for i in ids]
    want = [R.sort(i.tolist(), 64) for i in ids]
    streams = [torch.cuda.Stream() for _ in ids]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for st, i in zip(streams, ids):
            with torch.cuda.stream(st):
                got.append(B.expert_sort(i, 64))
        torch.cuda.synchronize()
        for (o, s), (ao, as_), (wo, ws) in zip(got, alone, want):
            assert torch.equal(o, ao) and torch.equal(s, as_)
    assert np.array_equal(o.cpu().numpy(), wo) and np.array_equal(s.cpu().numpy(), ws)
