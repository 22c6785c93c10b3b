"""Operators of a mixture-of-experts layer with microscaled 4-bit weights, and of its linear layers: what one pass of
each takes and returns, in plain torch operations (``own`` false) and as the library's user calls them (``own`` true).

MXFP4: blocks of 32 elements along the contracted axis share one power of two, an 8-bit exponent (value 2^(byte-127),
255 = NaN); an element is e2m1 (sign, 0 0.5 1 1.5 2 3 4 6), two to a byte, the lower half first.  The exponent is
floor(log2(largest magnitude)) - 2, at least -127; elements round to nearest even and stop at +-6; a block that holds a
NaN or an infinity is NaN.

Experts: ids[t, j] is the expert of token t's j-th choice, -1 (or any number outside the experts) for none.  Sorting
gives offsets (rows offsets[e] .. offsets[e + 1] belong to expert e) and slots (the row of each choice, -1 for none),
choices of one expert in the order of their place in ids.

Sizes: hidden 4096 and 14336 are the ones that the package's workloads use; the others are generic.
"""
import math
import os
import sys

import torch

own = False

_BLOCK = 32
_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _bsir():
    p = os.path.join(os.getcwd(), "ascendnpu-ir_b200")
    if p not in sys.path:
        sys.path.insert(0, p)
    import bsir
    return bsir


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one decode step's activations, quantised for a 4-bit product and read back
        {"name": "quant_small", "kind": "quant", "rows": 16, "cols": 4096, "axis": 1, "dtype": "f16"},
        # the activations of a prompt batch
        {"name": "quant_large", "kind": "quant", "rows": 16384, "cols": 4096, "axis": 1, "dtype": "bf16"},
        # one token against a feed-forward weight: the weight stream is all there is
        {"name": "product_one_row", "kind": "product", "m": 1, "n": 14336, "k": 4096, "out": "bf16", "bias": False},
        # a ragged batch against odd sizes, K not a multiple of a block
        {"name": "product_ragged", "kind": "product", "m": 333, "n": 5001, "k": 2900, "out": "f16", "bias": True},
        # a prompt batch against a feed-forward weight
        {"name": "product_large", "kind": "product", "m": 4096, "n": 14336, "k": 4096, "out": "bf16", "bias": False},
        # training: both gradients of a linear layer, operands quantised along the axis each product contracts
        {"name": "linear_backward", "kind": "backward", "m": 4096, "n": 4096, "k": 4096},
        # a decode step over experts: 32 tokens with 4 choices among 64 experts, two rows an expert
        {"name": "grouped_decode", "kind": "grouped", "tokens": 32, "top_k": 4, "experts": 64, "n": 2048, "k": 4096,
         "out": "bf16", "bias": False, "masked": 0.0, "skew": 0.0},
        # a prompt batch over experts, unevenly spread, some choices belonging to no expert here
        {"name": "grouped_large", "kind": "grouped", "tokens": 4096, "top_k": 4, "experts": 32, "n": 4096, "k": 4096,
         "out": "bf16", "bias": True, "masked": 0.05, "skew": 1.0},
        # sorting a decode step's tokens by expert
        {"name": "dispatch_small", "kind": "dispatch", "tokens": 32, "top_k": 4, "experts": 64, "cols": 4096,
         "dtype": "bf16", "ids": "i32", "masked": 0.0, "skew": 0.0},
        # sorting a prompt batch's tokens, padding tokens without an expert among them
        {"name": "dispatch_large", "kind": "dispatch", "tokens": 8192, "top_k": 8, "experts": 128, "cols": 4096,
         "dtype": "bf16", "ids": "i64", "masked": 0.05, "skew": 1.0},
        # a decode step's expert results back to their tokens
        {"name": "combine_small", "kind": "combine", "tokens": 32, "top_k": 4, "experts": 64, "cols": 4096, "dtype": "bf16",
         "masked": 0.0, "grad": False},
        # training: results back to their tokens, and the gradients of the results and of the weights
        {"name": "combine_grad_large", "kind": "combine", "tokens": 8192, "top_k": 8, "experts": 128, "cols": 4096,
         "dtype": "bf16", "masked": 0.05, "grad": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quant", "product", "product", "backward", "grouped", "grouped", "dispatch", "combine"])
    if kind == "quant":
        rows = _log(rng, 1, 16384)
        cols = _log(rng, 64, 16384)
        cols = min(cols, (1 << 26) // rows)
        if rng.random() < 0.7:
            cols = max(64, cols // 64 * 64)
        return {"kind": kind, "rows": rows, "cols": cols, "axis": rng.choice([1, 1, 0]), "dtype": rng.choice(["f32", "f16", "bf16"])}
    if kind == "product":
        k = _log(rng, 256, 14336)
        n = _log(rng, 256, 14336)
        if rng.random() < 0.6:
            k, n = max(256, k // 128 * 128), max(256, n // 128 * 128)
        m = min(_log(rng, 1, 4096), (4096 * 14336 * 4096) // (n * k))
        return {"kind": kind, "m": m, "n": n, "k": k, "out": rng.choice(["bf16", "bf16", "f16", "f32"]), "bias": rng.random() < 0.3}
    if kind == "backward":
        even = rng.choice([1, 8, 128])
        return {"kind": kind, "m": _log(rng, 64, 4096), "n": max(256, _log(rng, 256, 4096) // even * even),
                "k": max(256, _log(rng, 256, 4096) // even * even)}
    if kind == "grouped":
        experts = rng.choice([4, 8, 16, 32, 60, 64])
        n, k = _log(rng, 256, 4096) // 32 * 32, _log(rng, 256, 4096) // 32 * 32
        return {"kind": kind, "tokens": _log(rng, 1, 4096), "top_k": rng.choice([1, 2, 4]), "experts": experts, "n": n, "k": k,
                "out": rng.choice(["bf16", "f16"]), "bias": rng.random() < 0.3, "masked": rng.choice([0.0, 0.1]),
                "skew": rng.choice([0.0, 1.0])}
    experts, top_k, cols = rng.choice([8, 32, 60, 128, 256]), rng.choice([1, 2, 4, 6, 8]), _log(rng, 256, 8192)
    cols = max(256, cols // 8 * 8) if rng.random() < 0.8 else cols
    tokens = min(_log(rng, 1, 16384), (8192 * 8 * 4096) // (top_k * cols))
    c = {"kind": kind, "tokens": tokens, "top_k": top_k, "experts": experts, "cols": cols,
         "dtype": rng.choice(["f32", "f16", "bf16", "bf16"]), "masked": rng.choice([0.0, 0.1])}
    if kind == "dispatch":
        c["ids"], c["skew"] = rng.choice(["i32", "i64"]), rng.choice([0.0, 1.0])
    else:
        c["grad"] = rng.random() < 0.5
    if c["dtype"] == "f32":
        c["tokens"] = max(1, c["tokens"] // 2)
    return c


# ------------------------------------------------------------------------------------------------ plain forms
def _pad16(cols):
    return (cols + 15) // 16 * 16


def _bytes_rows(rows, cols, lead=()):
    """uint8 [.., rows, cols] whose rows start 16 bytes aligned, as the library lays codes and exponents out."""
    return torch.zeros(*lead, rows, _pad16(cols), dtype=torch.uint8, device="cuda")[..., :cols]


def _pow2(e):
    """2^e as a 64-bit float for whole e of a 64-bit float tensor, by its bits: exact, as a power function need not be."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _quant(x):
    """[rows, cols] -> (codes [rows, ceil(cols / 2)], exponents [rows, ceil(cols / 32)]), blocks along the row."""
    rows, cols = x.shape
    nb = -(-cols // _BLOCK)
    v = torch.zeros(rows, nb * _BLOCK, dtype=torch.float32, device=x.device)
    v[:, :cols] = x
    v = v.view(rows, nb, _BLOCK)
    amax = v.abs().amax(dim=2)
    bad = ~torch.isfinite(amax)
    e = torch.frexp(torch.where(bad, torch.ones_like(amax), amax))[1] - 3          # floor(log2) - 2
    e = torch.where(amax == 0, torch.full_like(e, -127), e).clamp(min=-127)
    inv = ((127 - e) << 23).view(torch.float32)                                    # 2^-e, exactly
    a = (v * inv[..., None]).abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = code + torch.signbit(v).to(torch.uint8) * 8
    code = torch.where(bad[..., None], torch.zeros_like(code), code).view(rows, nb * _BLOCK)
    q = _bytes_rows(rows, (cols + 1) // 2)
    q.copy_((code[:, 0::2] + code[:, 1::2] * 16)[:, :(cols + 1) // 2])
    s = _bytes_rows(rows, nb)
    s.copy_(torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8))
    return q, s


_VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]


def _dequant(q, s, cols, dtype=torch.float32):
    """codes and exponents -> [rows, cols] values (f32 or f64: exact)."""
    table = torch.tensor(_VALUES, dtype=dtype, device=q.device)
    code = torch.stack((q & 15, q >> 4), dim=-1).view(q.shape[0], -1)[:, :cols]
    scale = _pow2(s.double() - 127.0)
    scale = torch.where(s == 255, torch.full_like(scale, math.nan), scale).to(dtype)
    return table[code.int()] * scale.repeat_interleave(_BLOCK, dim=1)[:, :cols]


def _sort(ids, experts):
    flat = ids.reshape(-1).to(torch.int64)
    key = torch.where((flat >= 0) & (flat < experts), flat, torch.full_like(flat, experts))
    order = torch.argsort(key, stable=True)
    count = torch.bincount(key, minlength=experts + 1)
    offsets = torch.zeros(experts + 1, dtype=torch.int64, device=ids.device)
    offsets[1:] = torch.cumsum(count[:experts], 0)
    rank = torch.empty_like(order)
    rank[order] = torch.arange(order.numel(), device=ids.device)
    slots = torch.where(key < experts, rank, torch.full_like(rank, -1))
    return offsets.int(), slots.int().view(ids.shape)


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _activations(rows, cols, g, dtype=torch.float32):
    """Normal values with the few loud columns that hidden states have."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    loud = torch.rand(cols, generator=g, device="cuda") < 0.005
    return (x * torch.where(loud, 20.0, 1.0)).to(dtype)


def _ids(case, g):
    """Distinct experts per token, popular ones more often with `skew`; whole tokens masked (padding)."""
    t, k, e = case["tokens"], case["top_k"], case["experts"]
    logits = torch.randn(t, e, generator=g, device="cuda")
    logits = logits + case.get("skew", 0.0) * torch.randn(e, generator=g, device="cuda")
    top = torch.topk(logits, min(k, e), dim=1)
    ids, w = top.indices, torch.softmax(top.values, dim=1)
    drop = torch.rand(t, 1, generator=g, device="cuda") < case["masked"]
    return torch.where(drop, torch.full_like(ids, -1), ids), w


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    st = {"case": case}
    if kind == "quant":
        st["x"] = _activations(case["rows"], case["cols"], g, _DT[case["dtype"]])
    elif kind == "product":
        st["a"], st["sa"] = _quant(_activations(case["m"], case["k"], g))
        st["b"], st["sb"] = _quant(torch.randn(case["n"], case["k"], generator=g, device="cuda") * 0.02)
        st["bias"] = torch.randn(case["n"], generator=g, device="cuda") if case["bias"] else None
    elif kind == "backward":
        m, n, k = case["m"], case["n"], case["k"]
        st["dy"] = (torch.randn(m, n, generator=g, device="cuda") * 1e-3).bfloat16()
        st["x"] = _activations(m, k, g, torch.bfloat16)
        w = (torch.randn(n, k, generator=g, device="cuda") * 0.02).bfloat16()
        st["wt"], st["swt"] = _quant(w.t())                      # the weight along n: kept beside the forward's
    elif kind == "grouped":
        e, n, k = case["experts"], case["n"], case["k"]
        ids, _ = _ids(case, g)
        st["offsets"], _ = _sort(ids, e)
        st["a"], st["sa"] = _quant(_activations(case["tokens"] * min(case["top_k"], e), k, g))
        st["b"], st["sb"] = _bytes_rows(n, (k + 1) // 2, (e,)), _bytes_rows(n, -(-k // _BLOCK), (e,))
        for i in range(e):
            q, s = _quant(torch.randn(n, k, generator=g, device="cuda") * 0.02)
            st["b"][i].copy_(q)
            st["sb"][i].copy_(s)
        st["bias"] = torch.randn(e, n, generator=g, device="cuda") if case["bias"] else None
        # rows behind the last expert's are left as they were: a buffer that starts out as zeros
        st["out"] = torch.zeros(st["a"].shape[0], n, dtype=_DT[case["out"]], device="cuda")
    elif kind == "dispatch":
        ids, _ = _ids(case, g)
        st["ids"] = ids.int() if case["ids"] == "i32" else ids
        st["x"] = _activations(case["tokens"], case["cols"], g, _DT[case["dtype"]])
        st["out"] = torch.zeros(ids.numel(), case["cols"], dtype=_DT[case["dtype"]], device="cuda")
    elif kind == "combine":
        ids, st["w"] = _ids(case, g)
        _, st["slots"] = _sort(ids, case["experts"])
        rows = ids.numel()
        st["y"] = torch.randn(rows, case["cols"], generator=g, device="cuda").to(_DT[case["dtype"]])
        if case["grad"]:
            st["dout"] = torch.randn(case["tokens"], case["cols"], generator=g, device="cuda").to(_DT[case["dtype"]])
            st["dy"] = torch.zeros_like(st["y"])                 # rows that no choice names stay as they are
    else:
        raise ValueError(kind)
    return st


# ------------------------------------------------------------------------------------------------ one pass
def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_own(st):
    B = _bsir()
    c = st["case"]
    kind = c["kind"]
    if kind == "quant":
        q, s = B.quant_mxfp4(st["x"], axis=c["axis"])
        return B.dequant_mxfp4(q, s, st["x"].dtype, cols=st["x"].shape[c["axis"]])
    if kind == "product":
        return B.matmul_mxfp4(st["a"], st["sa"], st["b"], st["sb"], bias=st["bias"], out_dtype=_DT[c["out"]])
    if kind == "backward":
        dyq, dys, dytq, dyts = B.quant_mxfp4_both(st["dy"])
        xtq, xts = B.quant_mxfp4(st["x"], axis=0)
        dx = B.matmul_mxfp4(dyq, dys, st["wt"], st["swt"], out_dtype=torch.bfloat16)
        dw = B.matmul_mxfp4(dytq, dyts, xtq, xts, out_dtype=torch.float32)
        return dx, dw
    if kind == "grouped":
        return B.matmul_mxfp4(st["a"], st["sa"], st["b"], st["sb"], bias=st["bias"], offsets=st["offsets"], out=st["out"])
    if kind == "dispatch":
        offsets, slots = B.expert_sort(st["ids"], c["experts"])
        return offsets, slots, B.expert_dispatch(st["x"], slots, out=st["out"])
    out = B.expert_combine(st["y"], st["slots"], st["w"])
    if not c["grad"]:
        return out
    dy, dw = B.expert_combine_grad(st["dout"], st["y"], st["slots"], st["w"], out=st["dy"])
    return out, dy, dw


def _run_plain(st):
    c = st["case"]
    kind = c["kind"]
    if kind == "quant":
        x = st["x"] if c["axis"] == 1 else st["x"].t()
        q, s = _quant(x)
        return _dequant(q, s, x.shape[1]).to(x.dtype)
    if kind == "product":
        out = _dequant(st["a"], st["sa"], c["k"]) @ _dequant(st["b"], st["sb"], c["k"]).t()
        if st["bias"] is not None:
            out = out + st["bias"]
        return out.to(_DT[c["out"]])
    if kind == "backward":
        m, n = c["m"], c["n"]
        dx = _dequant(*_quant(st["dy"]), n) @ _dequant(st["wt"], st["swt"], n).t()
        dw = _dequant(*_quant(st["dy"].t()), m) @ _dequant(*_quant(st["x"].t()), m).t()
        return dx.bfloat16(), dw
    if kind == "grouped":
        out, off = st["out"], st["offsets"].tolist()
        a = _dequant(st["a"], st["sa"], c["k"])
        for e in range(c["experts"]):
            if off[e + 1] > off[e]:
                v = a[off[e]:off[e + 1]] @ _dequant(st["b"][e], st["sb"][e], c["k"]).t()
                out[off[e]:off[e + 1]] = v if st["bias"] is None else v + st["bias"][e]
        return out
    if kind == "dispatch":
        offsets, slots = _sort(st["ids"], c["experts"])
        flat = slots.reshape(-1).long()
        named = (flat >= 0).nonzero()[:, 0]
        out = st["out"]
        out[flat[named]] = st["x"][named // slots.shape[1]]
        return offsets, slots, out
    slots, w = st["slots"].long(), st["w"]
    live = slots >= 0
    acc = torch.zeros(slots.shape[0], c["cols"], dtype=torch.float32, device="cuda")
    for j in range(slots.shape[1]):
        y = st["y"][slots[:, j].clamp(min=0)].float()
        acc += torch.where(live[:, j, None], y * w[:, j, None], torch.zeros_like(y))
    out = acc.to(st["y"].dtype)
    if not c["grad"]:
        return out
    dy, dw, dout = st["dy"], torch.zeros_like(w), st["dout"].float()
    for j in range(slots.shape[1]):
        t = live[:, j].nonzero()[:, 0]
        r = slots[t, j]
        dw[t, j] = (dout[t] * st["y"][r].float()).sum(dim=1)
        dy[r] = (dout[t] * w[t, j, None]).to(dy.dtype)
    return out, dy, dw


# ------------------------------------------------------------------------------------------------ floors
def work(case):
    kind = case["kind"]
    size = {"f32": 4, "f16": 2, "bf16": 2, "i32": 4, "i64": 8}
    code = lambda rows, cols: rows * (-(-cols // 2) + -(-cols // _BLOCK))           # codes and exponents of a matrix
    if kind == "quant":
        e = case["rows"] * case["cols"]
        return {"bytes": 2 * e * size[case["dtype"]], "flops": 2 * e}
    if kind == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": code(m, k) + code(n, k) + m * n * size[case["out"]] + (4 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    if kind == "backward":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": 2 * m * n + 2 * m * k + code(k, n) + 2 * m * k + 4 * n * k, "flops": 4 * m * n * k}
    rows = case["tokens"] * min(case["top_k"], case["experts"])
    live = max(1, int(rows * (1.0 - case["masked"])))
    if kind == "grouped":
        n, k, e = case["n"], case["k"], case["experts"]
        hit = min(e, e * (1.0 - (1.0 - 1.0 / e) ** live))                            # experts with a row, evenly spread
        return {"bytes": code(live, k) + int(hit * code(n, k)) + live * n * size[case["out"]] + (4 * e * n if case["bias"] else 0),
                "flops": 2 * live * n * k}
    row = case["cols"] * size[case["dtype"]]
    if kind == "dispatch":
        return {"bytes": rows * (size[case["ids"]] + 4) + case["tokens"] * row + live * row, "flops": 0}
    if not case["grad"]:
        return {"bytes": rows * 8 + live * row + case["tokens"] * row, "flops": 2 * live * case["cols"]}
    return {"bytes": rows * 12 + 2 * live * row + 2 * case["tokens"] * row, "flops": 5 * live * case["cols"]}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_round(x, axis):
    """x with each block of 32 along `axis` rounded to MXFP4, in 64 bits, from the definition by steps of the grid."""
    v = (x if axis == 1 else x.t()).double()
    rows, cols = v.shape
    nb = -(-cols // _BLOCK)
    p = torch.nn.functional.pad(v, (0, nb * _BLOCK - cols)).reshape(rows, nb, _BLOCK)
    top = p.abs().amax(-1, keepdim=True)
    ok = torch.isfinite(top)
    expo = torch.where(ok & (top > 0), torch.frexp(torch.where(ok, top, torch.ones_like(top)))[1].double() - 3.0,
                       torch.full_like(top, -127.0)).clamp(min=-127.0)
    z = p * _pow2(-expo)
    step = torch.where(z.abs() < 2.0, 0.5, torch.where(z.abs() < 4.0, 1.0, 2.0))    # spacing of 0 .. 2, 2 .. 4, 4 .. 6
    z = (torch.round(z / step) * step).clamp(-6.0, 6.0)                             # torch.round: halves to even
    r = torch.where(ok, z * _pow2(expo), torch.full_like(z, math.nan))
    return r.reshape(rows, nb * _BLOCK)[:, :cols]


def _exact_decode(q, s, cols):
    """Codes and exponents as 64-bit values: (1 + m / 2) 2^(e - 1), or m / 2 with e = 0, times 2^(byte - 127)."""
    c = torch.stack((q & 15, q >> 4), dim=-1).flatten(-2)[..., :cols].long()
    m, e = (c & 1).double(), ((c >> 1) & 3)
    mag = torch.where(e == 0, m * 0.5, (1.0 + 0.5 * m) * _pow2((e - 1).double()))
    mag = torch.where(c >= 8, -mag, mag)
    scale = _pow2(s.double() - 127.0)
    scale = torch.where(s == 255, torch.full_like(scale, math.nan), scale)
    return mag * scale.repeat_interleave(_BLOCK, dim=-1)[..., :cols]


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "quant":
        return _exact_round(st["x"], case["axis"])
    if kind == "product":
        out = _exact_decode(st["a"], st["sa"], case["k"]) @ _exact_decode(st["b"], st["sb"], case["k"]).t()
        return out if st["bias"] is None else out + st["bias"].double()
    if kind == "backward":
        dy, x = st["dy"], st["x"]
        dx = _exact_round(dy, 1) @ _exact_decode(st["wt"], st["swt"], case["n"]).t()
        return dx, _exact_round(dy, 0) @ _exact_round(x, 0).t()
    if kind == "grouped":
        out = torch.zeros(st["out"].shape, dtype=torch.float64, device="cuda")
        off = st["offsets"].tolist()
        for e in range(case["experts"]):
            lo, hi = off[e], off[e + 1]
            if hi > lo:
                w = _exact_decode(st["b"][e], st["sb"][e], case["k"])
                out[lo:hi] = _exact_decode(st["a"][lo:hi], st["sa"][lo:hi], case["k"]) @ w.t()
                if st["bias"] is not None:
                    out[lo:hi] += st["bias"][e].double()
        return out
    if kind == "dispatch":
        ids = st["ids"].cpu().long()
        t, k = ids.shape
        rows = [[] for _ in range(case["experts"])]
        for i, e in enumerate(ids.reshape(-1).tolist()):
            if 0 <= e < case["experts"]:
                rows[e].append(i)
        offsets, slots, order = [0], torch.full((t * k,), -1, dtype=torch.int32), []
        for lst in rows:
            order += lst
            offsets.append(len(order))
        order = torch.tensor(order, dtype=torch.int64)
        slots[order] = torch.arange(order.numel(), dtype=torch.int32)
        out = torch.zeros(st["out"].shape, dtype=torch.float64, device="cuda")
        out[:order.numel()] = st["x"].double()[(order // k).cuda()]
        return torch.tensor(offsets, dtype=torch.int32).cuda(), slots.view(t, k).cuda(), out
    slots, w = st["slots"].long(), st["w"].double()
    live = (slots >= 0).double()
    picked = [st["y"][slots[:, j].clamp(min=0)] for j in range(slots.shape[1])]
    out = torch.zeros(case["tokens"], case["cols"], dtype=torch.float64, device="cuda")
    for j, y in enumerate(picked):
        out += y.double() * (w[:, j] * live[:, j])[:, None]
    if not case["grad"]:
        return out
    dout = st["dout"].double()
    dw = torch.stack([(dout * y.double()).sum(1) for y in picked], dim=1) * live
    dy = torch.zeros(st["y"].shape, dtype=torch.float64, device="cuda")
    for j in range(slots.shape[1]):
        t = (slots[:, j] >= 0).nonzero()[:, 0]
        dy[slots[t, j]] = dout[t] * w[t, j, None]
    return out, dy, dw
