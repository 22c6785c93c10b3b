"""Plain 64-bit statements of the microscaled 4-bit format and of expert routing, on the CPU (numpy)."""
import numpy as np
import torch

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quant(x):
    """[rows, cols] tensor -> (codes, exponents, values): nearest grid value, a tie to the even code."""
    x = x.detach().cpu().double().numpy()
    rows, cols = x.shape
    nb = -(-cols // 32)
    p = np.zeros((rows, nb * 32))
    p[:, :cols] = x
    p = p.reshape(rows, nb, 32)
    byte = np.zeros((rows, nb), np.int64)
    code = np.zeros(p.shape, np.int64)
    for r in range(rows):
        for b in range(nb):
            blk = p[r, b]
            if not np.isfinite(blk).all():
                byte[r, b] = 255
                continue
            top = np.abs(blk).max()
            e = -127 if top == 0 else max(-127, int(np.frexp(top)[1]) - 1 - 2)
            byte[r, b] = e + 127
            z = np.abs(np.ldexp(blk, -e))
            d = np.abs(z[:, None] - GRID[None, :])
            near = d == d.min(axis=1, keepdims=True)
            even = near & (np.arange(8) % 2 == 0)[None, :]
            code[r, b] = np.where(even.any(1), even.argmax(1), near.argmax(1)) + 8 * np.signbit(blk)
    values = decode_grid(code.reshape(rows, -1), byte)[:, :cols]
    c = code.reshape(rows, -1)
    packed = (c[:, 0::2] + 16 * c[:, 1::2])[:, :(cols + 1) // 2]
    return packed.astype(np.uint8), byte.astype(np.uint8), values


def decode_grid(code, byte):
    mag = GRID[code & 7] * np.where(code >= 8, -1.0, 1.0)
    scale = np.ldexp(1.0, byte.astype(np.int64) - 127)
    scale = np.where(byte == 255, np.nan, scale)
    return mag * np.repeat(scale, 32, axis=1)[:, :code.shape[1]]


def decode(q, s, cols):
    """uint8 tensors -> 64-bit values [rows, cols]."""
    q, s = q.detach().cpu().numpy().astype(np.int64), s.detach().cpu().numpy().astype(np.int64)
    code = np.stack((q & 15, q >> 4), axis=-1).reshape(q.shape[0], -1)[:, :cols]
    return decode_grid(code, s)


def product_tolerance(a, b, k, dtype):
    """What an f32 sum of k exact products may be off: every addition by a step of its result, at most the sum of the
    products' magnitudes (2^-23 of it: the tensor core's adder need not round to nearest), then half a step of C."""
    return lambda ref: (k + 1) * 2.0 ** -23 * (np.abs(a) @ np.abs(b).T) + torch.finfo(dtype).eps / 2 * np.abs(ref) + float(torch.finfo(dtype).tiny)


def random_codes(rows, k, seed, lo=120, hi=134, device="cuda"):
    """Random codes and exponents with 16-byte aligned rows (what bsir.quant_mxfp4 lays out)."""
    g = torch.Generator().manual_seed(seed)
    kb, ks = (k + 1) // 2, -(-k // 32)
    q = torch.zeros(rows, (kb + 15) // 16 * 16, dtype=torch.uint8)
    s = torch.zeros(rows, (ks + 15) // 16 * 16, dtype=torch.uint8)
    q[:, :kb] = torch.randint(0, 256, (rows, kb), generator=g, dtype=torch.uint8)
    if k % 2:
        q[:, kb - 1] &= 15
    s[:, :ks] = torch.randint(lo, hi + 1, (rows, ks), generator=g).to(torch.uint8)
    return q.to(device)[:, :kb], s.to(device)[:, :ks]


def sort(ids, experts):
    """ids (nested list) -> offsets, slots."""
    rows = [[] for _ in range(experts)]
    top_k = len(ids[0]) if ids else 0
    for t, choice in enumerate(ids):
        for j, e in enumerate(choice):
            if 0 <= e < experts:
                rows[e].append(t * top_k + j)
    offsets, slots, n = [0], [-1] * (len(ids) * top_k), 0
    for lst in rows:
        for i in lst:
            slots[i] = n
            n += 1
        offsets.append(n)
    return np.array(offsets, np.int32), np.array(slots, np.int32).reshape(len(ids), top_k)
