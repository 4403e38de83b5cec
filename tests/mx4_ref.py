"""64-bit plain forms of the MXFP4 cache's operators and of packed attention, for the tests (CPU, one head after another)."""
import math

import torch

F64 = torch.float64
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=F64)


def randn(shape, std, seed):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(torch.bfloat16)


def llama_table(positions, width):
    f = 10000.0 ** (-torch.arange(0, width, 2, dtype=F64) / width)
    a = torch.arange(positions, dtype=F64)[:, None] * f
    a = torch.cat((a, a), 1)
    return torch.stack((a.cos(), a.sin())).float()


def gptj_table(positions, width):
    f = 10000.0 ** (-torch.arange(0, width, 2, dtype=F64) / width)
    a = torch.arange(positions, dtype=F64)[:, None] * f
    return torch.cat((a.sin(), a.cos()), 1).float()


def turn(x, weight, eps, table, pos, style):
    """Norm and rotation of x [T][heads][H]; also the sum of the magnitudes that a rotated value is the sum of."""
    x = x.to(F64)
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.to(F64)
    y, size = x.clone(), x.abs().clone()
    if table is None:
        return y, size
    positions, width = table.shape[-2:]
    half = width // 2
    for t in range(x.shape[0]):
        p = int(pos[t])
        if not 0 <= p < positions:
            continue
        for i in range(half):
            a, b = (i, half + i) if style == "llama" else (2 * i, 2 * i + 1)
            c, s = (table[0, p, i], table[1, p, i]) if style == "llama" else (table[p, half + i], table[p, i])
            c, s = float(c), float(s)
            y[t, :, a], size[t, :, a] = x[t, :, a] * c - x[t, :, b] * s, (x[t, :, a] * c).abs() + (x[t, :, b] * s).abs()
            y[t, :, b], size[t, :, b] = x[t, :, b] * c + x[t, :, a] * s, (x[t, :, b] * c).abs() + (x[t, :, a] * s).abs()
    return y, size


def encode(x):
    """(codes [..][H/2], scales [..][H/32]) of x in 64 bits."""
    blocks = x.to(F64).unflatten(-1, (-1, 32))
    top = blocks.abs().amax(-1)
    finite = torch.isfinite(blocks).all(-1)
    exponent = torch.frexp(torch.where(finite, top, torch.ones_like(top))).exponent - 1
    byte = (exponent + 125).clamp(0, 254)
    byte = torch.where(top < 2.0 ** -124, torch.zeros_like(byte), byte)
    byte = torch.where(finite, byte, torch.full_like(byte, 255))
    some = (byte > 0) & (byte < 255)
    a = torch.where(some[..., None], blocks.abs() * 2.0 ** (127 - byte.to(F64))[..., None], torch.zeros_like(blocks))
    d = (a[..., None] - GRID).abs()
    # nearest; of two as near the even code
    order = d * 4 + torch.arange(8) % 2 * torch.finfo(F64).tiny
    near = (d == d.amin(-1, keepdim=True))
    order = torch.where(near, torch.arange(8).to(F64) % 2, torch.full_like(d, 9.0))
    code = order.argmin(-1)
    code = code + 8 * ((blocks < 0) & (code > 0))
    code = code.flatten(-2)
    return (code[..., 0::2] | code[..., 1::2] << 4).to(torch.uint8), byte.to(torch.uint8)


def decode(codes, scales):
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    v = torch.cat((GRID, -GRID))[code].unflatten(-1, (-1, 32))
    s = 2.0 ** (scales.to(F64) - 127)
    s = torch.where(scales == 0, torch.zeros_like(s), torch.where(scales == 255, torch.full_like(s, math.nan), s))
    return (v * s[..., None]).flatten(-2)


def attend(q, k, v, past, mask=None):
    """q [n][Nq][H] bf16 behind `past` keys, k, v [Nkv][keys][H] in 64 bits.  Returns the output and the largest error that
    the kernels' roundings may make of it: the probabilities in bf16 (half a step each, and their sum), scores and
    sums in fp32, the output rounded to bf16."""
    n, nq, H = q.shape
    nkv, keys = k.shape[:2]
    out = torch.zeros((n, nq, H), dtype=F64)
    tol = torch.zeros_like(out)
    for i in range(n):
        see = torch.arange(keys) <= past + i
        add = torch.zeros(keys, dtype=F64)
        if mask is not None:
            m = min(keys, mask.shape[0])
            add[:m] = mask[:m].to(F64)
            see &= ~torch.isneginf(add)
        if not bool(see.any()):
            continue
        for h in range(nq):
            kk, vv = k[h * nkv // nq][see], v[h * nkv // nq][see]
            s = kk @ q[i, h].to(F64) / math.sqrt(H) + add[see]
            p = torch.softmax(s, 0)
            out[i, h] = p @ vv
            # fp32 scores: H products and sums, the mask's rounding where it is finite and large
            es = (H + 4) * 2.0 ** -24 * float((kk.abs() @ q[i, h].to(F64).abs()).max()) / math.sqrt(H)
            es += 2.0 ** -23 * float(s.abs().max()) if float(s.abs().max()) < 1e30 else 0.0
            rel = 2.0 * 2.0 ** -8 + 2 * es + 2.0 ** -12 + keys * 2.0 ** -23
            tol[i, h] = 2.0 ** -8 * out[i, h].abs() + rel * (p @ vv.abs()) * 1.01
    return out, tol + 2.0 ** -126


def attend_rows(q, k, v, past):
    """`attend` without a mask, one head at a time instead of one token and head."""
    n, nq, H = q.shape
    nkv, keys = k.shape[:2]
    out, tol = torch.zeros((n, nq, H), dtype=F64), torch.zeros((n, nq, H), dtype=F64)
    hidden = torch.ones((n, keys), dtype=torch.bool).triu(past + 1)
    for h in range(nq):
        qq, kk, vv = q[:, h].to(F64), k[h * nkv // nq], v[h * nkv // nq]
        s = (qq @ kk.t() / math.sqrt(H)).masked_fill(hidden, -math.inf)
        p = torch.softmax(s, 1)
        out[:, h] = p @ vv
        es = (H + 4) * 2.0 ** -24 * (qq.abs() @ kk.abs().t()).amax(1, keepdim=True) / math.sqrt(H)
        es = es + 2.0 ** -23 * s.masked_fill(hidden, 0.0).abs().amax(1, keepdim=True)
        rel = 2.0 * 2.0 ** -8 + 2 * es + 2.0 ** -12 + keys * 2.0 ** -23
        tol[:, h] = 2.0 ** -8 * out[:, h].abs() + rel * (p @ vv.abs()) * 1.01
    return out, tol + 2.0 ** -126
