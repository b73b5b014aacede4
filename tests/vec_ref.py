"""TEST-ONLY: the document-vector operators from their definitions, in 64 bits on the CPU (torch float64 / numpy), and the
packed 4-bit layout of include/mdd.h read element by element."""
import numpy as np
import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # half a step, relative
SUBNORMAL = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
U32 = 2.0 ** -24


def half(dtype, magnitude):
    """half a step of a number of that magnitude.  Below the type's smallest normal number (2^-14 in float16) the step no longer
    shrinks with the number: it stays at 2^-24, so the rounding is off by up to 2^-25 whatever the value."""
    return HALF[dtype] * magnitude + SUBNORMAL[dtype]


GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def embed(table, ids, offsets, scale, mode):
    """(out, sum of the magnitudes that went into it, number of them), float64"""
    t = table.double().cpu()
    ids = ids.cpu().long()
    ok = (ids >= 0) & (ids < t.shape[0])
    rows = torch.zeros(ids.numel(), t.shape[1], dtype=torch.float64)
    rows[ok] = t[ids[ok]]
    if offsets is None:
        return rows * scale, rows.abs() * abs(scale), torch.ones(ids.numel())
    offs = offsets.cpu().tolist()
    n = len(offs) - 1
    out, mag, cnt = torch.zeros(n, t.shape[1], dtype=torch.float64), torch.zeros(n, t.shape[1], dtype=torch.float64), torch.zeros(n)
    for d in range(n):
        e = min(offs[d + 1], ids.numel())
        b = min(offs[d], e)
        k = int(ok[b:e].sum())
        f = (scale / k if k else 0.0) if mode == "mean" else scale
        part = rows[b:e][ok[b:e]]
        out[d], mag[d], cnt[d] = part.sum(0) * f, part.abs().sum(0) * abs(f), k
    return out, mag, cnt


def embed_backward(grad, ids, n_rows, offsets, scale, mode):
    g = grad.double().cpu()
    ids = ids.cpu().long()
    ok = (ids >= 0) & (ids < n_rows)
    out, mag, cnt = (torch.zeros(n_rows, g.shape[1], dtype=torch.float64) for _ in range(3))
    offs = list(range(ids.numel() + 1)) if offsets is None else offsets.cpu().tolist()
    for d in range(len(offs) - 1):
        e = min(offs[d + 1], ids.numel())
        b = min(offs[d], e)
        k = int(ok[b:e].sum())
        if not k:
            continue
        f = scale / k if mode == "mean" and offsets is not None else scale
        idx = ids[b:e][ok[b:e]]
        out.index_add_(0, idx, (g[d] * f).expand(k, -1))
        mag.index_add_(0, idx, (g[d] * f).abs().expand(k, -1))
        cnt.index_add_(0, idx, torch.ones(k, g.shape[1], dtype=torch.float64))
    return out, mag, cnt


def rms_norm(x, weight, residual, eps):
    h = x.double().cpu()
    if residual is not None:
        h = h + residual.double().cpu()
    r = 1 / torch.sqrt((h * h).mean(1) + eps)
    y = h * r[:, None]
    if weight is not None:
        y = y * weight.double().cpu()
    return y, h, r


def q8(x, weight, residual, eps, kind):
    """(codes as float64, scales)"""
    _, h, r = rms_norm(x, None, residual, eps)
    y = h if weight is None else h * weight.double().cpu()
    top = 127.0 if kind == "int8" else 448.0
    big = y.abs().amax(1)
    fine = torch.isfinite(y).all(1)
    z = torch.where((fine & (big > 0))[:, None], y * top / big[:, None], torch.zeros_like(y))
    if kind == "int8":
        q = torch.round(z)
    else:
        e = torch.floor(torch.log2(z.abs().clamp(min=2.0 ** -6)))
        q = torch.round(z / torch.exp2(e - 3)) * torch.exp2(e - 3)
    scale = torch.where(fine, big * r / top, torch.full_like(big, float("nan")))
    return q, scale


def mx_codes(x):
    """(codes 0..15 uint8 [n, dim], scale bytes uint8 [n, ceil(dim / 32)]) from the definition"""
    a = x.float().cpu().numpy().astype(np.float64)
    n, dim = a.shape
    kb = (dim + 31) // 32
    codes, sb = np.zeros((n, dim), np.uint8), np.zeros((n, kb), np.uint8)
    mid = (GRID[1:] + GRID[:-1]) / 2
    for b in range(kb):
        blk = a[:, b * 32: (b + 1) * 32]
        top = np.abs(blk).max(1)
        bad = ~np.isfinite(blk).all(1)
        e = np.full(n, -127.0)
        pos = (top > 0) & ~bad
        e[pos] = np.maximum(np.floor(np.log2(top[pos])) - 2, -127)
        m = np.abs(np.where(bad[:, None], 0, blk)) * np.exp2(-e)[:, None]
        c = np.zeros(m.shape, np.uint8)
        for k in range(7):                  # between grid values k and k + 1: up beyond the middle, and on it if k is odd
            c += ((m > mid[k]) | ((m == mid[k]) & (k % 2 == 1))).astype(np.uint8)
        c |= np.signbit(blk).astype(np.uint8) << 3
        codes[:, b * 32: (b + 1) * 32] = np.where(bad[:, None], 0, c)
        sb[:, b] = np.where(bad, 255, e + 127).astype(np.uint8)
    return codes, sb


def mx_unpack(codes, scales, rows, cols):
    """(codes [rt*32, ct*128], scale bytes [rt*32, ct*4]) of the packed layout, padding included"""
    c, s = codes.cpu().numpy(), scales.cpu().numpy()
    rt, ct = (rows + 31) // 32, (cols + 127) // 128
    c, s = c.reshape(rt, ct, 4, 32, 16), s.reshape(rt, ct, 2, 32, 2)
    full, sb = np.zeros((rt * 32, ct * 128), np.uint8), np.zeros((rt * 32, ct * 4), np.uint8)
    for i in range(rt):
        for j in range(ct):
            for b in range(4):
                full[i * 32: i * 32 + 32, j * 128 + b * 32: j * 128 + b * 32 + 32: 2] = c[i, j, b] & 15
                full[i * 32: i * 32 + 32, j * 128 + b * 32 + 1: j * 128 + b * 32 + 32: 2] = c[i, j, b] >> 4
                sb[i * 32: i * 32 + 32, j * 4 + b] = s[i, j, b & 1, :, b >> 1]
    return full, sb


def mx_values(codes, sb):
    v = np.where(codes & 8, -1.0, 1.0) * GRID[codes & 7]
    f = np.where(sb == 255, np.nan, np.exp2(sb.astype(np.float64) - 127))
    return v * np.repeat(f, 32, 1)[:, : codes.shape[1]]


def cosines(a, b):
    a, b = a.double(), b.double()
    n = torch.sqrt((a * a).sum(1) * (b * b).sum(1))
    return torch.where(n > 0, (a * b).sum(1) / torch.where(n > 0, n, torch.ones_like(n)), torch.zeros_like(n))
