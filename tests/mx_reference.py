"""Plain 64-bit implementations of scored routing and of MXFP4 arithmetic, for the tests."""
from __future__ import annotations

import math

import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def route(logits, bias, K, score, groups=1, topk_groups=1, group_top=1, renorm=True, scale=1.0):
    """(ids int32 [T,K], weights float64 [T,K]) token by token, from the definition."""
    T, E = logits.shape
    per = E // groups
    ids, w = np.full((T, K), -1, np.int32), np.zeros((T, K))
    for t in range(T):
        l = [float(v) for v in logits[t]]
        live = [e for e in range(E) if not math.isnan(l[e]) and l[e] > -math.inf]
        l = [min(v, float(np.finfo(np.float32).max)) for v in l]
        if not live:
            continue
        if score == "sigmoid":
            s = {e: 1.0 / (1.0 + math.exp(-l[e])) if l[e] > -700 else 0.0 for e in live}
        else:
            m = max(l[e] for e in live)
            ex = {e: math.exp(l[e] - m) for e in live}
            d = math.fsum(ex.values())
            s = {e: ex[e] / d for e in live}
        if bias is None:
            key, c = {e: l[e] for e in live}, s
        else:
            ok = [e for e in live if not math.isnan(float(bias[e])) and float(bias[e]) > -math.inf]
            c = {e: s[e] + min(float(bias[e]), float(np.finfo(np.float32).max)) for e in ok}
            key = c
        mine = sorted(key)
        if groups > 1:
            total = {}
            for g in range(groups):
                of = sorted((e for e in mine if e // per == g), key=lambda e: (-key[e], e))[:group_top]
                if of:
                    total[g] = key[of[0]] if group_top == 1 else sum(c[e] for e in of)
            good = sorted(total, key=lambda g: (-total[g], g))[:topk_groups]
            mine = [e for e in mine if e // per in good]
        take = sorted(mine, key=lambda e: (-key[e], e))[:K]
        ids[t, :len(take)] = take
        w[t, :len(take)] = [s[e] for e in take]
    if renorm:
        w = w / (w.sum(1, keepdims=True) + 1e-20)
    return ids, w * scale


def quantize(x):
    """fp64 values [..., cols] -> (codes uint8 [..., cols], scale bytes uint8 [..., cols/32])."""
    x = np.asarray(x, np.float64)
    b = x.reshape(*x.shape[:-1], -1, 32)
    bad = ~np.isfinite(b).all(-1)
    amax = np.abs(np.where(np.isfinite(b), b, 0.0)).max(-1)
    exp = np.where(amax > 0, np.frexp(amax)[1] - 1 - 2, -127)
    s = np.maximum(exp, -127) + 127
    m = np.abs(np.where(np.isfinite(b), b, 0.0)) * 2.0 ** (127.0 - s)[..., None]
    # nearest of the grid, a tie to the even code
    low = np.clip(np.searchsorted(GRID, m, side="right") - 1, 0, 7)
    high = np.minimum(low + 1, 7)
    dl, dh = m - GRID[low], GRID[high] - m
    code = np.where((dl < dh) | ((dl == dh) & (low % 2 == 0)) | (low == 7), low, high).astype(np.uint8)
    code |= (np.signbit(b).astype(np.uint8) << 3)
    return code.reshape(x.shape), np.where(bad, 255, s).astype(np.uint8)


def decode(codes, scales):
    v = np.concatenate([GRID, -GRID])[codes]
    p = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return v * np.repeat(p, 32, -1)


def pack(codes):
    return np.ascontiguousarray(codes[..., 0::2] | (codes[..., 1::2] << 4))


def unpack(q):
    return np.stack((q & 15, q >> 4), -1).reshape(*q.shape[:-1], -1)


def tile(scales):
    """Row-major scales [rows, blocks] -> tiles [ceil(rows/128), ceil(blocks/4), 512], byte by byte's address."""
    rows, nb = scales.shape
    out = np.zeros((-(-rows // 128), -(-nb // 4), 512), np.uint8)
    for r in range(rows):
        for k in range(nb):
            out[r // 128, k // 4, 16 * (r % 32) + 4 * (r % 128 // 32) + k % 4] = scales[r, k]
    return out


def product_error(a, b):
    """What fp32 accumulation may lose of a @ b.T: every product is exact (2 x 2 significant bits), the tensor core
    adds blocks of them aligned to the largest (dropping what lies below 2^-23 of it, at most one part per product
    of a block) and rounds the sum once a block of 32 -- a bound of (K / 32 + 32) 2^-23 of the sum of magnitudes."""
    return (a.shape[-1] / 32 + 32) * 2.0 ** -23 * (np.abs(a) @ np.abs(b).T)


HALF = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


def experts(x, ids, w, w13, w2, out):
    """The expert layer on decoded weights w13 [E,2I,H], w2 [E,H,I]: (y, how far a kernel's y may be off).

    What a correct kernel may do otherwise is to round h at a border to the other side, since its h differs from the
    64-bit one by the accumulation error: each h whose distance to a rounding border is within that error may move by
    one grid step, and a block whose largest magnitude is that near to a power of two may take the other scale."""
    T, H = x.shape
    E, I = w13.shape[0], w2.shape[2]
    y, tol, mag = np.zeros((T, H)), np.zeros((T, H)), np.zeros((T, H))
    xq = decode(*quantize(x))
    for t in range(T):
        for k in range(ids.shape[1]):
            e = ids[t, k]
            if not 0 <= e < E:
                continue
            wg, wu, wd = w13[e, :I], w13[e, I:], w2[e]
            g, u = wg @ xq[t], wu @ xq[t]
            with np.errstate(over="ignore"):
                sig = 1 / (1 + np.exp(-g))
            h = g * sig * u
            dg = product_error(xq[t:t + 1], wg)[0]
            du = product_error(xq[t:t + 1], wu)[0]
            # |silu'| <= 1.1; the kernel's exp, division and products: 8 roundings of 2^-23
            dh = 1.1 * dg * np.abs(u) + np.abs(g * sig) * du + 8 * 2.0 ** -23 * np.abs(h) + 1.1 * dg * du
            codes, s = quantize(h)
            hq = decode(codes, s)
            unit = np.repeat(2.0 ** (s.astype(np.float64) - 127), 32)
            m = np.abs(h) / unit
            mid = (GRID[1:] + GRID[:-1]) / 2
            near = np.abs(m[:, None] - mid[None]).min(1) <= dh / unit
            step = np.where(near, np.where(m < 1.9, 0.5, np.where(m < 3.9, 1.0, 2.0)) * unit, 0.0)
            hb, db = np.abs(h).reshape(-1, 32), dh.reshape(-1, 32)
            top = hb.max(1)
            lo, hi = (hb - db).max(1), (hb + db).max(1)
            other = np.floor(np.log2(np.maximum(lo, 1e-300))) != np.floor(np.log2(np.maximum(hi, 1e-300)))
            step = np.maximum(step, np.repeat(np.where(other & (top > 0), 2.0 * 2.0 ** (s.astype(np.float64) + 1 - 127), 0.0), 32))
            p = wd @ hq
            y[t] += w[t, k] * p
            tol[t] += np.abs(w[t, k]) * (product_error(hq[None], wd)[0] + np.abs(wd) @ step)
            if out != "float32":  # parts may be kept as 16-bit integers: a step of 2^-14 of the block's power of two
                amax = np.maximum(np.abs(p).reshape(-1, 32).max(1), 1e-300)
                tol[t] += np.abs(w[t, k]) * np.repeat(2.0 ** (np.floor(np.log2(amax)) - 14), 32)
            mag[t] += np.abs(w[t, k] * p)
    # the weighted sum in fp32, then one rounding to the output type
    tol += (ids.shape[1] + 2) * 2.0 ** -24 * mag
    return y, tol + HALF[out] * (np.abs(y) + tol) + (2.0 ** -25 if out == "float16" else 0.0)
