"""Caches with a scale per block and head, in plain 64-bit form, for the tests."""

import numpy as np
import torch

MOST = 240.0


def code_values():
    """What the 256 codes stand for (4 exponent bits of bias 7, exponent 15: inf and NaN), float64."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, (c & 7).astype(np.float64)
    size = np.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * 2.0 ** (e - 7.0))
    size = np.where(e == 15, np.where(m == 0, np.inf, np.nan), size)
    return np.where(c >= 128, -size, size)


VALUES = code_values()


def encode(q):
    """Codes of float64 values of at most 240 where finite: to nearest even; inf 0x78, NaN 0x79, each with its sign."""
    q = np.asarray(q, np.float64)
    a = np.abs(np.where(np.isfinite(q), q, 0.0))
    e = np.floor(np.log2(np.maximum(a, 2.0 ** -6)))
    step = 2.0 ** (e - 3)
    r = np.rint(a / step) * step  # (the quotient is exact: a power of two divides)
    assert (r <= MOST).all()
    e = np.floor(np.log2(np.maximum(r, 2.0 ** -6)))
    code = np.where(r < 2.0 ** -6, np.rint(r * 512), (e + 7) * 8 + np.rint((r / 2.0 ** e - 1) * 8)).astype(np.int64)
    code = np.where(np.isinf(q), 0x78, np.where(np.isnan(q), 0x79, code))
    return (code | np.where(np.signbit(q), 0x80, 0)).astype(np.uint8)


def scale_for(a):
    """The least power of two, at least 2^-126, that brings a (float64) to at most 240."""
    s = 2.0 ** -126
    while a / s > MOST:
        s *= 2.0
    return s


def finite_max(x):
    x = np.abs(x[np.isfinite(x)])
    return x.max() if x.size else 0.0


def store(key, value, kc, vc, scales, tables, ctx, start):
    """The append on host copies: key, value float32 [N, H, D]; kc, vc uint8; scales float32.  Updated in place."""
    nb, H, _, bs, _ = kc.shape
    D = vc.shape[2]
    N = key.shape[0]
    for s in range(len(ctx)):
        a, b = (min(max(int(x), 0), N) for x in (start[s], start[s + 1]))
        c, n = int(np.uint32(ctx[s])), b - a
        if n <= 0 or c == 0 or c > tables.shape[1] * bs:
            continue
        lo = max(c - n, 0)
        for j in range(lo // bs, -(-c // bs)):
            block = int(tables[s, j])
            if not 0 <= block < nb:
                continue
            o0, o1 = max(lo, j * bs) - j * bs, min(c, (j + 1) * bs) - j * bs
            rows = slice(a + j * bs + o0 - (c - n), a + j * bs + o1 - (c - n))
            for h in range(H):
                for which, src in ((0, key), (1, value)):
                    x = src[rows, h].astype(np.float64)  # [tokens, D]
                    scale = scale_for(finite_max(x))
                    old = scales[block, h, which]
                    view = (kc[block, h].transpose(1, 0, 2).reshape(bs, D) if which == 0 else vc[block, h].T).copy()
                    if o0 > 0 and float(old) >= scale:
                        scale = float(old)
                    elif o0 > 0:
                        was = VALUES[view[:o0]].astype(np.float32) * old  # (one float32 rounding, as the kernel's)
                        again = encode(np.where(np.isfinite(was), was.astype(np.float64) / scale, 0.0))
                        view[:o0] = np.where(np.isfinite(was), again, view[:o0])
                    with np.errstate(invalid="ignore"):
                        q = src[rows, h].astype(np.float32) / np.float32(scale)
                    view[o0:o1] = encode(q)
                    if which == 0:
                        kc[block, h] = view.reshape(bs, D // 16, 16).transpose(1, 0, 2)
                    else:
                        vc[block, h] = view.T
                    scales[block, h, which] = scale


def rows_of(kc, vc, scales, table, lo, hi):
    """Keys and values of tokens [lo, hi): float64 tensors [T, H, D] on the caches' device; all caches tensors."""
    bs = kc.shape[3]
    values = torch.from_numpy(VALUES).to(kc.device)
    pos = torch.arange(lo, hi, device=kc.device)
    block = table.long()[pos // bs]
    s = scales.double()[block]
    k = values[kc[block, :, :, pos % bs, :].long()].flatten(2) * s[:, :, :1]
    v = values[vc[block, :, :, pos % bs].long()] * s[:, :, 1:]
    return k, v


def attend(q, k, v, first, scale, window=0, sinks=0):
    """q [n, Hq, D] at positions first, first + 1, ...; k, v [T, H, D].  Returns the output and the most that a
    kernel may be off, both float64 [n, Hq, D].

    The bound, with u half a step of the type: each weight is rounded to the type (u of it) before the second
    product, the output once (u of it).  A score's float32 sum of D products is off by at most (D + 8) 2^-24 of the
    sum of their sizes (8: products with the scales and the reference point), in numerator and denominator, and
    2^-20 covers exponentials, float32 sums and the division.  A float16 weight below its normal range (2^-14, where
    the largest is at least 2^11) is off by 2^-25: 2^-36 of the largest for each token.  An output below the type's
    normal range is a multiple of its smallest subnormal, eps * smallest_normal: half of that."""
    n, Hq, D = q.shape
    T, H = k.shape[:2]
    u = torch.finfo(q.dtype).eps / 2
    least = u * torch.finfo(q.dtype).smallest_normal
    pos = torch.arange(T, device=q.device)
    mine = torch.arange(first, first + n, device=q.device)[:, None]
    sees = pos <= mine
    if window:
        sees &= (pos > mine - window) | (pos < sinks)
    some = sees.any(1)
    out = torch.zeros((n, Hq, D), dtype=torch.float64, device=q.device)
    off = torch.zeros_like(out)
    for h in range(Hq):
        kh, vh = k[:, h // (Hq // H)].contiguous(), v[:, h // (Hq // H)].contiguous()
        qh = q[:, h].double()
        s = (qh @ kh.t().contiguous()) * scale
        p = torch.softmax(s.masked_fill(~sees, float("-inf")), -1)
        p = torch.where(some[:, None], p, 0.0)
        # (What no row sees takes no part, whatever it holds.)
        seen = sees.any(0)[:, None]
        size = (qh.abs() @ torch.where(seen, kh, 0.0).abs().t().contiguous()).mul(abs(scale))
        e32 = 2 * (D + 8) * 2.0 ** -24 * torch.where(sees, size, 0.0).amax(1, keepdim=True) + 2.0 ** -20
        vh = torch.where(seen, vh, 0.0)
        o = p @ vh
        out[:, h] = o
        off[:, h] = (u + e32) * (p @ vh.abs()) + (u + e32) * o.abs() + T * 2.0 ** -36 * vh.abs().amax() + least
    return out, off
