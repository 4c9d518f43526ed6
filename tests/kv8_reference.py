"""A plain restatement of the 8-bit paged cache in 64 bits, for the tests: formats, append,
gather and decode, on the host and one block at a time."""
import math

import numpy as np
import torch

LARGEST = {"e4m3": 448.0, "int8": 127.0}
TORCH = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def e4m3_value(code: int) -> float:
    """Sign, 4 exponent bits (bias 7), 3 mantissa bits; exponent 0: steps of 2^-9; 0x7f: NaN."""
    sign, e, m = -1.0 if code & 0x80 else 1.0, code >> 3 & 15, code & 7
    if e == 15 and m == 7:
        return math.nan
    return sign * (m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10))


E4M3 = np.array([e4m3_value(c) for c in range(256)])
_POS = E4M3[:127]  # ascending, codes 0 .. 126


def values(codes: np.ndarray, fmt: str) -> np.ndarray:
    """uint8 codes -> fp64 values."""
    return E4M3[codes] if fmt == "e4m3" else codes.view(np.int8).astype(np.float64)


def encode(x: np.ndarray, fmt: str) -> np.ndarray:
    """Nearest code of fp64 values within the format's range, ties to the even code."""
    if fmt == "int8":
        return np.rint(x).astype(np.int8).view(np.uint8)
    a = np.abs(x)
    hi = np.clip(np.searchsorted(_POS, a), 1, 126)
    lo = hi - 1
    dl, dh = a - _POS[lo], _POS[hi] - a
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    return (code | np.where(np.signbit(x), 0x80, 0)).astype(np.uint8)


def power_scale(amax: float, fmt: str) -> float:
    """Least power of two, 2^-100 at least, with amax <= largest * it."""
    e = -100
    while LARGEST[fmt] * 2.0 ** e < amax:
        e += 1
    return 2.0 ** e


def append(codes, scales, k, v, slots, fmt):
    """codes uint8 [2, nb, bs, H, D], scales fp32 [2, nb, H] (both changed), k / v fp64 [H, T, D]."""
    bs, heads = codes.shape[2], codes.shape[3]
    t = 0
    while t < len(slots):
        if slots[t] < 0 or slots[t] >= codes.shape[1] * bs:
            t += 1
            continue
        blk, a = divmod(int(slots[t]), bs)
        n = 1
        while t + n < len(slots) and slots[t + n] == slots[t] + n and a + n < bs:
            n += 1
        for plane, src in enumerate((k, v)):
            for h in range(heads):
                x = src[h, t: t + n]
                old = float(scales[plane, blk, h]) if a > 0 else 0.0
                if not np.isfinite(x).all() or not (0 <= old < math.inf):
                    scales[plane, blk, h] = math.nan
                    codes[plane, blk, a: a + n, h] = 0
                    continue
                s = max(old, power_scale(float(np.abs(x).max()), fmt))
                if a > 0 and s != old:
                    codes[plane, blk, :a, h] = encode(values(codes[plane, blk, :a, h], fmt) * (old / s), fmt)
                codes[plane, blk, a: a + n, h] = encode(x / s, fmt)
                scales[plane, blk, h] = s
        t += n


def rows(codes, scales, table, fmt, plane, t0, t1, off=0):
    """Values of tokens [t0, t1) of a table in fp64: [H, t1 - t0, D]."""
    bs = codes.shape[2]
    at = np.arange(t0, t1) - off
    blk = np.asarray(table)[at // bs]
    c = values(codes[plane, blk, at % bs], fmt)  # [T, H, D]
    return (c * scales[plane, blk].astype(np.float64)[..., None]).transpose(1, 0, 2)


def random_cache(r, nb, bs, heads, d, fmt, spread=3):
    """Random valid codes and power-of-two scales that differ by up to 2^spread."""
    if fmt == "e4m3":
        codes = r.integers(0, 127, (2, nb, bs, heads, d)).astype(np.uint8) | (r.integers(0, 2, (2, nb, bs, heads, d)) << 7).astype(np.uint8)
        low = -9
    else:
        codes = r.integers(-127, 128, (2, nb, bs, heads, d)).astype(np.int8).view(np.uint8)
        low = -7
    return codes, (2.0 ** r.integers(low, low + spread, (2, nb, heads))).astype(np.float32)


def attend(q, k, v, scale):
    """softmax(scale q k^T) v and its log-sum-exp in fp64; no keys: 0 and -inf."""
    if k.shape[0] == 0:
        return np.zeros((q.shape[0], v.shape[1])), np.full(q.shape[0], -math.inf)
    s = (q @ k.T) * scale
    m = s.max(1, keepdims=True)
    p = np.exp(s - m)
    return (p @ v) / p.sum(1, keepdims=True), (m + np.log(p.sum(1, keepdims=True)))[:, 0]


def to_device(codes, scales, fmt):
    return (torch.from_numpy(codes.copy()).cuda().view(TORCH[fmt]), torch.from_numpy(scales.copy()).cuda())


def to_host(pool, scales):
    return pool.view(torch.uint8).cpu().numpy(), scales.cpu().numpy()
