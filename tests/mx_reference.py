"""Microscaled operands restated in 64 bits (numpy / torch CPU), from the definition of the formats."""
import numpy as np
import torch

E4M3, E5M2, E2M3, E2M1 = 0, 1, 3, 4
FORMATS = {E4M3: (8, 3, 7), E5M2: (8, 2, 15), E2M3: (6, 3, 1), E2M1: (4, 1, 1)}   # width, mantissa bits, bias
HAS_NAN = {E4M3: lambda c: (c & 0x7F) == 0x7F, E5M2: lambda c: (c & 0x7F) > 0x7C}


def decode_codes(c, fmt):
    """Unpacked codes (numpy integers) to float64."""
    width, mant, bias = FORMATS[fmt]
    c = c.astype(np.int64)
    sign = np.where((c >> (width - 1)) & 1, -1.0, 1.0)
    e = (c & ((1 << (width - 1)) - 1)) >> mant
    f = (c & ((1 << mant) - 1)) / float(1 << mant)
    v = sign * np.where(e > 0, 1.0 + f, f) * 2.0 ** (np.maximum(e, 1) - bias)
    if fmt == E5M2:
        v = np.where((c & 0x7F) == 0x7C, sign * np.inf, v)
    if fmt in HAS_NAN:
        v = np.where(HAS_NAN[fmt](c), np.nan, v)
    return v


def unpack4(p):
    return np.stack((p & 15, p >> 4), -1).reshape(p.shape[0], 2 * p.shape[1])


def pack4(c):
    return (c[:, 0::2] | (c[:, 1::2] << 4)).astype(np.uint8)


def decode(payload, scales, fmt, group=32):
    """float64 values of an MX matrix (torch uint8 tensors on any device)."""
    p, s = payload.cpu().numpy(), scales.cpu().numpy().astype(np.int64)
    v = decode_codes(unpack4(p) if fmt == E2M1 else p, fmt)
    k = np.where(s == 255, np.nan, 2.0 ** (s - 127.0))
    with np.errstate(invalid="ignore"):
        return torch.from_numpy(v * np.repeat(k, group, axis=1))


def quantize_fp4(x):
    """(payload, scales) of a float64 matrix holding the input's values."""
    x = np.asarray(x, np.float64)
    g = x.reshape(x.shape[0], -1, 32)
    with np.errstate(invalid="ignore", over="ignore"):
        finite = np.isfinite(g).all(2)
        amax = np.abs(np.where(np.isfinite(g), g, 0.0)).max(2)
    m, e = np.frexp(np.where(amax > 0, amax, 1.0))           # m in [1/2, 1)
    s = np.where(amax > 0, np.clip(e - 1 - 2 + (2 * m > 1.5) + 127, 0, 254), 127)
    s = np.where(finite, s, 255)
    q = np.where(finite[:, :, None], g, 0.0) * 2.0 ** (127.0 - np.where(finite, s, 127))[:, :, None]
    a = np.abs(q)
    grid = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
    hi = np.clip(np.searchsorted(grid, a), 0, 7)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - grid[lo], grid[hi] - a
    c = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    c = c + 8 * np.signbit(q)
    c = np.where(finite[:, :, None], c, 0)
    return torch.from_numpy(pack4(c.reshape(x.shape).astype(np.uint8))), torch.from_numpy(s.astype(np.uint8))


def random_codes(rows, cols, fmt, seed, lo=118, hi=130):
    """Every finite code with equal chance, scale bytes between the two."""
    g = torch.Generator().manual_seed(seed)
    width = FORMATS[fmt][0]
    c = torch.randint(0, 1 << width, (rows, cols), generator=g).numpy().astype(np.uint8)
    if fmt == E4M3:
        c = np.where((c & 0x7F) == 0x7F, 0, c)
    if fmt == E5M2:
        c = np.where((c & 0x7F) >= 0x70, c & 0x8F, c)        # leave out the eight largest binades: products stay in range
    s = torch.randint(lo, hi, (rows, cols // 32), generator=g, dtype=torch.uint8)
    return torch.from_numpy(pack4(c) if fmt == E2M1 else c.astype(np.uint8)), s
