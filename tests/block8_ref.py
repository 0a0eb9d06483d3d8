"""The 8-bit block-scaled format restated on the host in NumPy, from its definition: every code's
value by its fields, rounding by a search among all of them, the scale's exponent by trial."""
import numpy as np

BLOCK = 128


def _code_values():
    v = np.zeros(256)
    for c in range(256):
        e, f = (c >> 3) & 15, c & 7
        m = (1 + f / 8) * 2.0 ** (e - 7) if e else f / 8 * 2.0 ** -6
        v[c] = np.nan if c & 127 == 127 else (-m if c & 128 else m)
    return v


CODES = _code_values()
_POS = CODES[:127]


def round_codes(v):
    """Codes nearest to the values v (magnitude at most 448), ties to the even code; not finite: NaN."""
    v = np.asarray(v, np.float64)
    a = np.minimum(np.abs(np.nan_to_num(v, nan=0.0, posinf=0.0, neginf=0.0)), 448.0)
    hi = np.clip(np.searchsorted(_POS, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    up, down = _POS[hi] - a, a - _POS[lo]
    c = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    c = np.where(_POS[hi] == a, hi, c)
    c = np.where(np.isfinite(v), c, 127)
    return (c | np.where(np.signbit(v), 128, 0)).astype(np.uint8)


def scale_exponent(amax):
    if not amax > 0:
        return 0
    e = -117
    while amax > 448.0 * 2.0 ** e and e < 120:
        e += 1
    return e


def quantize(x, tile_rows=1):
    """(codes, exponents) of x [rows, cols]."""
    x = np.asarray(x, np.float64)
    rows, cols = x.shape
    tr = tile_rows
    codes = np.zeros(x.shape, np.uint8)
    exps = np.zeros((-(-rows // tr), -(-cols // BLOCK)), int)
    for i in range(exps.shape[0]):
        for j in range(exps.shape[1]):
            s = (slice(i * tr, (i + 1) * tr), slice(j * BLOCK, (j + 1) * BLOCK))
            mag = np.abs(x[s])
            e = scale_exponent(mag[np.isfinite(mag)].max(initial=0.0))
            exps[i, j] = e
            codes[s] = round_codes(x[s] / 2.0 ** e)
    return codes, exps


def values(codes, scales, tile_rows=1):
    """Codes times scales [rows or tiles, blocks] as float64."""
    rows, cols = codes.shape
    r = np.arange(rows) // tile_rows
    c = np.arange(cols) // BLOCK
    return CODES[codes] * np.asarray(scales, np.float64)[r][:, c]
