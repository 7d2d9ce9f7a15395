"""Plain 64-bit form of the microscaled 4-bit calls, from their definition: loops over
blocks and grid values where they are clearest, numpy otherwise.  CPU only."""
import numpy as np

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)


def padded(k):
    return -(-k // 128) * 128


def scale_of(top, rule):
    """Scale byte of a block whose largest magnitude is top (a Python float)."""
    if not np.isfinite(top):
        return 255
    if top == 0:
        return 0
    if rule == "fit":
        e = max(-127, int(np.floor(np.log2(top))) - 5)      # below every power that holds top
        while top > 6 * 2.0 ** e:
            e += 1
    else:
        e = max(-127, int(np.floor(np.log2(top))) - 2)
        assert e == -127 or 4 * 2.0 ** e <= top < 8 * 2.0 ** e
    return e + 127


def quantize(x, rule="fit", rand=None):
    """(codes, scales) of the rows of x (float64 holding the input's values exactly)."""
    x = np.asarray(x, dtype=np.float64)
    rows, k = x.shape
    kp = padded(k)
    v = np.zeros((rows, kp))
    v[:, :k] = x
    r = np.zeros((rows, kp), dtype=np.int64)
    if rand is not None:
        r[:, :k] = rand
    v, r = v.reshape(rows, -1, 32), r.reshape(rows, -1, 32)
    with np.errstate(invalid="ignore"):
        top = np.abs(v).max(-1)
    scales = np.array([[scale_of(float(t), rule) for t in row] for row in top], dtype=np.uint8).reshape(rows, -1)
    p = 2.0 ** (scales.astype(np.float64) - 127)[..., None]
    nan = (scales == 255)[..., None]
    mag = np.where(nan, 0, np.minimum(np.abs(np.where(nan, 0, v)) / p, 6))
    above = np.searchsorted(GRID, mag)              # the first grid value >= mag
    hi = GRID[above]
    below = np.where(hi > mag, above - 1, above)
    lo = GRID[below]
    if rand is None:
        up = (hi - mag < mag - lo) | ((hi - mag == mag - lo) & (above % 2 == 0))
    else:
        share = np.where(hi > lo, (mag - lo) / np.where(hi > lo, hi - lo, 1), 0)
        up = share + (r + 0.5) / 256 >= 1
    code = np.where(up, above, below) + 8 * np.signbit(v)
    code = np.where(nan, 0, code).astype(np.uint8).reshape(rows, kp)
    return code[:, 0::2] + 16 * code[:, 1::2], scales


def values(codes, scales, k):
    """Blocks to 64-bit values (NaN for scale 255)."""
    codes, scales = np.asarray(codes), np.asarray(scales)
    q = np.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1)
    v = GRID[q & 7] * np.where(q >= 8, -1.0, 1.0)
    p = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return (v * np.repeat(p, 32, axis=1))[:, :k]


def history(codes, scales, table, length, channels):
    """(length, channels) of one sequence; codes (pages, page, ...)."""
    pages, page = codes.shape[:2]
    n = max(0, min(int(length), len(table) * page))
    out = np.zeros((n, channels))
    for t in range(n):
        pg = int(table[t // page])
        if 0 <= pg < pages:
            out[t] = values(codes[pg, t % page][None], scales[pg, t % page][None], channels)[0]
    return out


def conv_step(hist, taps):
    """Value of the causal convolution at the last token of hist (n, channels), and the sum of
    the terms' magnitudes."""
    n = min(len(hist), len(taps))
    terms = np.asarray(taps[:n], dtype=np.float64) * hist[::-1][:n]
    return terms.sum(0), np.abs(terms).sum(0)


def within(got, want, magnitudes, terms, dtype):
    """Whether every element of the tensor `got` is one that a sum of `terms` fp32 terms, rounded to
    got's type once, can give for the exact value `want`: each term is added at most `terms` times
    at 2^-24 of the sum of the magnitudes (and the smallest normal number, below which a
    sum may be anything that small), and rounding is monotonic, so the result lies between
    the rounded ends of that interval."""
    import torch
    err = (terms + 2) * 2.0 ** -24 * magnitudes + 2.0 ** -126
    lo, hi = (torch.from_numpy(np.asarray(want + d, dtype=np.float64)).to(dtype).double().numpy() for d in (-err, err))
    got = got.double().cpu().numpy()
    return bool(np.all((got >= lo) & (got <= hi)))
