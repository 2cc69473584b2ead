"""64-bit oracles of the 8-bit store's format and of the teacher's loss, in numpy."""
import numpy as np

BLOCK = 128


def quantise(x):
    """(values of the codes before the scale, scale bytes) of rows of x (any float array), from the definition: the smallest power of two
    2^e, e >= -126, with amax <= 448 * 2^e; the multiple of the e4m3 spacing nearest to x / 2^e, ties to even; non-finite values NaN."""
    x = np.asarray(x, np.float64)
    n, dim = x.shape
    codes = np.zeros((n, dim))
    bytes_ = np.zeros((n, -(-dim // BLOCK)), np.int64)
    for b, lo in enumerate(range(0, dim, BLOCK)):
        y = x[:, lo:lo + BLOCK]
        fine = np.isfinite(y)
        amax = np.where(fine, np.abs(y), 0.0).max(1) if y.size else np.zeros(n)
        part, power = np.frexp(amax / 448.0)
        power = np.where(part == 0.5, power - 1, power)
        power = np.where(amax == 0, -126, np.maximum(power, -126))
        z = np.where(fine, y, 0.0) * np.ldexp(1.0, -power)[:, None]
        spacing = np.ldexp(1.0, np.maximum(np.frexp(z)[1] - 1, -6) - 3)
        codes[:, lo:lo + BLOCK] = np.where(fine, np.rint(z / spacing) * spacing, np.nan)
        bytes_[:, b] = power + 127
    return codes, bytes_


def values(x):
    codes, bytes_ = quantise(x)
    scale = np.ldexp(1.0, bytes_ - 127).repeat(BLOCK, 1)[:, :codes.shape[1]]
    return codes * scale


def teacher(logits, idx, vals, kind="proba", temperature=1.0, weight=None):
    """(loss, stats, gradient of loss.sum()) of the definition in 64 bits; idx < 0 is an empty place."""
    s = np.asarray(logits, np.float64)
    rows, cols = s.shape
    w = np.ones(rows) if weight is None else np.asarray(weight, np.float64)
    loss, grad = np.zeros(rows), np.zeros((rows, cols))
    stats = np.tile([-np.inf, 0.0], (rows, 1))
    with np.errstate(all="ignore"):
        for r in range(rows):
            if w[r] == 0 or np.all(s[r] == -np.inf):
                continue
            if np.isnan(s[r]).any() or (s[r] == np.inf).any() or (idx[r] >= cols).any():
                loss[r], grad[r] = np.nan, np.nan
                stats[r] = np.nan
                continue
            m = s[r].max()
            lnsum = np.log(np.exp((s[r] - m) / temperature).sum())
            stats[r] = m, lnsum
            lnq = (s[r] - m) / temperature - lnsum
            at = idx[r] >= 0
            p = np.zeros(len(at))
            if kind == "proba":
                p[at] = vals[r][at]
            elif at.any() and np.max(vals[r][at]) > -np.inf:
                t = np.asarray(vals[r][at], np.float64)
                e = np.exp((t - t.max()) / temperature)
                p[at] = e / e.sum()
            d = np.exp(lnq) * p.sum()
            for j in np.nonzero(at)[0]:
                if p[j] != 0:
                    loss[r] += w[r] * p[j] * (np.log(p[j]) - lnq[idx[r][j]])
                d[idx[r][j]] -= p[j]
            grad[r] = d * w[r] / temperature
    return loss, stats, grad
