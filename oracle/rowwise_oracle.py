"""Row-wise INT8 and the answers of a language-model head in 64 bits (test infrastructure only)."""
import numpy as np


def quantize_rows(x):
    """(q, scales): scale = max|row| / 127 as the FP32 number, q = 127 x / max|row| to the nearest whole number, halves to even. Rows of zeros:
    0, 0; rows with NaN or infinity: q 0, scale NaN. The quotient in 64 bits rounds like the exact one: it is a fraction of 31-bit over
    24-bit whole numbers, never nearer to a half than 2^-25 unless it is one."""
    x = np.asarray(x, dtype=np.float64)
    amax = np.abs(x).max(axis=-1, keepdims=True)
    good = np.isfinite(amax)
    with np.errstate(invalid="ignore", divide="ignore"):
        q = np.where(good & (amax > 0), np.rint(127.0 * x / amax), 0.0)
        scales = np.where(good, amax.astype(np.float32) / np.float32(127), np.float32("nan"))
    return q.astype(np.int8), scales[..., 0].astype(np.float32)


def gelu(x):
    from scipy.special import erfc

    return 0.5 * x * erfc(-x / np.sqrt(2.0))


def fc_rowwise(a, a_scales, wt, wt_scales, bias=None, activation=0):
    """(value before the activation, result, sum of the magnitudes of its two terms)."""
    acc = np.asarray(a, np.float64) @ np.asarray(wt, np.float64).T  # whole numbers below 2^53: exact
    prod = acc * np.asarray(a_scales, np.float64)[:, None] * np.asarray(wt_scales, np.float64)[None, :]
    b = 0.0 if bias is None else np.asarray(bias, np.float64)[None, :]
    v = prod + b
    return v, gelu(v) if activation else v, np.abs(prod) + np.abs(b)


def layer_norm(x, skip, gamma, beta, bias, eps):
    v = np.asarray(x, np.float64) + (0.0 if skip is None else np.asarray(skip, np.float64)) + (0.0 if bias is None else np.asarray(bias, np.float64))
    v = v - v.mean(axis=-1, keepdims=True)
    return v / np.sqrt((v * v).mean(axis=-1, keepdims=True) + eps) * np.asarray(gamma, np.float64) + np.asarray(beta, np.float64)


def token_log_probs(logits, ids, top_k):
    """(log probs of ids, entropy, top ids, top log probs, mean of |x - max| under p) row by row."""
    x = np.asarray(logits, np.float64)
    rows, vocab = x.shape
    lp = np.full(ids.shape, -np.inf)
    ent = np.zeros(rows)
    tid = np.full((rows, top_k), -1, dtype=np.int32)
    tlp = np.full((rows, top_k), -np.inf)
    mean = np.zeros(rows)
    for r in range(rows):
        v = x[r]
        if np.isnan(v).any() or np.isposinf(v).any():
            lp[r], ent[r], tlp[r] = np.nan, np.nan, np.nan
            continue
        if np.isneginf(v).all():
            continue
        m = v.max()
        d = v - m
        e = np.exp(d)
        others = e[d < 0].sum()
        count = (d == 0).sum()
        lse = np.log(count) + np.log1p(others / count)
        with np.errstate(invalid="ignore"):
            w = np.where(e > 0, e * d, 0.0).sum() / (count + others)
        ent[r] = lse - w
        mean[r] = -w
        for j, i in enumerate(ids[r]):
            if 0 <= i < vocab:
                lp[r, j] = d[i] - lse
        best = np.argsort(-v, kind="stable")[:top_k]
        best = best[v[best] > -np.inf]
        tid[r, :len(best)] = best
        tlp[r, :len(best)] = d[best] - lse
    return lp, ent, tid, tlp, mean
