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


def encoder(p, ids, seg, cu, S):
    """The encoder with row-wise INT8 projections in 64 bits, every stored tensor rounded to FP16: weights with a scale per output channel, each
    projection's input with a scale per token (of the LayerNorm's unrounded result where a LayerNorm precedes it)."""
    from oracle import bert_oracle as O

    h = lambda t: t.astype(np.float16).astype(np.float64)
    B = len(cu) - 1
    x, _ = O.emb_layer_norm_var_seqlen(ids, seg, cu, p.word_emb, p.pos_emb, p.tok_emb, p.emb_gamma, p.emb_beta)
    x = h(x)
    q = quantize_rows(x)
    for lp in p.layers:
        weights = {n: quantize_rows(np.asarray(getattr(lp, n), np.float32).T) for n in ("w_qkv", "w_out", "w_ffn1", "w_ffn2")}
        product = lambda a, name, bias=None, act=0: h(fc_rowwise(a[0], a[1], *weights[name], bias, act)[1])
        ctx = h(O.mha(product(q, "w_qkv", lp.b_qkv), B, S, p.heads, x.shape[1] // p.heads, cu=cu))
        y = layer_norm(product(quantize_rows(ctx), "w_out"), x, lp.ln1_gamma, lp.ln1_beta, lp.b_out, 0.0)
        h1 = h(y)
        f1 = product(quantize_rows(y), "w_ffn1", lp.b_ffn1, 1)
        y = layer_norm(product(quantize_rows(f1), "w_ffn2"), h1, lp.ln2_gamma, lp.ln2_beta, lp.b_ffn2, 0.0)
        x, q = h(y), quantize_rows(y)
    return x
