"""Log probabilities of tokens, entropy and most likely tokens against 64-bit NumPy.

Tolerances, u = 2^-24: a term exp(x - M) is off by 2^-22 (ex2.approx) and 3 u |x - M| (difference, factor, product); the sum adds at most 45 u (32 values
per accumulator, then trees), so S is off by 2^-22 + (45 + 3 D) u with D the mean of |x - M| under p, at most ln V + a little: with D <= 13 that is
5.3e-6, the error of its logarithm. A log probability adds 2 u (|x - M| + |result|); the entropy the weighted sum's error, 2 D times the same. Sure rows:
the sum of the others keeps its digits, so log p of the likely token is right to 6e-6 of itself.
"""
import numpy as np
import pytest
import torch

from oracle import rowwise_oracle as R

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"fp16": (torch.float16, np.float16), "fp32": (torch.float32, np.float32)}


def _logits(rng, rows, vocab, dtype, sigma=2.5):
    return (sigma * rng.standard_normal((rows, vocab))).astype(dtype)


def _close(got, ref, tol):
    got = got.double().cpu().numpy()
    special = ~np.isfinite(ref)
    np.testing.assert_array_equal(got[special], ref[special])
    err = np.abs(np.where(special, 0, got) - np.where(special, 0, ref))
    assert (err <= tol).all(), (float((err / tol).max()), np.unravel_index(np.argmax(err / tol), err.shape))


def _check(T, cuda, x, ids, top, view=None):
    lp, ent, tid, tlp, mean = R.token_log_probs(x, ids, top)
    t = torch.from_numpy(x).to(cuda) if view is None else view
    r = T.token_log_probs(t, torch.from_numpy(ids).to(cuda), top_k=top)
    base = 5.3e-6
    mag = lambda ref: np.where(np.isfinite(ref), np.abs(ref), 0)
    _close(r.log_probs, lp, base + 4 * U * (2 * mag(lp) + 13))
    _close(r.entropy, ent, base * (1 + 2 * mean) + 4 * U)
    if top:
        np.testing.assert_array_equal(r.top_ids.cpu().numpy(), tid)
        _close(r.top_log_probs, tlp, np.minimum(base + 4 * U * (2 * mag(tlp) + 13), np.maximum(6e-6 * mag(tlp), 1e-38) + 1e9 * (tlp < -0.5)))
    return r


# vocabularies around vectors and parts: one warp per row up to 504 halves / 252 floats (4088 / 2044 of many rows),
# then eight warps, beyond 32760 / 16380 with several parts
@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
@pytest.mark.parametrize("vocab", [1, 2, 5, 8, 31, 100, 252, 253, 500, 504, 505, 1016, 1100, 4092, 4093, 8184, 8185, 16385, 30522, 32768, 32769, 50001, 120000])
def test_log_probs(cuda, dtype, vocab):
    import tensorrt_b200 as T

    rng = np.random.default_rng(vocab)
    for rows, tokens, top in ((1, 1, 5), (3, 4, 32), (18, 2, 1)):
        x = _logits(rng, rows, vocab, TYPES[dtype][1])
        ids = rng.integers(0, vocab, size=(rows, tokens)).astype(np.int32)
        _check(T, cuda, x, ids, top)


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
@pytest.mark.parametrize("rows,vocab", [(700, 50), (650, 3000), (1300, 4001), (400, 30522), (640, 30522), (310, 70001), (250, 120000)])
def test_log_probs_many_rows(cuda, dtype, rows, vocab):
    """More rows than fit the GPU: one CTA per row, also where a row has several parts, and clusters that take several rows by turns."""
    import tensorrt_b200 as T

    rng = np.random.default_rng(rows)
    x = _logits(rng, rows, vocab, TYPES[dtype][1])
    _check(T, cuda, x, rng.integers(0, vocab, size=(rows, 1)).astype(np.int32), 10)


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
@pytest.mark.parametrize("vocab", [17, 33, 64, 130, 231, 281, 504, 1500, 3500])
def test_log_probs_most_tokens_of_short_rows(cuda, dtype, vocab):
    """As many likely tokens as there may be of rows that one warp has: random, sorted, of few different values, mostly masked."""
    import tensorrt_b200 as T

    n = TYPES[dtype][1]
    rng = np.random.default_rng(vocab)
    rows = 1300 if vocab > 252 else 40
    x = _logits(rng, rows, vocab, n)
    x[1:rows:5] = -np.sort(-x[1:rows:5], axis=1)
    x[2:rows:5] = np.round(x[2:rows:5])
    x[3:rows:5] = np.where(rng.random(x[3:rows:5].shape) < 0.95, n(-np.inf), x[3:rows:5])
    x[4:rows:10] = n(0)
    x[9:rows:10] *= n(-0.0)
    ids = rng.integers(0, vocab, size=(rows, 1)).astype(np.int32)
    for top in (12, 13, 16, 17, 32):
        _check(T, cuda, x, ids, top)


@pytest.mark.parametrize("dtype,vocab", [("fp16", 5111), ("fp16", 6640), ("fp32", 2500), ("fp32", 3320)])
def test_log_probs_warp_with_many_vectors(cuda, dtype, vocab):
    """The longest rows that one warp has, more than sixteen vectors of each lane: few candidates in all of its places, many equal ones."""
    import tensorrt_b200 as T

    n = TYPES[dtype][1]
    rng = np.random.default_rng(vocab)
    x = _logits(rng, 1800, vocab, n)
    x[np.arange(600), rng.integers(0, vocab, size=600)] = 20
    x[600:900] = np.round(x[600:900])
    x[900:1000, ::3] = -np.inf
    x[1000:1010, 4000 % vocab:] = x.max()
    ids = rng.integers(0, vocab, size=(1800, 2)).astype(np.int32)
    for top in (0, 3, 32):
        _check(T, cuda, x, ids, top)


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
@pytest.mark.parametrize("vocab", [40, 999, 5001, 30522, 70000])
def test_log_probs_special_rows(cuda, dtype, vocab):
    import tensorrt_b200 as T

    n = TYPES[dtype][1]
    info = np.finfo(n)
    rng = np.random.default_rng(vocab)
    x = _logits(rng, 24, vocab, n)
    x[0] = -np.inf                                   # nothing left
    x[1] = -np.inf
    x[1, vocab - 1] = 3                              # one token left
    x[2, vocab // 2] = np.nan
    x[3, 0] = np.inf
    x[4] = 1.5                                       # all the same: the first ids
    x[5] = info.min                                  # masks of the type's lowest value, everywhere ...
    x[6, 1:] = info.min                              # ... and everywhere but once
    x[7, :vocab // 2] = -np.inf
    x[8] = -np.inf
    x[8, ::7] = 0.25                                 # many equal values between masked ones
    x[9] = np.where(np.arange(vocab) % 2 == 0, n(-0.0), n(0.0))  # equal
    x[10] = -5
    x[10, [3, vocab - 2]] = 0.0
    x[11] = np.sort(x[11])                           # the likely ones side by side
    x[12] = np.sort(x[12])[::-1]
    x[13, vocab // 3] = 40                           # sure: 1 - p far below 2^-24
    x[14, vocab // 3] = 20
    x[15, :] = np.round(x[15].astype(np.float64))    # few values, many ties
    x[16] = info.max
    x[17] = -np.inf
    x[17, -3:] = info.min                            # lowest values left among masked ones
    x[18, vocab - 1] = -np.inf
    x[19] = 0
    x[19, 5] = 1
    ids = rng.integers(0, vocab, size=(24, 3)).astype(np.int32)
    ids[:, 1] = vocab - 1
    ids[20] = (-1, vocab, vocab + 12345)             # no such tokens
    ids[13, 0] = ids[14, 0] = vocab // 3
    ids[21, :] = 7                                   # the same token more than once
    for top in (1, 5, 32):
        r = _check(T, cuda, x, ids, top)
        lp = r.log_probs.cpu().numpy()
        assert np.isneginf(lp[20]).all() and np.isneginf(lp[0]).all() and np.isnan(lp[2:4]).all()
        assert float(r.entropy[0]) == 0 and (r.top_ids[0] == -1).all() and (r.top_ids[2:4] == -1).all()
    # sure rows keep the digits of log p
    ref = R.token_log_probs(x, ids, 1)
    for row in (13, 14):
        assert abs(lp[row, 0] - ref[0][row, 0]) <= 6e-6 * abs(ref[0][row, 0])


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
@pytest.mark.parametrize("vocab,pad,offset", [(1000, 8, 0), (1001, 0, 0), (5000, 3, 1), (30522, 6, 0), (30522, 1, 5), (70001, 0, 0)])
def test_log_probs_strides_and_alignment(cuda, dtype, vocab, pad, offset):
    """Rows that begin anywhere; what lies around them (NaN) is not theirs."""
    import tensorrt_b200 as T

    n = TYPES[dtype][1]
    rng = np.random.default_rng(vocab + pad)
    for rows in (5, 9):
        buf = np.full((rows, vocab + pad + offset), np.nan, dtype=n)
        buf[:, offset:offset + vocab] = _logits(rng, rows, vocab, n)
        view = torch.from_numpy(buf).to(cuda)[:, offset:offset + vocab]
        ids = rng.integers(0, vocab, size=(rows, 2)).astype(np.int32)
        _check(T, cuda, np.ascontiguousarray(buf[:, offset:offset + vocab]), ids, 7, view=view)


def test_log_probs_what_is_asked_for(cuda):
    import tensorrt_b200 as T

    rng = np.random.default_rng(0)
    x = torch.from_numpy(_logits(rng, 6, 3001, np.float32)).to(cuda)
    ids = torch.from_numpy(rng.integers(0, 3001, size=(6, 700)).astype(np.int32)).to(cuda)
    full = T.token_log_probs(x, ids, top_k=9)
    assert T.token_log_probs(x, ids[:, 0].contiguous()).log_probs.shape == (6,)
    assert torch.equal(T.token_log_probs(x, ids[:, 0].contiguous()).log_probs, full.log_probs[:, 0])
    only = T.token_log_probs(x)
    assert only.log_probs is None and only.top_ids is None and torch.equal(only.entropy, full.entropy)
    alone = T.token_log_probs(x, top_k=9)
    assert torch.equal(alone.top_ids, full.top_ids) and torch.equal(alone.top_log_probs, full.top_log_probs)
    ref = R.token_log_probs(x.cpu().numpy(), ids.cpu().numpy(), 9)
    np.testing.assert_allclose(full.log_probs.cpu().numpy(), ref[0], atol=3e-5, rtol=0)
    empty = T.token_log_probs(x[:0], ids[:0], top_k=2)
    assert empty.log_probs.shape == (0, 700) and empty.top_ids.shape == (0, 2)
    none = T.token_log_probs(x, ids[:, :0].contiguous(), top_k=1)
    assert none.log_probs.shape == (6, 0) and torch.equal(none.top_ids[:, 0], full.top_ids[:, 0])


@pytest.mark.parametrize("rows,vocab", [(2, 30522), (500, 30522), (40, 900)])
def test_log_probs_same_bits_every_time(cuda, rows, vocab):
    """The order in which candidates are listed does not matter; a side stream and a replayed graph give the same bits."""
    import tensorrt_b200 as T

    rng = np.random.default_rng(rows)
    x = torch.from_numpy(np.round(_logits(rng, rows, vocab, np.float16))).to(cuda)
    ids = torch.from_numpy(rng.integers(0, vocab, size=(rows, 1)).astype(np.int32)).to(cuda)
    ref = T.token_log_probs(x, ids, top_k=20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        others = [T.token_log_probs(x, ids, top_k=20) for _ in range(10)]
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = T.token_log_probs(x, ids, top_k=20)
    graph.replay()
    torch.cuda.synchronize()
    for r in others + [captured]:
        assert all(torch.equal(a, b) for a, b in zip(ref, r))
