"""Row-wise INT8 and log probabilities where the documentation promises more than the sizes in use show."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"fp16": (torch.float16, np.float16), "fp32": (torch.float32, np.float32)}


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
@pytest.mark.parametrize("ld", [8, 64, 248, 256, 520, 768, 1024, 1528, 2048, 4096, 8192])
@pytest.mark.parametrize("biased", [False, True])
def test_skip_layer_norm_quantize_rows_at_any_address(cuda, dtype, ld, biased):
    """Where the INT8 rows are written changes no bit: y is that of skip_layer_norm, rows and scales those of any other place; the bytes around them stay."""
    import tensorrt_b200 as T

    t, _ = TYPES[dtype]
    gen = torch.Generator(device=cuda).manual_seed(ld)
    rnd = lambda *s: torch.randn(s, device=cuda, generator=gen).to(t)
    eps = 0.0 if dtype == "fp16" else float(np.finfo(np.float32).eps)
    for rows in (1, 45, 1500):
        x, s, g, b, bi = rnd(rows, ld), rnd(rows, ld), rnd(ld), rnd(ld), rnd(ld) if biased else None
        want = T.skip_layer_norm(x, s, g, b, bi)
        y0, q0, s0 = T.skip_layer_norm_quantize(x, s, g, b, bi, eps=eps)
        assert torch.equal(y0, want)
        for offset in (1, 2, 4, 7):
            y, q, scales = torch.empty_like(x), torch.full((rows * ld + 16,), 99, dtype=torch.int8, device=cuda), torch.empty(rows, device=cuda)
            assert T._lib.lib.bert_b200_skip_layer_norm_quantize(
                torch.cuda.current_stream().cuda_stream, 1 if dtype == "fp16" else 0, ld, rows * ld, x.data_ptr(), s.data_ptr(), b.data_ptr(), g.data_ptr(), y.data_ptr(),
                q.data_ptr() + offset, scales.data_ptr(), None if bi is None else bi.data_ptr(), eps) == 0
            assert torch.equal(y, want), offset
            assert torch.equal(q[offset:offset + rows * ld].view(rows, ld), q0) and torch.equal(scales, s0)
            assert (q[:offset] == 99).all() and (q[offset + rows * ld:] == 99).all()


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
@pytest.mark.parametrize("rows", [1, 99, 101, 102, 201, 203, 204])
@pytest.mark.parametrize("top", [0, 5, 32])
def test_log_probs_of_rows_that_share_their_ctas_with_none(cuda, dtype, rows, top):
    """Four or two CTAs for each row, up to as many rows as find places for them, and one beyond: what makes a row special lies in the share of any of them."""
    import tensorrt_b200 as T
    from oracle import rowwise_oracle as R
    from tests.test_log_probs_gpu import _check

    n = TYPES[dtype][1]
    vocab = 60001 if dtype == "fp32" else 120001
    rng = np.random.default_rng(rows)
    base = (2.5 * rng.standard_normal((13, vocab))).astype(n)
    quarter = vocab // 4
    for i in range(4):
        base[i, i * quarter:(i + 1) * quarter] = -np.inf              # nothing left in one share
        base[4 + i] = -np.inf
        base[4 + i, i * quarter + 5:i * quarter + 9] = n(1.5)         # all that is left in one share
    base[8, 3 * quarter + 7] = np.nan
    base[9, quarter + 7] = np.inf
    base[10, ::quarter] = 30                                          # the likely ones in different shares
    base[11] = 0
    x = base[np.arange(rows) % 13]
    ids = rng.integers(0, vocab, size=(rows, 2)).astype(np.int32)
    if rows <= 102:
        _check(T, cuda, x, ids, top)
        return
    # many rows: each as alone
    t, i = torch.from_numpy(x).to(cuda), torch.from_numpy(ids).to(cuda)
    got = T.token_log_probs(t, i, top_k=top)
    ref = R.token_log_probs(x[:13], ids[:13], max(top, 1))
    for r in range(rows):
        k = r % 13
        if top:
            assert (got.top_ids[r].cpu().numpy() == ref[2][k]).all(), r
        e = float(got.entropy[r])
        assert (np.isnan(e) and np.isnan(ref[1][k])) or abs(e - ref[1][k]) <= 5.3e-6 * (1 + 2 * ref[4][k]) + 2.0 ** -22, r


@pytest.mark.parametrize("dtype,vocab", [("fp16", v) for v in (497, 504, 505, 528, 560, 600, 608, 616, 640)] + [("fp32", v) for v in (249, 252, 253, 272, 288, 300, 304, 308, 320)])
@pytest.mark.parametrize("rows", [1, 60, 460])
def test_log_probs_rows_of_few_vectors_and_many_likely_tokens(cuda, dtype, vocab, rows):
    """Rows with about as many vectors as there are groups of threads that bound the likely tokens: some groups are empty, the list may overflow."""
    import tensorrt_b200 as T
    from tests.test_log_probs_gpu import _check

    n = TYPES[dtype][1]
    rng = np.random.default_rng(vocab + rows)
    x = (2.5 * rng.standard_normal((rows, vocab))).astype(n)
    x[1:rows:4] = np.round(x[1:rows:4])
    x[2:rows:4] = np.where(rng.random(x[2:rows:4].shape) < 0.9, n(-np.inf), x[2:rows:4])
    ids = rng.integers(0, vocab, size=(rows, 1)).astype(np.int32)
    for top in (13, 16, 17, 18, 20, 21):
        _check(T, cuda, x, ids, top)


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
@pytest.mark.parametrize("vocab", [300, 2000, 4001, 30522])
def test_log_probs_masks_of_the_lowest_value(cuda, dtype, vocab):
    """Masked by the type's lowest value instead of -infinity, with fewer tokens left than are asked for: masked ones follow, lowest ids first."""
    import tensorrt_b200 as T
    from tests.test_log_probs_gpu import _check

    n = TYPES[dtype][1]
    rng = np.random.default_rng(vocab)
    x = np.full((12, vocab), np.finfo(n).min, dtype=n)
    for r in range(12):
        x[r, rng.choice(vocab, size=r % 6, replace=False)] = rng.standard_normal(r % 6)
    ids = rng.integers(0, vocab, size=(12, 2)).astype(np.int32)
    for top in (0, 1, 5, 20, 32):
        _check(T, cuda, x, ids, top)


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
@pytest.mark.parametrize("tokens", [1, 31, 32, 33, 64, 65, 160, 161, 5000])
def test_log_probs_of_any_number_of_tokens(cuda, dtype, tokens):
    import tensorrt_b200 as T
    from tests.test_log_probs_gpu import _check

    rng = np.random.default_rng(tokens)
    for rows, vocab in ((3, 90), (2, 5001), (1, 70001)):
        x = (2.5 * rng.standard_normal((rows, vocab))).astype(TYPES[dtype][1])
        _check(T, cuda, x, rng.integers(-2, vocab + 2, size=(rows, tokens)).astype(np.int32), 3)


def test_log_probs_of_the_longest_rows(cuda):
    """2^24 values; against 64-bit sums on the device: FP32 terms within 2^-22 + 3 u |x - M|, summed in runs of at most 2^24 / 1024 values and trees."""
    import tensorrt_b200 as T

    g = torch.Generator(device=cuda).manual_seed(1)
    for dtype in (torch.float16, torch.float32):
        x = (2 * torch.randn((2, 2 ** 24), device=cuda, generator=g)).to(dtype)
        x[1, -1] = 14
        ids = torch.tensor([[0, 2 ** 24 - 1, 2 ** 24], [5, 2 ** 24 - 1, -1]], dtype=torch.int32, device=cuda)
        r = T.token_log_probs(x, ids, top_k=5)
        lp = torch.log_softmax(x.double(), dim=1)
        want = torch.gather(lp, 1, ids.long().clamp(0, 2 ** 24 - 1))
        # 64 values per accumulator of a part (32 of each of two sums), trees over a CTA's threads, then at most 256 parts one after the other: 400 u at most
        tol = 2.0 ** -22 + (400 + 3 * 20 + 2 * 30) * 2.0 ** -24
        assert ((r.log_probs[:, :2].double() - want[:, :2]).abs() <= tol).all() and torch.isneginf(r.log_probs[:, 2]).all()
        v, i = torch.topk(x.double() - torch.arange(2 ** 24, device=cuda) * 1e-12, 5, dim=1)  # of equal ones the lower id first
        assert torch.equal(r.top_ids.long(), i)
        ent = -(lp.exp() * lp).sum(1)
        assert ((r.entropy.double() - ent).abs() <= tol * (1 + 2 * 30)).all()


def test_offsets_that_pass_32_bits(cuda):
    """Rows that lie more than 2^31 values, and bytes, behind the first: the answers of the same rows alone."""
    import tensorrt_b200 as T

    g = torch.Generator(device=cuda).manual_seed(2)
    rnd = lambda *s: torch.randn(s, device=cuda, generator=g)
    for dtype, stride in ((torch.float16, 2 ** 30 + 8), (torch.float16, 2 ** 30 + 3), (torch.float32, 2 ** 30 + 1)):
        buf = torch.empty(3 * stride + 1000, dtype=dtype, device=cuda)
        for width in (1000, 999):
            rows = buf.as_strided((4, width), (stride, 1))
            rows.copy_(rnd(4, width))
            alone = rows.contiguous()
            assert all(torch.equal(a, b) for a, b in zip(T.quantize_rows(rows), T.quantize_rows(alone)))
            ids = torch.tensor([[3], [998], [0], [500]], dtype=torch.int32, device=cuda)
            # each row alone where it lies: its values are dealt over threads by their place in 16-byte vectors, so a copy that begins at another
            # place in a vector may be summed in another order
            got, each = T.token_log_probs(rows, ids, 7), [T.token_log_probs(rows[r:r + 1], ids[r:r + 1], 7) for r in range(4)]
            assert all(torch.equal(a, torch.cat([e[i] for e in each])) for i, a in enumerate(got))
        del buf, rows
    # operands and results of the product
    stride = 2 ** 30 + 16
    a8 = torch.zeros(2 * stride + 256, dtype=torch.int8, device=cuda).as_strided((3, 200), (stride, 1))
    w8 = torch.zeros(2 * stride + 256, dtype=torch.int8, device=cuda).as_strided((3, 200), (stride, 1))
    for t in (a8, w8):
        t.copy_(torch.randint(-127, 128, (3, 200), device=cuda, generator=g).to(torch.int8))
    s = rnd(3).abs()
    out = torch.empty(2 * stride + 64, dtype=torch.float32, device=cuda).as_strided((3, 3), (stride, 1))
    pad = lambda t: torch.nn.functional.pad(t, (0, 8))[:, :200]
    assert torch.equal(T.fc_rowwise(a8, s, w8, s, out_dtype=torch.float32, out=out), T.fc_rowwise(pad(a8), s, pad(w8), s, out_dtype=torch.float32))
    del a8, w8, out
    # and where there are that many rows
    n = 2 ** 21 + 100
    x = torch.empty((n, 1024), dtype=torch.float16, device=cuda).normal_(generator=g)
    gamma, beta = (1 + 0.1 * rnd(1024)).half(), rnd(1024).half()
    last = slice(n - 70, n)
    whole, part = T.skip_layer_norm_quantize(x, x, gamma, beta), T.skip_layer_norm_quantize(x[last], x[last], gamma, beta)
    assert all(torch.equal(a[last], b) for a, b in zip(whole, part))
    del whole
    odd = x.view(-1)[:(n - 2) * 1023].view(n - 2, 1023)
    last = slice(n - 72, n - 2)
    whole, part = T.skip_layer_norm_quantize(odd, None, gamma[:1023], beta[:1023], eps=1e-6), T.skip_layer_norm_quantize(odd[last].clone(), None, gamma[:1023], beta[:1023], eps=1e-6)
    assert all(torch.equal(a[last], b) for a, b in zip(whole, part))
    del whole
    whole, part = T.quantize_rows(x), T.quantize_rows(x[n - 70:])
    assert all(torch.equal(a[n - 70:], b) for a, b in zip(whole, part))
    del whole
    ids = torch.randint(0, 1024, (n, 1), device=cuda, generator=g).int()
    whole, part = T.token_log_probs(x, ids, 3), T.token_log_probs(x[n - 70:], ids[n - 70:], 3)
    # another kernel may take fewer rows: its sums go in another order (at most 45 u each, see the other tests)
    assert torch.equal(whole.top_ids[n - 70:], part.top_ids)
    assert all(((a[n - 70:] - b).abs() <= 2 * 5.3e-6 * 15).all() for a, b in ((whole.log_probs, part.log_probs), (whole.entropy, part.entropy)))


@pytest.mark.parametrize("out", ["fp16", "fp32"])
def test_fc_rowwise_gelu_over_its_whole_range(cuda, out):
    """One product of ones, the row's scale is the value. FP16 results: within 2.6e-5 + |x| 2^-12 of the exact GELU (fit; tanh.approx, 2^-11 relative), |x| 2^-20
    for its FP32 arithmetic, and the rounding of the result: in the negative tail that is the absolute error, whatever is left of the result. FP32 results: erff."""
    import tensorrt_b200 as T

    x = torch.cat([torch.linspace(-14, 14, 2 ** 17 + 3), torch.tensor([0.0, -0.0, 1e-30, -1e-30, -60000.0, 60000.0, -1e30])]).to(cuda)
    one = torch.ones((len(x), 16), dtype=torch.int8, device=cuda)[:, :1]
    w = torch.ones((8, 16), dtype=torch.int8, device=cuda)[:, :1]
    dtype = TYPES[out][0]
    y = T.fc_rowwise(one, x, w, torch.ones(8, device=cuda), None, T.ACT_GELU_ERF, out_dtype=dtype).double()
    assert torch.equal(y, y[:, :1].expand_as(y))
    v = x.double()
    ref = 0.5 * v * torch.special.erfc(-v / 2 ** 0.5)
    if out == "fp16":
        tol = 2.6e-5 + v.abs() * (2.0 ** -12 + 2.0 ** -20) + torch.clamp(ref.abs() * 2.0 ** -11, min=2.0 ** -25)
    else:
        tol = v.abs() * 2.0 ** -22 + ref.abs() * 2.0 ** -23
    fits = ref.abs() < 65504
    err = (y[:, 0] - ref).abs()
    assert (err <= tol)[fits].all(), float((err / tol)[fits].max())
