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
