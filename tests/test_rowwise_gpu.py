"""Row-wise INT8 (through the C ABI): quantisation of rows, residual + LayerNorm with quantised rows, the INT8 product with a scale per row and per
output channel, against 64-bit NumPy.

Tolerances, u = 2^-24 (half a step of FP32), h = 2^-11 (of FP16):
* quantised rows and scales are exact: one right answer each;
* product: int32 -> FP32, times the row's scale, multiply-add with the channel's scale and the bias: 3 u (|a b s| + |bias|) + u |result|, then h |result|
  (2^-25 below the smallest normal FP16);
* its GELU, FP16: fitted form 2.6e-5, tanh.approx 2^-11 relative: |x| 2^-12, its FP32 arithmetic 2^-20 |x|; FP32: erff 2 units in the last place and its
  argument: 2^-22 |x|; both: 1.13 times the error of x;
* LayerNorm: FP16 results as skip_layer_norm, to the bit.
"""
import numpy as np
import pytest
import torch

from oracle import rowwise_oracle as R

pytestmark = pytest.mark.gpu

U, H = 2.0 ** -24, 2.0 ** -11
TYPES = {"fp16": (torch.float16, np.float16), "fp32": (torch.float32, np.float32)}


def _rows(rng, rows, width, dtype):
    x = rng.standard_normal((rows, width)) * np.exp(rng.standard_normal((rows, 1)))
    return x.astype(dtype)


def _check_rows(q, scales, x):
    rq, rs = R.quantize_rows(x)
    np.testing.assert_array_equal(q.cpu().numpy(), rq)
    np.testing.assert_array_equal(scales.cpu().numpy(), rs)


# widths around the borders of 16-byte chunks and of the kernels: one warp per row up to 1024 halves / 512 floats, eight up to 8192 / 4096, then the
# kernel that reads a row twice
@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
@pytest.mark.parametrize("width", [1, 2, 7, 8, 31, 255, 256, 257, 500, 768, 1000, 1024, 1025, 2048, 3001, 4096, 4097, 8192, 8193, 20000])
def test_quantize_rows_is_exact(cuda, dtype, width):
    import tensorrt_b200 as T

    t, n = TYPES[dtype]
    rng = np.random.default_rng(width)
    for rows in (1, 3, 77):
        x = _rows(rng, rows, width, n)
        q, s = T.quantize_rows(torch.from_numpy(x).to(cuda))
        assert q.shape == (rows, width) and q.dtype == torch.int8 and s.shape == (rows,)
        _check_rows(q, s, x)


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
def test_quantize_rows_many_rows(cuda, dtype):
    """More rows than the grid has places for."""
    import tensorrt_b200 as T

    t, n = TYPES[dtype]
    for width in (64, 4096, 1001):
        x = _rows(np.random.default_rng(3), 20001 if width < 4096 else 5001, width, n)
        _check_rows(*T.quantize_rows(torch.from_numpy(x).to(cuda)), x)


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
def test_quantize_rows_halves_between_steps(cuda, dtype):
    """Quotients that are exactly, or next to, a half between two steps: rounded as the exact quotient, halves to even."""
    import tensorrt_b200 as T

    t, n = TYPES[dtype]
    rng = np.random.default_rng(0)
    amax = (127 * 2.0 ** rng.integers(-6, 3, size=(50, 1))).astype(n)
    k = rng.integers(-127, 127, size=(50, 1024)) + 0.5
    x = (k * amax.astype(np.float64) / 127).astype(n)
    x[:, 0] = amax[:, 0]
    assert (np.abs(np.abs(127.0 * x.astype(np.float64) / amax) % 1 - 0.5) == 0).mean() > 0.9
    _check_rows(*T.quantize_rows(torch.from_numpy(x).to(cuda)), x)
    # one step of the type away from where a half would be, for maxima that are no powers of two
    amax = rng.uniform(0.5, 100, size=(200, 1)).astype(n)
    x = ((rng.integers(-126, 126, size=(200, 1000)) + 0.5) * amax.astype(np.float64) / 127).astype(n)
    x = np.where(rng.random(x.shape) < 0.5, np.nextafter(x, n(0)), x)
    x[:, 7] = -amax[:, 0]
    _check_rows(*T.quantize_rows(torch.from_numpy(x).to(cuda)), x)


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
@pytest.mark.parametrize("width", [96, 1003])
def test_quantize_rows_special_rows(cuda, dtype, width):
    """Zeros, the smallest and the largest numbers, infinities and NaN; the rows beside them keep theirs."""
    import tensorrt_b200 as T

    t, n = TYPES[dtype]
    x = _rows(np.random.default_rng(1), 12, width, n)
    info = np.finfo(n)
    x[1] = 0
    x[2] = 0
    x[2, 3] = info.smallest_subnormal
    x[3] = x[3] / np.abs(x[3]).max() * n(info.smallest_subnormal) * n(90)
    x[4, 5] = info.max
    x[5, width - 1] = -info.max
    x[6, 0] = np.inf
    x[7, width - 1] = -np.inf
    x[8, width // 2] = np.nan
    x[9] = -0.0
    x[10] = np.nan
    q, s = T.quantize_rows(torch.from_numpy(x).to(cuda))
    _check_rows(q, s, x)
    assert s[1] == 0 and torch.isnan(s[[6, 7, 8, 10]]).all()


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
@pytest.mark.parametrize("pad,offset", [(8, 0), (3, 0), (8, 1), (1, 3), (0, 1)])
def test_quantize_rows_strides_and_alignment(cuda, dtype, pad, offset):
    import tensorrt_b200 as T

    t, n = TYPES[dtype]
    for width in (64, 257, 1000):
        buf = _rows(np.random.default_rng(pad), 33, width + pad + offset, n)
        view = torch.from_numpy(buf).to(cuda)[:, offset:offset + width]
        _check_rows(*T.quantize_rows(view), buf[:, offset:offset + width])


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
@pytest.mark.parametrize("width", [1, 5, 300, 505, 510, 513, 770, 1017, 1018, 1025, 1533, 2041, 3000, 4081, 4090, 4095, 4097, 6001, 8185, 8192, 8193])
def test_quantize_rows_that_begin_anywhere(cuda, dtype, width):
    """Row strides that are no multiple of 16 bytes, every kernel for few and for many rows; NaN before, between and behind the rows, and what lies between
    the results' rows, are left alone."""
    from tensorrt_b200 import _lib

    t, n = TYPES[dtype]
    rng = np.random.default_rng(width)
    for rows, pad, offset in ((1, 0, 3), (2, 1, 1), (9, 1, 5), (9, 6, 0), (9, 0, 2), (330, 3, 7)):
        stride = width + pad
        buf = np.full(offset + rows * stride + 3, np.nan, dtype=n)
        x = _rows(rng, rows, width, n)
        buf[offset:offset + rows * stride].reshape(rows, stride)[:, :width] = x
        d = torch.from_numpy(buf).to(cuda)
        ld = (width + 23) // 8 * 8
        out = torch.full((rows, ld), 99, dtype=torch.int8, device=cuda)
        scales = torch.full((rows + 1,), 5.0, device=cuda)
        assert _lib.lib.bert_b200_quantize_rows(torch.cuda.current_stream().cuda_stream, 1 if dtype == "fp16" else 0, rows, width,
                                                d.data_ptr() + offset * d.element_size(), stride, out.data_ptr(), ld, scales.data_ptr()) == 0
        _check_rows(out[:, :width], scales[:rows], x)
        assert (out[:, width:] == 99).all() and scales[rows] == 5


def test_quantize_rows_shapes_and_untouched_padding(cuda):
    import ctypes as C

    import tensorrt_b200 as T
    from tensorrt_b200 import _lib

    x = torch.randn(5, 3, 64, device=cuda).half()
    q, s = T.quantize_rows(x)
    assert q.shape == x.shape and s.shape == (5, 3)
    _check_rows(q.reshape(15, 64), s.reshape(15), x.reshape(15, 64).cpu().numpy())
    q, s = T.quantize_rows(x[0, 0])
    assert q.shape == (64,) and s.shape == ()
    q, s = T.quantize_rows(x[:0])
    assert q.shape == (0, 3, 64) and s.shape == (0, 3)
    # rows of a wider output: what lies between them stays as it was; output rows of any alignment
    for width, stride in ((64, 70), (61, 61), (100, 104), (9000, 9001)):
        y = torch.randn(7, width, device=cuda).half()
        out = torch.full((7 * stride + 5,), 99, dtype=torch.int8, device=cuda)
        scales = torch.full((9,), 5.0, device=cuda)
        st = _lib.lib.bert_b200_quantize_rows(torch.cuda.current_stream().cuda_stream, 1, 7, width, y.data_ptr(), width, out.data_ptr() + 1, stride,
                                              scales.data_ptr() + 4)
        assert st == 0
        o = out.cpu().numpy()
        rows = o[1:1 + 7 * stride].reshape(7, stride)
        _check_rows(torch.from_numpy(rows[:, :width].copy()), scales[1:8], y.cpu().numpy())
        assert (rows[:, width:] == 99).all() and o[0] == 99 and (o[1 + 7 * stride:] == 99).all()
        assert scales[0] == 5 and scales[8] == 5


def _fc_case(rng, m, n, k, full=False):
    hi = 128 if full else 127
    a = rng.integers(-hi, 128, size=(m, k)).astype(np.int8)
    w = rng.integers(-hi, 128, size=(n, k)).astype(np.int8)
    sa = np.exp(rng.standard_normal(m) - 4).astype(np.float32)
    sw = (rng.uniform(0.5, 2, n) * 0.02 / np.sqrt(k)).astype(np.float32)
    b = rng.standard_normal(n).astype(np.float32)
    return a, sa, w, sw, b


def _padded(a, cuda, mult=16):
    t = torch.full((a.shape[0], (a.shape[1] + mult - 1) // mult * mult), 77, dtype=torch.int8)  # what lies behind a row must not matter
    t[:, :a.shape[1]] = torch.from_numpy(a)
    return t.to(cuda)[:, :a.shape[1]]


def _fc_tolerance(v, ref, mags, act, fp16):
    err = 3 * U * mags + U * np.abs(v)
    if act:
        err = 1.13 * err + (2.6e-5 + np.abs(v) * (2.0 ** -12 + 2.0 ** -20) if fp16 else np.abs(v) * 2.0 ** -22) + 2 * U * np.abs(ref)
    return err + (np.maximum(H * np.abs(ref), 2.0 ** -25) if fp16 else U * np.abs(ref))


def _check_fc(T, cuda, case, out_dtype, bias, act):
    a, sa, w, sw, b = case
    t = lambda x: torch.from_numpy(x).to(cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    y = T.fc_rowwise(_padded(a, cuda), t(sa), _padded(w, cuda), t(sw), bias=t(b) if bias else None, activation=T.ACT_GELU_ERF if act else T.ACT_NONE,
                     out_dtype=out_dtype, status=status)
    assert int(status) == 0
    assert y.shape == (a.shape[0], w.shape[0]) and y.dtype == out_dtype
    v, ref, mags = R.fc_rowwise(a, sa, w, sw, b if bias else None, act)
    err = np.abs(y.double().cpu().numpy() - ref)
    tol = _fc_tolerance(v, ref, mags, act, out_dtype == torch.float16)
    assert (err <= tol).all(), (float((err / tol).max()), np.unravel_index(np.argmax(err / tol), err.shape))
    return y


# rows, columns and depths around tiles, 16-byte pieces and swizzle spans; tile kernels of 16 to 128 columns
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 16, 16), (1, 30522, 64), (3, 7, 33), (5, 17, 100), (8, 1000, 128), (37, 1024, 1024), (64, 100, 513), (65, 31, 64),
                                   (127, 33, 129), (128, 640, 256), (129, 15, 1000), (130, 1001, 384), (257, 1001, 96), (130, 3500, 200), (130, 5003, 64), (300, 4100, 1024)])
@pytest.mark.parametrize("out", ["fp16", "fp32"])
def test_fc_rowwise(cuda, m, n, k, out):
    import tensorrt_b200 as T

    case = _fc_case(np.random.default_rng(m + n + k), m, n, k)
    for bias, act in ((True, 0), (False, 0), (True, 1)):
        _check_fc(T, cuda, case, TYPES[out][0], bias, act)


# pair kernels of 128, 160, 192, 224 and 256 columns; the last columns of each end inside a 16-byte piece
@pytest.mark.parametrize("m,n,k", [(38000, 100, 64), (1000, 5003, 200), (700, 8009, 260), (700, 10007, 128), (1500, 6007, 500), (640, 30522, 256)])
@pytest.mark.parametrize("out", ["fp16", "fp32"])
def test_fc_rowwise_pair_tiles(cuda, m, n, k, out):
    import tensorrt_b200 as T

    case = _fc_case(np.random.default_rng(m + n + k), m, n, k)
    _check_fc(T, cuda, case, TYPES[out][0], True, 0)
    _check_fc(T, cuda, case, TYPES[out][0], False, 1)


def test_fc_rowwise_largest_sums(cuda):
    """Sums close to the end of 32 bits."""
    import tensorrt_b200 as T

    k = 131071
    a = np.full((9, k), -128, dtype=np.int8)
    w = np.full((40, k), -128, dtype=np.int8)
    a[3] = 127
    w[5] = 127
    a[4, ::2] = 127
    case = (a, np.full(9, 1e-4, np.float32), w, np.full(40, 1e-4, np.float32), np.zeros(40, np.float32))
    y = _check_fc(T, cuda, case, torch.float32, False, 0)
    assert abs(float(y[0, 0]) - 128.0 * 128 * k * 1e-8) < 1e-3


def test_fc_rowwise_row_does_not_depend_on_the_others(cuda):
    import tensorrt_b200 as T

    rng = np.random.default_rng(5)
    a, sa, w, sw, b = _fc_case(rng, 3000, 1000, 700)
    t = lambda x: torch.from_numpy(x).to(cuda)
    ta, tw = _padded(a, cuda), _padded(w, cuda)
    whole = T.fc_rowwise(ta, t(sa), tw, t(sw), t(b))
    for m in (1, 37, 100, 200, 900):
        part = T.fc_rowwise(ta[:m], t(sa)[:m], tw, t(sw), t(b))
        assert torch.equal(part, whole[:m]), m


def test_fc_rowwise_special_scales(cuda):
    """A row of zeros (scale 0) gives the bias, a row without a scale NaN, and only that row."""
    import tensorrt_b200 as T

    rng = np.random.default_rng(6)
    x = rng.standard_normal((40, 256)).astype(np.float32)
    x[3] = 0
    x[7, 5] = np.nan
    x[39, 0] = np.inf
    w = rng.standard_normal((72, 256)).astype(np.float32)
    b = torch.from_numpy(rng.standard_normal(72).astype(np.float32)).to(cuda)
    q, s = T.quantize_rows(torch.from_numpy(x).to(cuda))
    wq, ws = T.quantize_rows(torch.from_numpy(w).to(cuda))
    y = T.fc_rowwise(q, s, wq, ws, b, out_dtype=torch.float32)
    bad = torch.isnan(y).all(dim=1)
    assert bad.nonzero().flatten().tolist() == [7, 39] and not torch.isnan(y[~bad]).any()
    assert torch.equal(y[3], b)


def test_fc_rowwise_writes_only_its_columns(cuda):
    """C as columns of a wider tensor: the neighbours, and rows behind the last, stay as they were."""
    import tensorrt_b200 as T

    rng = np.random.default_rng(7)
    for m, n, k in ((37, 1001, 64), (130, 77, 64), (700, 8009, 64), (1, 3, 16), (39000, 3, 16), (39000, 45, 16)):
        for dtype in (torch.float16, torch.float32):
            a, sa, w, sw, b = _fc_case(rng, m, n, k)
            t = lambda x: torch.from_numpy(x).to(cuda)
            wide = torch.full((m + 2, (n + 32) // 16 * 16 + 16), 3.0, dtype=dtype, device=cuda)
            out = wide[1:m + 1, 8:8 + n]
            ref = T.fc_rowwise(t(a), t(sa), t(w), t(sw), t(b), out_dtype=dtype)
            got = T.fc_rowwise(t(a), t(sa), t(w), t(sw), t(b), out_dtype=dtype, out=out)
            assert got is out and torch.equal(out, ref)
            wide[1:m + 1, 8:8 + n] = 3.0
            assert (wide == 3.0).all(), (m, n, dtype)


def test_fc_rowwise_operands_in_wider_tensors(cuda):
    import tensorrt_b200 as T

    rng = np.random.default_rng(8)
    a, sa, w, sw, b = _fc_case(rng, 50, 48, 96)
    t = lambda x: torch.from_numpy(x).to(cuda)
    ref = T.fc_rowwise(t(a), t(sa), t(w), t(sw), t(b))
    wa = torch.full((50, 160), 5, dtype=torch.int8, device=cuda)
    wa[:, 32:128] = t(a)
    ww = torch.full((48, 112), 5, dtype=torch.int8, device=cuda)
    ww[:, :96] = t(w)
    assert torch.equal(T.fc_rowwise(wa[:, 32:128], t(sa), ww[:, :96], t(sw), t(b)), ref)
    # a single row whose stride says nothing
    one = T.fc_rowwise(wa[7:8, 32:128], t(sa)[7:8], ww[:, :96], t(sw), t(b))
    assert torch.equal(one, ref[7:8])
    assert T.fc_rowwise(t(a)[:0], t(sa)[:0], t(w), t(sw)).shape == (0, 48)


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
@pytest.mark.parametrize("ld", [1, 4, 8, 30, 100, 104, 256, 768, 1000, 1024, 2048, 4096, 8192, 8200])
def test_skip_layer_norm_quantize(cuda, dtype, ld):
    """y: the bits of skip_layer_norm. The INT8 rows: those of the FP32 result, which is known to a few units in the last place, so a value may lie on
    the neighbouring step only where the exact quotient lies that near a half."""
    import tensorrt_b200 as T

    t, n = TYPES[dtype]
    rng = np.random.default_rng(ld)
    rows = 45
    x, s = (rng.standard_normal((rows, ld)).astype(n) for _ in range(2))
    g = (1 + 0.02 * rng.standard_normal(ld)).astype(n)
    b, bi = (0.02 * rng.standard_normal(ld).astype(n) for _ in range(2))
    d = lambda v: None if v is None else torch.from_numpy(v).to(cuda)
    eps0 = 0.0 if dtype == "fp16" else float(np.finfo(np.float32).eps)
    for bias in (None, bi):
        if ld > 1:  # (a row of one value has no variance: with eps 0 there is nothing to compare)
            y, _, _ = T.skip_layer_norm_quantize(d(x), d(s), d(g), d(b), d(bias), eps=eps0)
            assert torch.equal(y, T.skip_layer_norm(d(x), d(s), d(g), d(b), d(bias)))
        for skip in (s, None):
            eps = 1e-6
            y, q, scales = T.skip_layer_norm_quantize(d(x), d(skip), d(g), d(b), d(bias), eps=eps)
            none, q2, scales2 = T.skip_layer_norm_quantize(d(x), d(skip), d(g), d(b), d(bias), eps=eps, with_output=False)
            assert none is None and torch.equal(q, q2) and torch.equal(scales, scales2)
            ref = R.layer_norm(x, skip, g, b, bias, eps)
            # FP32 error of y: sums of ld values over at most 32 chained additions and a tree, mean and variance, five roundings at the end;
            # relative to the row's largest magnitude, which is what a step is a part of
            amax = np.abs(ref).max(axis=1, keepdims=True)
            rel = 64 * U * (1 + np.abs(ref)) / np.maximum(amax, 1e-30) + 64 * U
            np.testing.assert_allclose(scales.cpu().numpy(), (amax / 127)[:, 0], rtol=0, atol=float((64 * U * (1 + amax) / 127).max()))
            exact = 127 * ref / amax
            assert (np.abs(q.cpu().numpy() - exact) <= 0.5 + 127 * rel).all()
            assert np.abs(y.double().cpu().numpy() - ref).max() <= (H if dtype == "fp16" else 0) * np.abs(ref).max() + 64 * U * (1 + np.abs(ref).max())


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
@pytest.mark.parametrize("ld", [3, 31, 255, 257, 510, 513, 767, 769, 770, 1001, 1023, 1025, 2041, 2047, 2049, 4001, 4095, 4097, 8001, 8191, 8193])
def test_skip_layer_norm_quantize_odd_widths(cuda, dtype, ld):
    """Rows that begin at any value, tensors that do too, few and many of them, in place: y to the bit that of skip_layer_norm, the INT8 rows those of any
    other call with the same values; what lies around the tensors is left alone."""
    import tensorrt_b200 as T

    t, n = TYPES[dtype]
    gen = torch.Generator(device=cuda).manual_seed(ld)
    eps = 0.0 if dtype == "fp16" else float(np.finfo(np.float32).eps)

    def tensor(shape, offset, of=None):
        """`shape` values that begin `offset` values behind a multiple of 16 bytes, between NaN."""
        size = int(np.prod(shape))
        buf = torch.full((offset + size + 9,), float("nan"), dtype=t, device=cuda)
        buf[offset:offset + size] = (torch.randn(size, device=cuda, generator=gen) if of is None else of.flatten()).to(t)
        return buf[offset:offset + size].view(shape)

    for rows, skipped, biased in ((1, True, False), (7, True, True), (45, False, True), (1500 if ld < 1100 else 700, True, True)):
        x, s = tensor((rows, ld), rows % 5), tensor((rows, ld), 3) if skipped else None
        g, b, bi = tensor((ld,), 1), tensor((ld,), 0), tensor((ld,), 2) if biased else None
        y, q, scales = T.skip_layer_norm_quantize(x, s, g, b, bi, eps=eps)
        if skipped:
            assert torch.equal(y, T.skip_layer_norm(x, s, g, b, bi))
        else:
            assert torch.equal(y, T.skip_layer_norm_quantize(x, torch.zeros_like(x), g, b, bi, eps=eps)[0])
        ref = R.layer_norm(*(None if v is None else v.cpu().numpy() for v in (x, s, g, b, bi)), eps)
        amax = np.abs(ref).max(axis=1, keepdims=True)
        # as above, the sums here over up to 256 chained additions
        err = 288 * U * (1 + np.abs(ref).max())
        np.testing.assert_allclose(scales.cpu().numpy(), amax[:, 0] / 127, rtol=2 * U, atol=err / 127)
        assert (np.abs(q.cpu().numpy() - 127 * ref / amax) <= 0.5 + 127 * 2 * err / amax).all()
        # other places in memory, and in place: the same answers
        x2 = tensor((rows, ld), 6, x)
        y2, q2, scales2 = T.skip_layer_norm_quantize(x2, None if s is None else tensor((rows, ld), 0, s), g, b, bi, eps=eps)
        assert torch.equal(y, y2) and torch.equal(q, q2) and torch.equal(scales, scales2)
        q3, scales3 = torch.full((rows * ld + 2,), 99, dtype=torch.int8, device=cuda), torch.full((rows + 1,), 5.0, device=cuda)
        x3 = x2._base.clone()
        assert T._lib.lib.bert_b200_skip_layer_norm_quantize(
            torch.cuda.current_stream().cuda_stream, 1 if dtype == "fp16" else 0, ld, rows * ld, x3.data_ptr() + 6 * x3.element_size(), None if s is None else s.data_ptr(),
            b.data_ptr(), g.data_ptr(), x3.data_ptr() + 6 * x3.element_size(), q3.data_ptr() + 1, scales3.data_ptr(), None if bi is None else bi.data_ptr(), eps) == 0
        assert torch.equal(x3[6:6 + rows * ld].view(rows, ld), y) and torch.isnan(x3[:6]).all() and torch.isnan(x3[6 + rows * ld:]).all()
        assert torch.equal(q3[1:-1].view(rows, ld), q) and q3[0] == 99 and q3[-1] == 99 and torch.equal(scales3[:-1], scales) and scales3[-1] == 5


def test_skip_layer_norm_quantize_special_rows(cuda):
    import tensorrt_b200 as T

    for ld in (64, 1024, 100):
        x = torch.randn(9, ld, device=cuda).half()
        x[2, 3] = float("nan")
        x[5, ld - 1] = float("inf")
        x[7] = 4.0  # no variance: with eps the row is beta
        g, b = torch.ones(ld, device=cuda).half(), torch.zeros(ld, device=cuda).half()
        y, q, s = T.skip_layer_norm_quantize(x, None, g, b, eps=1e-12)
        assert torch.isnan(s).nonzero().flatten().tolist() == [2, 5] and (q[[2, 5]] == 0).all()
        assert s[7] == 0 and (q[7] == 0).all() and (y[7] == 0).all()
        # in place: the output over the input, and over the residual
        x2, s2 = torch.randn(9, ld, device=cuda).half(), torch.randn(9, ld, device=cuda).half()
        ref = T.skip_layer_norm_quantize(x2, s2, g, b)
        from tensorrt_b200 import _lib
        for over in (0, 1):
            ins = [x2.clone(), s2.clone()]
            q, sc = torch.empty_like(ref[1]), torch.empty_like(ref[2])
            assert _lib.lib.bert_b200_skip_layer_norm_quantize(torch.cuda.current_stream().cuda_stream, 1, ld, x2.numel(), ins[0].data_ptr(), ins[1].data_ptr(),
                                                               b.data_ptr(), g.data_ptr(), ins[over].data_ptr(), q.data_ptr(), sc.data_ptr(), None, 0.0) == 0
            assert torch.equal(ins[over], ref[0]) and torch.equal(q, ref[1]) and torch.equal(sc, ref[2])
    e = torch.empty((0, 64), dtype=torch.float16, device=cuda)
    y, q, s = T.skip_layer_norm_quantize(e, e, torch.ones(64, device=cuda).half(), torch.ones(64, device=cuda).half())
    assert y.shape == (0, 64) and q.shape == (0, 64) and s.shape == (0,)


def test_a_block_of_layers(cuda):
    """LayerNorm -> product with GELU -> quantisation -> product -> LayerNorm, on a side stream, then captured and replayed on other inputs."""
    import tensorrt_b200 as T

    g = torch.Generator(device=cuda).manual_seed(0)
    E, F, rows = 256, 1000, 150
    rnd = lambda *s: torch.randn(s, device=cuda, generator=g)
    w1, s1 = T.quantize_rows((0.05 * rnd(F, E)).half())
    w2, s2 = T.quantize_rows((0.05 * rnd(E, F)).half())
    gamma, beta, b1, b2 = (1 + 0.1 * rnd(E)).half(), (0.1 * rnd(E)).half(), rnd(F), (0.1 * rnd(E)).half()
    x = rnd(rows, E).half()

    def block():
        y, q, s = T.skip_layer_norm_quantize(x, None, gamma, beta, eps=1e-12)
        f, fs = T.quantize_rows(T.fc_rowwise(q, s, w1, s1, b1, T.ACT_GELU_ERF))
        o = T.fc_rowwise(f, fs, w2, s2)
        return T.skip_layer_norm_quantize(o, y, gamma, beta, b2, eps=1e-12)

    ref = [t.clone() for t in block()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = block()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(ref, again))
    # against the same block in floating point: INT8 with a scale per row and channel is off by about 1 % of a layer's results
    yf = torch.nn.functional.layer_norm(x.double(), (E,), gamma.double(), beta.double(), 1e-12)
    f = torch.nn.functional.gelu(yf @ (w1.double() * s1.double()[:, None]).T + b1.double())
    o = f @ (w2.double() * s2.double()[:, None]).T
    out = torch.nn.functional.layer_norm(o + yf + b2.double(), (E,), gamma.double(), beta.double(), 1e-12)
    assert float((ref[0].double() - out).norm() / out.norm()) < 0.03
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = block()
    other = rnd(rows, E).half()
    x.copy_(other)
    graph.replay()
    torch.cuda.synchronize()
    now = block()
    assert all(torch.equal(a, b) for a, b in zip(captured, now)) and not torch.equal(now[0], ref[0])


def test_scales_and_bias_of_any_alignment(cuda):
    """Output channels of a larger layer: weights from any row on, with their scales and biases."""
    import tensorrt_b200 as T

    a, sa, w, sw, b = _fc_case(np.random.default_rng(9), 150, 500, 64)
    t = lambda x: torch.from_numpy(x).to(cuda)
    ta, tsa, tw, tsw, tb = (t(x) for x in (a, sa, w, sw, b))
    whole = T.fc_rowwise(ta, tsa, tw, tsw, tb)
    for i in (1, 3, 250):
        assert torch.equal(T.fc_rowwise(ta[i:], tsa[i:], tw[i:], tsw[i:], tb[i:]), whole[i:, i:])


def test_threads_and_streams_at_once(cuda):
    """Calls of different shapes from several threads, each on a stream of its own, give what they give one after the other."""
    import threading

    import tensorrt_b200 as T

    shapes = [(37, 1024, 1024), (300, 4100, 512), (1000, 5003, 200), (5, 70, 33)]
    cases = []
    for m, n, k in shapes:
        g = torch.Generator(device=cuda).manual_seed(m)
        x, w = torch.randn((m, k), device=cuda, generator=g).half(), torch.randn((n, k), device=cuda, generator=g).half()
        cases.append((x, *T.quantize_rows(w), torch.ones(k, device=cuda).half(), torch.zeros(k, device=cuda).half()))

    def call(case):
        x, w, s, gamma, beta = case
        _, _, _ = T.skip_layer_norm_quantize(x, x, gamma, beta)
        q, qs = T.quantize_rows(x)
        y = T.fc_rowwise(q, qs, w, s, out_dtype=torch.float32)
        return [q, qs, y, *T.token_log_probs(y, top_k=7)[1:]]

    want = [call(c) for c in cases]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = call(cases[i])
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    failed.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not failed, failed
