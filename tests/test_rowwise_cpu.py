"""Refusals of the row-wise INT8 operators and of the log probabilities: bad arguments are turned away by host code, before any launch."""
import ctypes as C

import numpy as np
import pytest
import torch

FAKE = 0x10000  # never dereferenced


def _lib():
    from tensorrt_b200 import _lib

    return _lib


def test_quantize_rows_refusals():
    L = _lib()
    f = L.lib.bert_b200_quantize_rows
    assert f(None, 1, 0, 64, None, 64, None, 64, None) == 0          # no rows: nothing to do
    for args in ((2, 4, 64, FAKE, 64, FAKE, 64, FAKE), (1, -1, 64, FAKE, 64, FAKE, 64, FAKE), (1, 4, 0, FAKE, 64, FAKE, 64, FAKE), (1, 4, 64, FAKE, 63, FAKE, 64, FAKE),
                 (1, 4, 64, FAKE, 64, FAKE, 63, FAKE), (1, 4, 64, None, 64, FAKE, 64, FAKE), (1, 4, 64, FAKE, 64, None, 64, FAKE), (1, 4, 64, FAKE, 64, FAKE, 64, None),
                 (1, 4, 64, FAKE + 1, 64, FAKE, 64, FAKE), (0, 4, 64, FAKE + 2, 64, FAKE, 64, FAKE), (1, 4, 64, FAKE, 64, FAKE, 64, FAKE + 2),
                 (1, 4, 2 ** 30 + 1, FAKE, 2 ** 31, FAKE, 2 ** 31, FAKE)):
        assert f(None, *args) == 2, args
        assert b"quantize_rows" in L.lib.bert_b200_last_error()


def test_skip_layer_norm_quantize_refusals():
    L = _lib()
    f = L.lib.bert_b200_skip_layer_norm_quantize
    good = dict(type_id=1, ld=64, n=640, x=FAKE, skip=FAKE, beta=FAKE, gamma=FAKE, y=FAKE, q=FAKE, s=FAKE, bias=FAKE, eps=0.0)
    for change in (dict(type_id=2), dict(ld=0), dict(n=-64), dict(n=641), dict(x=None), dict(beta=None), dict(gamma=None), dict(q=None), dict(s=None), dict(eps=-1.0),
                   dict(eps=float("nan"))):
        assert f(None, *{**good, **change}.values()) == 2, change
    assert f(None, *{**good, "n": 0}.values()) == 0


def test_fc_rowwise_refusals():
    L = _lib()
    f = L.lib.bert_b200_fc_rowwise
    names = [n for n, _ in L.FcRowwiseParams._fields_]
    good = dict(zip(names, (1, 0, 8, 20, 100, FAKE, 112, FAKE, FAKE, 112, FAKE, FAKE, 24, FAKE, None)))
    assert f(None, None) == 2
    for change in (dict(out_type_id=2), dict(activation=7), dict(m=-1), dict(n=0), dict(k=0), dict(k=131072, lda=131072, ldw=131072), dict(lda=96), dict(ldw=99), dict(ldc=16),
                   dict(lda=104), dict(ldw=120), dict(ldc=20), dict(out_type_id=0, ldc=22), dict(a=None), dict(a_scales=None), dict(wt=None), dict(wt_scales=None), dict(c=None),
                   dict(a=FAKE + 8), dict(wt=FAKE + 8), dict(c=FAKE + 8), dict(wt_scales=FAKE + 2), dict(bias=FAKE + 1), dict(a_scales=FAKE + 2), dict(m=2 ** 31),
                   dict(n=2 ** 31, ldc=2 ** 31 + 8)):
        p = L.FcRowwiseParams(*{**good, **change}.values())
        assert f(C.byref(p), None) == 2, change
        assert b"fc_rowwise" in L.lib.bert_b200_last_error()
    assert f(C.byref(L.FcRowwiseParams(*{**good, "m": 0}.values())), None) == 0


def test_token_log_probs_refusals():
    L = _lib()
    f = L.lib.bert_b200_token_log_probs
    names = [n for n, _ in L.LogProbsParams._fields_]
    good = dict(zip(names, (1, 4, 100, FAKE, 100, 2, FAKE, 5, FAKE, FAKE, FAKE, FAKE, None)))
    assert f(None, None) == 2
    for change in (dict(type_id=2), dict(rows=-1), dict(vocab=0), dict(vocab=2 ** 24 + 1, logits_stride=2 ** 25), dict(logits_stride=99), dict(num_tokens=-1), dict(top_k=-1),
                   dict(top_k=33), dict(logits=None), dict(token_ids=None), dict(log_probs=None), dict(top_ids=None), dict(top_log_probs=None), dict(logits=FAKE + 1),
                   dict(type_id=0, logits=FAKE + 2), dict(token_ids=FAKE + 2), dict(entropy=FAKE + 1), dict(num_tokens=0, top_k=0, entropy=None), dict(rows=2 ** 31)):
        p = L.LogProbsParams(*{**good, **change}.values())
        assert f(C.byref(p), None) == 2, change
        assert b"token_log_probs" in L.lib.bert_b200_last_error()
    assert f(C.byref(L.LogProbsParams(*{**good, "rows": 0}.values())), None) == 0


def test_token_log_probs_sizes_beyond_its_counters_are_refused():
    L = _lib()
    good = (1, 4, 100, FAKE, 100, 2, FAKE, 5, FAKE, FAKE, FAKE, FAKE, None)
    names = [n for n, _ in L.LogProbsParams._fields_]
    for change in (dict(num_tokens=2 ** 24 + 1), dict(num_tokens=2 ** 31 - 1), dict(rows=2 ** 28)):
        p = L.LogProbsParams(*{**dict(zip(names, good)), **change}.values())
        assert L.lib.bert_b200_token_log_probs(C.byref(p), None) == 2, change
        assert b"token_log_probs" in L.lib.bert_b200_last_error()


def test_tensors_off_the_gpu_are_refused():
    import tensorrt_b200 as T

    x = torch.zeros(4, 64, dtype=torch.float16)
    q, s = torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4)
    with pytest.raises(ValueError, match="CUDA"):
        T.quantize_rows(x)
    with pytest.raises(ValueError, match="CUDA"):
        T.fc_rowwise(q, s, q, s)
    with pytest.raises(ValueError, match="CUDA"):
        T.skip_layer_norm_quantize(x, x, x[0], x[0])
    with pytest.raises(ValueError, match="CUDA"):
        T.token_log_probs(x, torch.zeros(4, dtype=torch.int32))


def test_oracle_of_quantised_rows():
    """The oracle against whole-number arithmetic."""
    from fractions import Fraction

    from oracle import rowwise_oracle as R

    rng = np.random.default_rng(0)
    x = rng.standard_normal((20, 30)).astype(np.float32)
    x[0] = np.arange(-15, 15) / 2
    x[0, 0] = 127
    q, s = R.quantize_rows(x)
    for r in range(20):
        most = max(abs(Fraction(float(v))) for v in x[r])
        for j in range(30):
            assert q[r, j] == round(127 * Fraction(float(x[r, j])) / most)  # halves to even


def test_rowwise_encoder_refusals():
    L = _lib()
    layers = (L.LayerWeights * 2)()
    scales = (L.RowwiseScales * 2)()
    for lw in layers:
        for n, _ in L.LayerWeights._fields_:
            if not n.startswith("s_"):
                setattr(lw, n, C.c_void_p(FAKE))
    for s in scales:
        for n, _ in L.RowwiseScales._fields_:
            setattr(s, n, C.c_void_p(FAKE))
    f = C.c_void_p(FAKE)
    make = lambda type_id: L.EncoderConfig(type_id, 2, 128, 2, 512, 100, 64, 2, 0.0, f, f, f, f, f, layers)
    h = C.c_void_p()
    cfg = make(2)
    assert L.lib.bert_b200_encoder_create_rowwise(C.byref(cfg), scales, C.byref(h)) == 0     # no steps, no dq_probs needed
    L.lib.bert_b200_encoder_destroy(h)
    plain, rowwise = (f(C.byref(cfg), 100, 4) for f in (L.lib.bert_b200_encoder_workspace_size, L.lib.bert_b200_encoder_rowwise_workspace_size))
    assert rowwise > plain > 0
    assert L.lib.bert_b200_encoder_rowwise_workspace_size(C.byref(make(1)), 100, 4) == -1
    assert L.lib.bert_b200_encoder_create_rowwise(C.byref(make(1)), scales, C.byref(h)) == 2
    assert L.lib.bert_b200_encoder_create_rowwise(C.byref(cfg), None, C.byref(h)) == 2
    assert L.lib.bert_b200_encoder_create_rowwise(None, scales, C.byref(h)) == 2
    scales[1].wt_ffn2 = None
    assert L.lib.bert_b200_encoder_create_rowwise(C.byref(cfg), scales, C.byref(h)) == 2
    assert L.lib.bert_b200_encoder_create(C.byref(cfg), C.byref(h)) == 2                      # without them the steps are needed
