"""Sizes at the ends of the row-wise operators' counters: turned away by host code, before any launch."""
import ctypes as C

FAKE = 0x10000  # never dereferenced


def test_fc_rowwise_strides_whose_bytes_pass_64_bits():
    from tensorrt_b200 import _lib as L

    names = [n for n, _ in L.FcRowwiseParams._fields_]
    good = dict(zip(names, (0, 0, 8, 20, 100, FAKE, 112, FAKE, FAKE, 112, FAKE, FAKE, 24, FAKE, None)))
    for change in (dict(ldc=2 ** 62), dict(ldc=2 ** 62 + 24), dict(ldc=2 ** 38), dict(out_type_id=1, ldc=2 ** 62), dict(out_type_id=1, ldc=2 ** 39), dict(lda=2 ** 62), dict(ldw=2 ** 40)):
        p = L.FcRowwiseParams(*{**good, **change}.values())
        assert L.lib.bert_b200_fc_rowwise(C.byref(p), None) == 2, change
        assert b"40 bits" in L.lib.bert_b200_last_error()
