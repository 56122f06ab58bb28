"""The masked-language-model head's weights and refusals, as far as they need no GPU."""
import numpy as np
import pytest
import torch


def _state_dict(hidden=32, vocab=50):
    rng = np.random.default_rng(0)
    a = lambda *s: rng.standard_normal(s).astype(np.float32)
    p = "cls.predictions."
    return {p + "transform.dense.weight": a(hidden, hidden), p + "transform.dense.bias": a(hidden), p + "transform.LayerNorm.weight": a(hidden),
            p + "transform.LayerNorm.bias": a(hidden), p + "bias": a(vocab), "bert.embeddings.word_embeddings.weight": a(vocab, hidden)}


def test_hidden_states_of_another_type_or_width_are_refused():
    """The FP16 product goes by the hidden states' type and width: others would be read past the weights' end."""
    from tensorrt_b200.checkpoint import MaskedLmHead

    head = MaskedLmHead(_state_dict(), device="cpu", rowwise=False)
    for bad in (torch.zeros(4, 32), torch.zeros(4, 40).half(), torch.zeros(4, 24).half(), torch.zeros(2, 4, 32).half(), torch.zeros(32).half(), torch.zeros(4, 32).bfloat16()):
        with pytest.raises(ValueError, match="hidden states"):
            head.logits(bad)
        with pytest.raises(ValueError, match="hidden states"):
            head(bad, top_k=1)
    with pytest.raises(ValueError, match="CUDA"):
        head.logits(torch.zeros(4, 32).half())


def test_weights_in_any_order_of_storage():
    """A checkpoint's arrays may be views (a transposed kernel of another framework): the kernels get contiguous weights of the same values."""
    from tensorrt_b200.checkpoint import MaskedLmHead

    sd = _state_dict()
    turned = {k: np.asfortranarray(v) for k, v in sd.items()}
    turned["cls.predictions.transform.dense.bias"] = np.repeat(sd["cls.predictions.transform.dense.bias"], 2)[::2]
    turned["cls.predictions.bias"] = np.repeat(sd["cls.predictions.bias"], 2)[::2]
    turned["bert.embeddings.word_embeddings.weight"] = torch.from_numpy(np.ascontiguousarray(sd["bert.embeddings.word_embeddings.weight"].T)).t()
    a, b = (MaskedLmHead(d, device="cpu", rowwise=False) for d in (sd, turned))
    for name in ("dense", "dense_bias", "gamma", "beta", "decoder", "bias"):
        x, y = getattr(a, name), getattr(b, name)
        assert torch.equal(x, y) and y.is_contiguous(), name


@pytest.mark.parametrize("name", ["transform.dense.weight", "transform.LayerNorm.bias", "bias"])
def test_a_missing_weight_is_named(name):
    from tensorrt_b200.checkpoint import MaskedLmHead

    sd = _state_dict()
    del sd["cls.predictions." + name]
    with pytest.raises(KeyError, match="cls.predictions." + name):
        MaskedLmHead(sd, device="cpu", rowwise=False)
