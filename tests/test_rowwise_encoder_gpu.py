"""INT8 without calibration: the encoder with a scale per token and output channel, and the masked-language-model head on top of it."""
import numpy as np
import pytest
import torch

from oracle import bert_oracle as O
from oracle import rowwise_oracle as R
from tests.test_checkpoint_cpu import make_hf, padded_batch

pytestmark = pytest.mark.gpu


def _t(a, cuda):
    return torch.from_numpy(np.ascontiguousarray(a)).to(cuda)


def _case(lengths, seed, layers=2, hidden=128, heads=2, ffn=512):
    rng = np.random.default_rng(seed)
    p = O.make_bert_params(rng, layers, hidden, heads, ffn, vocab=1000, max_pos=512)
    cu = O.cu_seqlens(np.array(lengths, dtype=np.int32))
    total = int(cu[-1])
    return p, rng.integers(0, 1000, size=total).astype(np.int32), rng.integers(0, 2, size=total).astype(np.int32), cu, int(max(lengths))


@pytest.mark.parametrize("lengths", [[128, 128], [384, 17, 200, 1], [1]])
def test_encoder_rowwise(cuda, lengths):
    """Against the same arithmetic in 64 bits. What differs is the rounding of FP16 intermediates, which moves a value to the neighbouring INT8 step
    now and then (a step is some 1 / 30 of a standard deviation, a product of 128 ... 512 terms moves by 1 / 30 * 0.02 with one of them): the
    whole-model bounds of the FP16 encoder hold."""
    import tensorrt_b200 as T

    p, ids, seg, cu, S = _case(lengths, len(lengths))
    ref = R.encoder(p, ids, seg, cu, S)
    enc = T.BertEncoder(p, T.INT8, cuda, rowwise=True)
    out = enc.forward(_t(ids, cuda), _t(seg, cuda), _t(cu, cuda), S)
    assert enc.status_word() == 0
    assert enc.launches_per_forward == 2 + 9 * len(p.layers)
    ok, worst, bad = O.close_abs_or_rel(out.cpu().numpy(), ref, 1e-2, 1e-2)
    assert bad <= out.numel() * 1e-3 and worst < 5e-2, (worst, bad)
    # and against floating point: 8 bits per token and channel
    fp = O.encoder_fp(p, ids, seg, cu, S, round_fp16=False)
    assert np.linalg.norm(out.cpu().numpy() - fp) / np.linalg.norm(fp) < 0.03
    # host buffers, the built-in workspace and a replayed graph give the same bytes
    total = len(ids)
    dev, host = torch.empty_like(out), torch.empty(out.shape, dtype=torch.float16).pin_memory()
    enc.forward_host(*(torch.from_numpy(a).pin_memory() for a in (ids, seg, cu)), S, dev, host)
    assert torch.equal(host, out.cpu())
    from tensorrt_b200._lib import lib

    args = (_t(ids, cuda), _t(seg, cuda), _t(cu, cuda))
    dev.zero_()
    assert lib.bert_b200_encoder_forward_static(enc._h, torch.cuda.current_stream().cuda_stream, len(lengths), total, S, *(a.data_ptr() for a in args),
                                                dev.data_ptr()) == 0
    assert torch.equal(dev, out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        enc.forward(*args, S, out=dev)
    dev.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(dev, out)
    enc.close()


def test_encoder_rowwise_full_width(cuda):
    """One layer of the large model's sizes on more rows than a row block, against the FP16 encoder of the same weights."""
    import tensorrt_b200 as T
    from tensorrt_b200 import synthetic

    p = synthetic.make_params(1, 1024, 16, 4096, vocab=2000, device=cuda)
    ids, seg, cu, lengths = synthetic.make_inputs(9, 384, vocab=2000, min_len=32, device=cuda)
    S = int(lengths.max())
    want = T.BertEncoder(p, T.FP16, cuda).forward(ids, seg, cu, S).float()
    enc = T.BertEncoder(p, T.INT8, cuda, rowwise=True)
    got = enc.forward(ids, seg, cu, S).float()
    assert enc.status_word() == 0
    assert float((got - want).norm() / want.norm()) < 0.02


def test_encoder_rowwise_needs_int8(cuda):
    import tensorrt_b200 as T

    p, *_ = _case([4], 0)
    with pytest.raises(ValueError, match="INT8"):
        T.BertEncoder(p, T.FP16, cuda, rowwise=True)


@pytest.mark.parametrize("tied", [True, False])
def test_masked_lm_head_matches_huggingface(cuda, tied):
    """BertForMaskedLM end to end: encoder and head, INT8 and FP16, against Hugging Face in FP32."""
    import transformers

    import tensorrt_b200 as T
    from tensorrt_b200.checkpoint import MaskedLmHead, pack_padded_batch, params_from_bert_state_dict

    torch.manual_seed(5)
    vocab = 907
    cfg = transformers.BertConfig(vocab_size=vocab, hidden_size=256, num_hidden_layers=2, num_attention_heads=4, intermediate_size=1000 // 16 * 16,
                                  max_position_embeddings=128, hidden_act="gelu", hidden_dropout_prob=0.0, attention_probs_dropout_prob=0.0,
                                  tie_word_embeddings=tied)
    model = transformers.BertForMaskedLM(cfg).eval()
    with torch.no_grad():
        for p in model.parameters():
            p.copy_((p + 0.05 * torch.randn_like(p)).half().float())
    rng = np.random.default_rng(4)
    B, S = 4, 96
    ids, seg, mask, lengths = padded_batch(rng, B, S, vocab)
    with torch.no_grad():
        logits = model(input_ids=torch.from_numpy(ids), token_type_ids=torch.from_numpy(seg), attention_mask=torch.from_numpy(mask)).logits
    want = torch.log_softmax(torch.cat([logits[b, :lengths[b]] for b in range(B)]).double(), dim=-1)
    sd = {k: v for k, v in model.state_dict().items() if not (tied and k.endswith("decoder.weight"))}
    params = params_from_bert_state_dict(sd, num_heads=4)
    pid, pseg, cu = pack_padded_batch(ids, seg, mask)
    dev = lambda a: torch.from_numpy(a).to(cuda)
    positions = torch.from_numpy(rng.choice(len(pid), size=40, replace=False)).to(cuda)
    tokens = torch.from_numpy(rng.integers(0, vocab, size=(40, 3)).astype(np.int32)).to(cuda)
    for rowwise in (False, True):
        enc = T.BertEncoder(params, T.INT8 if rowwise else T.FP16, cuda, rowwise=rowwise)
        hidden = enc.forward(dev(pid), dev(pseg), dev(cu), S)
        head = MaskedLmHead(sd, cuda, rowwise=rowwise)
        assert head.logits(hidden).shape == (len(pid), vocab)
        r = head(hidden, positions, tokens, top_k=5)
        ref = want.to(cuda)[positions]
        err = (r.log_probs.double() - torch.gather(ref, 1, tokens.long())).abs()
        spread = float(ref.std())
        # FP16: hidden states of O(1) off by a few 1e-3; INT8: two layers' and two products' steps, 1 % each of their results
        assert float(err.max()) < (0.05 if rowwise else 0.02) * max(spread, 1) * 4, (rowwise, float(err.max()), spread)
        assert float((r.entropy.double() + (ref.exp() * ref).sum(1)).abs().max()) < 0.2
        # what it says about its own logits is exact
        own = head.logits(hidden).float()[positions]
        assert torch.equal(r.top_ids.long(), torch.sort(own, dim=1, descending=True, stable=True).indices[:, :5])
        everywhere = head(hidden, top_k=1)
        assert everywhere.top_ids.shape == (len(pid), 1) and torch.equal(everywhere.top_ids[positions], r.top_ids[:, :1])
        enc.close()
