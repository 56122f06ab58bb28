"""BERT checkpoint -> encoder parameters.

Takes a state dict in the Hugging Face `BertModel` naming (`embeddings.word_embeddings.weight`,
`encoder.layer.{i}.attention.self.query.weight`, ...; an optional leading `bert.` is stripped) and packs it the way
the plugins expect it: FC weights as [in, out] (the checkpoint stores [out, in]), and the three attention projections
of a layer fused into one [E, 3E] matrix whose output channels are ordered [head][q | k | v][d]
(ref: plugin/bertQKVToContextPlugin/README.md:26-30). The result has the attributes `BertEncoder` reads
(`synthetic.make_params` builds the same object from random numbers).

This is the step the removed `demo/BERT` builder performed before it wired the plugins into a network; the wiring
itself is `BertEncoder` / `bert_b200_encoder_forward`.
"""
from __future__ import annotations

from types import SimpleNamespace

import numpy as np


def _np(a) -> np.ndarray:
    if hasattr(a, "detach"):
        a = a.detach().cpu().float().numpy()
    return np.asarray(a, dtype=np.float32)


def params_from_bert_state_dict(state_dict, num_heads: int) -> SimpleNamespace:
    sd = {}
    for k, v in state_dict.items():
        k = k[5:] if k.startswith("bert.") else k
        sd[k] = v
    get = lambda name: _np(sd[name])
    word = get("embeddings.word_embeddings.weight")
    hidden = word.shape[1]
    if hidden % num_heads:
        raise ValueError(f"hidden size {hidden} is not a multiple of num_heads {num_heads}")
    d = hidden // num_heads
    layers = []
    i = 0
    while f"encoder.layer.{i}.attention.self.query.weight" in sd:
        p = f"encoder.layer.{i}."
        # checkpoint [out, in] -> [in, out]; output channels regrouped per head as (q, k, v)
        q, k, v = (get(p + f"attention.self.{n}.weight").T.reshape(hidden, num_heads, d) for n in ("query", "key", "value"))
        bq, bk, bv = (get(p + f"attention.self.{n}.bias").reshape(num_heads, d) for n in ("query", "key", "value"))
        w_qkv = np.stack([q, k, v], axis=2).reshape(hidden, 3 * hidden)
        b_qkv = np.stack([bq, bk, bv], axis=1).reshape(3 * hidden)
        h16 = lambda a: np.ascontiguousarray(a).astype(np.float16)
        layers.append(SimpleNamespace(
            w_qkv=h16(w_qkv), b_qkv=b_qkv.astype(np.float32),
            w_out=h16(get(p + "attention.output.dense.weight").T), b_out=h16(get(p + "attention.output.dense.bias")),
            ln1_gamma=h16(get(p + "attention.output.LayerNorm.weight")), ln1_beta=h16(get(p + "attention.output.LayerNorm.bias")),
            w_ffn1=h16(get(p + "intermediate.dense.weight").T), b_ffn1=get(p + "intermediate.dense.bias"),
            w_ffn2=h16(get(p + "output.dense.weight").T), b_ffn2=h16(get(p + "output.dense.bias")),
            ln2_gamma=h16(get(p + "output.LayerNorm.weight")), ln2_beta=h16(get(p + "output.LayerNorm.bias")), scales={}))
        i += 1
    if not layers:
        raise ValueError("no encoder.layer.* entries in the state dict")
    ffn = layers[0].w_ffn1.shape[1]
    return SimpleNamespace(
        hidden=hidden, heads=num_heads, ffn=ffn, word_emb=word.astype(np.float16),
        pos_emb=get("embeddings.position_embeddings.weight").astype(np.float16),
        tok_emb=get("embeddings.token_type_embeddings.weight").astype(np.float16),
        emb_gamma=get("embeddings.LayerNorm.weight"), emb_beta=get("embeddings.LayerNorm.bias"), layers=layers,
        dq_probs=1.0 / 127.0)


def pack_padded_batch(input_ids, token_type_ids, attention_mask):
    """[B, S] padded arrays (mask 1 = valid, valid tokens first) -> packed (ids, segment ids, cu_seqlens) int32."""
    ids, seg, mask = (np.asarray(a) for a in (input_ids, token_type_ids, attention_mask))
    lengths = mask.astype(np.int64).sum(axis=1)
    if (lengths == 0).any():
        raise ValueError("pack_padded_batch: sequence(s) %s have no valid token; drop them before packing (an empty "
                         "sequence has no [CLS] row for the heads to read)" % np.nonzero(lengths == 0)[0].tolist())
    cu = np.zeros(len(lengths) + 1, dtype=np.int32)
    cu[1:] = np.cumsum(lengths)
    pid = np.concatenate([ids[b, :lengths[b]] for b in range(len(lengths))]).astype(np.int32)
    pseg = np.concatenate([seg[b, :lengths[b]] for b in range(len(lengths))]).astype(np.int32)
    return pid, pseg, cu


class QaHead:
    """The span-prediction head of `BertForQuestionAnswering` (`qa_outputs`: hidden -> start / end logits) on top of
    the encoder output, run through the FC kernel. The two output channels are padded to 16 (the kernel's granularity);
    the padding rows are zero and dropped from the result."""

    def __init__(self, state_dict, device="cuda:0"):
        import torch

        w = _np(state_dict["qa_outputs.weight"])  # [2, hidden]
        b = _np(state_dict["qa_outputs.bias"])
        wt = np.zeros((16, w.shape[1]), dtype=np.float16)
        wt[:2] = w.astype(np.float16)
        bias = np.zeros(16, dtype=np.float32)
        bias[:2] = b
        self.wt = torch.from_numpy(wt).to(device)      # already [out, in], the layout the FC kernel reads
        self.bias = torch.from_numpy(bias).to(device)

    def __call__(self, hidden):
        """hidden: FP16 [total, hidden] (packed tokens) -> FP16 [total, 2] (start logit, end logit)."""
        from . import ops

        return ops.fc(hidden, self.wt, bias=self.bias)[:, :2]


class PoolerHead:
    """The pooler of `BertModel` (`pooler.dense` + tanh on the first token of every sequence) on top of the packed
    encoder output: the [CLS] rows are gathered with `cu_seqlens`, the dense layer runs through the FC kernel; the tanh
    of the B x hidden result is left to torch (the FC plugin has no tanh epilogue, neither has the reference's)."""

    def __init__(self, state_dict, device="cuda:0", prefix=""):
        import torch

        w = _np(state_dict[prefix + "pooler.dense.weight"])  # [hidden, hidden] = [out, in]
        b = _np(state_dict[prefix + "pooler.dense.bias"])
        self.wt = torch.from_numpy(np.ascontiguousarray(w.astype(np.float16))).to(device)
        self.bias = torch.from_numpy(b.astype(np.float32)).to(device)

    def __call__(self, hidden, cu_seqlens):
        """hidden: FP16 [total, hidden]; cu_seqlens: int32 [B + 1] -> FP16 [B, hidden]."""
        import torch

        from . import ops

        starts = cu_seqlens[:-1].long()
        if bool((cu_seqlens[1:].long() <= starts).any()):
            raise ValueError("PoolerHead: every sequence needs at least one token (its first row is the [CLS] row)")
        first = hidden.index_select(0, starts).contiguous()
        return torch.tanh(ops.fc(first, self.wt, bias=self.bias).float()).half()


class MaskedLmHead:
    """The head of `BertForMaskedLM` (`cls.predictions`: dense + erf-GELU + LayerNorm, then the product with the vocabulary) on top of the
    encoder output, and what it is asked: log probabilities of given tokens, entropy, the most likely tokens. The product with the vocabulary is
    usually tied to the word embeddings (no `decoder.weight` in the state dict). rowwise=True, which is what a caller gets who chooses nothing, also on
    an FP16 encoder: both products in INT8 with a scale per token and per output channel, logits FP32. False: both products in FP16, logits FP16, so that
    log probabilities carry the logits' rounding (2^-11 of their size: 1e-2 at logits of 20)."""

    def __init__(self, state_dict, device="cuda:0", rowwise=True, eps=1e-12):
        import torch

        from . import ops

        p = "cls.predictions."

        def get(*names):  # the first of them that is there
            name = next((n for n in names if n in state_dict), names[-1])
            return torch.from_numpy(np.ascontiguousarray(_np(state_dict[name]))).to(device)

        dense = get(p + "transform.dense.weight")
        decoder = get(p + "decoder.weight", "bert.embeddings.word_embeddings.weight", "embeddings.word_embeddings.weight")
        self.vocab = decoder.shape[0]
        self.rowwise, self.eps = rowwise, eps
        self.dense_bias = get(p + "transform.dense.bias")
        self.gamma, self.beta = (get(p + "transform.LayerNorm." + n).half() for n in ("weight", "bias"))
        bias = get(p + "decoder.bias", p + "bias")  # where both are there, the product's own is the one that is added
        if rowwise:
            with torch.cuda.device(dense.device):
                self.dense, self.dense_scales = ops.quantize_rows(dense)
                self.decoder, self.decoder_scales = ops.quantize_rows(decoder)
            self.bias = bias
        else:  # the FP16 product takes whole 16 columns: rows of zeros behind the vocabulary
            pad = -self.vocab % 16
            self.dense = dense.half()
            self.decoder = torch.nn.functional.pad(decoder, (0, 0, 0, pad)).half()
            self.bias = torch.nn.functional.pad(bias, (0, pad))

    def logits(self, hidden):
        """hidden: FP16 [tokens, hidden] -> [tokens, vocab], FP32 (rowwise) or FP16."""
        import torch

        from . import ops

        if self.rowwise:
            q, s = ops.quantize_rows(hidden)
            t = ops.fc_rowwise(q, s, self.dense, self.dense_scales, self.dense_bias, ops.ACT_GELU_ERF)
            _, q, s = ops.skip_layer_norm_quantize(t, None, self.gamma, self.beta, eps=self.eps, with_output=False)
            return ops.fc_rowwise(q, s, self.decoder, self.decoder_scales, self.bias, out_dtype=self.bias.dtype)
        # ops.fc goes by the type and the width of what it is given: others than the weights' would be read past the weights' end
        if hidden.dtype is not torch.float16 or hidden.dim() != 2 or hidden.shape[1] != self.dense.shape[1]:
            raise ValueError(f"hidden states must be float16 [tokens, {self.dense.shape[1]}], got {hidden.dtype} {tuple(hidden.shape)}")
        ops._here(hidden, self.dense)
        t = ops.fc(hidden, self.dense, self.dense_bias, ops.ACT_GELU_ERF)
        y, _, _ = ops.skip_layer_norm_quantize(t, None, self.gamma, self.beta, eps=self.eps)
        return ops.fc(y, self.decoder, self.bias)[:, :self.vocab]

    def __call__(self, hidden, positions=None, token_ids=None, top_k=5):
        """hidden: FP16 [total, hidden] (packed tokens); positions: the rows that are asked about (None: all), each within
        [0, total) (they are not looked at on the host); token_ids: int32 [positions, tokens] or
        [positions] -> ops.LogProbs."""
        from . import ops

        if positions is not None:
            hidden = hidden.index_select(0, positions)
        return ops.token_log_probs(self.logits(hidden.contiguous()), token_ids, top_k)
