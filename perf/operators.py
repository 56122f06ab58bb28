"""The operators around row-wise INT8 and the masked-language-model head, as cases that can be timed and compared.

Four kinds:

* quantize  - rows of activations to INT8 with a scale for each row (each token);
* fc        - the INT8 product with a scale for each row of A and each output channel, bias, erf-GELU;
* skip_ln   - residual + bias + LayerNorm whose result is also quantised row by row;
* log_probs - from a head's logits: log probabilities of given tokens, entropy, the most likely alternatives.

`run` is the plain form, elementary torch operations in 32 or 64 bits; with `own` it is the framework's operators.
"""
import math

import torch

own = False

DEV = "cuda:0"
VOCAB = 30522
TYPES = {"fp32": torch.float32, "fp16": torch.float16}
SIZE = {"fp32": 4, "fp16": 2}
EPS = 1e-12


def listed():
    return [
        # the hidden states of one short question, on their way to a projection of the large model
        {"name": "quantize_one_query", "kind": "quantize", "dtype": "fp16", "rows": 37, "width": 1024, "pad": 0},
        # a ragged FP32 batch of an odd width, rows of a wider tensor
        {"name": "quantize_fp32_odd", "kind": "quantize", "dtype": "fp32", "rows": 5001, "width": 1001, "pad": 7},
        # the feed-forward activations of 64 sequences of 384 tokens
        {"name": "quantize_ffn_64x384", "kind": "quantize", "dtype": "fp16", "rows": 24576, "width": 4096, "pad": 0},
        # output projection of one short question
        {"name": "fc_one_query", "kind": "fc", "out": "fp16", "m": 37, "n": 1024, "k": 1024, "bias": False, "gelu": False},
        # feed-forward up projection of a ragged batch
        {"name": "fc_gelu_5001", "kind": "fc", "out": "fp16", "m": 5001, "n": 4096, "k": 1024, "bias": True, "gelu": True},
        # feed-forward down projection of the throughput workload
        {"name": "fc_down_64x384", "kind": "fc", "out": "fp16", "m": 24576, "n": 1024, "k": 4096, "bias": False, "gelu": False},
        # the vocabulary's logits of the masked tokens of some sequences, in FP32
        {"name": "fc_vocabulary_fp32", "kind": "fc", "out": "fp32", "m": 640, "n": VOCAB, "k": 1024, "bias": True, "gelu": False},
        # end of a block for a few dozen tokens
        {"name": "skip_ln_one_query", "kind": "skip_ln", "dtype": "fp16", "rows": 37, "width": 1024, "bias": True},
        # end of a block of the throughput workload
        {"name": "skip_ln_64x384", "kind": "skip_ln", "dtype": "fp16", "rows": 24576, "width": 1024, "bias": True},
        # one masked token of a query: its likeliest fillers
        {"name": "log_probs_one_mask", "kind": "log_probs", "dtype": "fp16", "rows": 1, "vocab": VOCAB, "pad": 0, "tokens": 1, "top": 5},
        # some candidates scored for each masked token, FP32 logits
        {"name": "log_probs_candidates", "kind": "log_probs", "dtype": "fp32", "rows": 640, "vocab": VOCAB, "pad": 2, "tokens": 8, "top": 20},
        # 15 % of 64 x 384 tokens masked and scored against the original text
        {"name": "log_probs_corpus", "kind": "log_probs", "dtype": "fp16", "rows": 3686, "vocab": VOCAB, "pad": 6, "tokens": 1, "top": 10},
    ]


def _log(rng, lo, hi):
    """A whole number, spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A row length: half of the time a multiple of 64."""
    w = _log(rng, lo, hi)
    return max(64, w // 64 * 64) if rng.random() < 0.5 else w


def draw(rng):
    kind = rng.choice(["quantize", "fc", "fc", "skip_ln", "log_probs", "log_probs"])
    if kind == "quantize":
        while True:
            c = {"kind": kind, "dtype": rng.choice(["fp16", "fp16", "fp32"]), "rows": _log(rng, 1, 24576), "width": _width(rng, 64, 8192), "pad": rng.choice([0, 0, 3, 64])}
            if c["rows"] * c["width"] * SIZE[c["dtype"]] <= 24576 * 4096 * 2:
                return c
    if kind == "fc":
        while True:
            c = {"kind": kind, "out": rng.choice(["fp16", "fp16", "fp32"]), "m": _log(rng, 1, 24576), "n": VOCAB if rng.random() < 0.2 else _width(rng, 16, 4096),
                 "k": _width(rng, 64, 4096), "bias": rng.random() < 0.6, "gelu": rng.random() < 0.3}
            if c["m"] * c["n"] * c["k"] <= 24576 * 1024 * 4096 and c["m"] * c["n"] * SIZE[c["out"]] <= 640 * VOCAB * 4:
                return c
    if kind == "skip_ln":
        while True:
            c = {"kind": kind, "dtype": rng.choice(["fp16", "fp16", "fp32"]), "rows": _log(rng, 1, 24576), "width": _width(rng, 64, 8192), "bias": rng.random() < 0.7}
            if c["rows"] * c["width"] * SIZE[c["dtype"]] <= 24576 * 1024 * 2:
                return c
    while True:
        c = {"kind": kind, "dtype": rng.choice(["fp16", "fp32"]), "rows": _log(rng, 1, 24576), "vocab": VOCAB if rng.random() < 0.4 else _log(rng, 2, 120000),
             "pad": rng.choice([0, 0, 6, 1]), "tokens": rng.choice([1, 1, 3, 8]), "top": rng.choice([0, 1, 5, 10, 32])}
        if c["rows"] * c["vocab"] * SIZE[c["dtype"]] <= 3686 * VOCAB * 2:
            return c


def _quantised(x):
    """Rows of x to INT8 as a user's checkpoint or the layer before has them, with their scales."""
    amax = x.abs().amax(dim=1, keepdim=True)
    return torch.round(x * (127.0 / amax)).to(torch.int8), (amax / 127.0).squeeze(1).contiguous()


def _padded(x):
    """The INT8 matrix with rows that begin on 16 bytes, as quantize_rows and a checkpoint loader lay it out."""
    rows, k = x.shape
    t = torch.zeros((rows, (k + 15) // 16 * 16), dtype=x.dtype, device=x.device)
    t[:, :k] = x
    return t[:, :k]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, device=DEV, generator=g)

    def rows_of(rows, width):
        # activations: tokens differ in size, a few channels are much larger than the others
        x = normal(rows, width) * torch.exp(0.5 * normal(rows, 1))
        return x * (1 + 8 * (torch.rand((width,), device=DEV, generator=g) < 0.01))

    kind = case["kind"]
    if kind == "quantize":
        x = rows_of(case["rows"], case["width"] + case["pad"]).to(TYPES[case["dtype"]])
        return {"case": case, "x": x[:, :case["width"]]}
    if kind == "fc":
        m, n, k = case["m"], case["n"], case["k"]
        a, a_scales = _quantised(rows_of(m, k))
        w, w_scales = _quantised(0.02 * normal(n, k))
        return {"case": case, "a": _padded(a), "a_scales": a_scales, "w": _padded(w), "w_scales": w_scales, "bias": 0.02 * normal(n) if case["bias"] else None}
    if kind == "skip_ln":
        t, w = TYPES[case["dtype"]], case["width"]
        return {"case": case, "x": normal(case["rows"], w).to(t), "skip": rows_of(case["rows"], w).to(t), "gamma": (1 + 0.02 * normal(w)).to(t), "beta": (0.02 * normal(w)).to(t),
                "bias": (0.02 * normal(w)).to(t) if case["bias"] else None}
    rows, vocab = case["rows"], case["vocab"]
    x = 2.5 * normal(rows, vocab + case["pad"])
    # some tokens are sure, some are open; the first ids (padding and the like) are masked for every other row
    x.scatter_add_(1, torch.randint(0, vocab, (rows, 1), device=DEV, generator=g), 12 * torch.rand((rows, 1), device=DEV, generator=g))
    x[1::2, :vocab // 300] = -math.inf
    ids = torch.randint(0, vocab, (rows, case["tokens"]), device=DEV, generator=g, dtype=torch.int32)
    return {"case": case, "logits": x.to(TYPES[case["dtype"]])[:, :vocab], "ids": ids}


def _quantise_plain(x):
    """(values of the INT8 rows, scales): scale = amax / 127, q = 127 x / amax rounded to even, in 64 bits next to the halves between two steps."""
    amax = x.abs().amax(dim=1, keepdim=True)
    q = torch.round(x.double() * 127.0 / amax.double().clamp_min(1e-300))
    scales = amax / 127.0
    return q.float() * scales, scales.squeeze(1)


def _gelu(x):
    return 0.5 * x * (1 + torch.erf(x * 0.7071067811865476))


def _log_probs_plain(x, ids, top):
    x = x.float()
    m = x.amax(dim=1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    total = e.sum(dim=1, keepdim=True)
    lse = torch.log(total)
    entropy = (lse - (e * torch.where(e > 0, d, torch.zeros_like(d))).sum(dim=1, keepdim=True) / total).squeeze(1)
    out = [torch.gather(x, 1, ids.long()) - m - lse, entropy]
    if top:
        # one whole number for each value and place: larger values first, of equal ones the lower place
        bits = (x + 0.0).view(torch.int32)
        order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long()
        places = torch.arange(x.shape[1], device=x.device)
        key = torch.topk(order * (1 << 32) + ((1 << 32) - 1 - places), min(top, x.shape[1]), dim=1).values
        best = (1 << 32) - 1 - (key & 0xFFFFFFFF)
        value = torch.gather(x, 1, best)
        best = torch.where(torch.isneginf(value), -1, best).to(torch.int32)
        value = value - m - lse
        missing = top - best.shape[1]
        out += [torch.nn.functional.pad(best, (0, missing), value=-1), torch.nn.functional.pad(value, (0, missing), value=-math.inf)]
    return out


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        import tensorrt_b200 as T

        if kind == "quantize":
            q, scales = T.quantize_rows(s["x"])
            return [torch.mul(q, scales[:, None]), scales]
        if kind == "fc":
            return T.fc_rowwise(s["a"], s["a_scales"], s["w"], s["w_scales"], bias=s["bias"], activation=T.ACT_GELU_ERF if case["gelu"] else T.ACT_NONE, out_dtype=TYPES[case["out"]])
        if kind == "skip_ln":
            y, q, scales = T.skip_layer_norm_quantize(s["x"], s["skip"], s["gamma"], s["beta"], s["bias"], eps=EPS)
            return [y, torch.mul(q, scales[:, None], out=torch.empty_like(q, dtype=torch.float16)), scales]
        r = T.token_log_probs(s["logits"], s["ids"], top_k=case["top"])
        return [r.log_probs, r.entropy] + ([r.top_ids, r.top_log_probs] if case["top"] else [])
    if kind == "quantize":
        return list(_quantise_plain(s["x"].float()))
    if kind == "fc":
        y = torch.matmul(s["a"].float(), s["w"].float().t()) * s["a_scales"][:, None] * s["w_scales"]
        y = y if s["bias"] is None else y + s["bias"]
        return (_gelu(y) if case["gelu"] else y).to(TYPES[case["out"]])
    if kind == "skip_ln":
        v = s["x"].float() + s["skip"].float()
        v = v if s["bias"] is None else v + s["bias"].float()
        v = v - v.mean(dim=1, keepdim=True)
        y = v * torch.rsqrt((v * v).mean(dim=1, keepdim=True) + EPS) * s["gamma"].float() + s["beta"].float()
        values, scales = _quantise_plain(y)
        return [y.to(s["x"].dtype), values.half(), scales]
    return _log_probs_plain(s["logits"], s["ids"], case["top"])


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]

    def rounded_rows(x):
        most = x.abs().max(dim=1).values
        q = torch.round(127 * x / torch.where(most > 0, most, torch.ones_like(most))[:, None])
        return q * (most / 127)[:, None], most / 127

    if kind == "quantize":
        return list(rounded_rows(s["x"].to(torch.float64)))
    if kind == "fc":
        y = (s["a"].double() @ s["w"].double().T) * (s["a_scales"].double()[:, None] * s["w_scales"].double()[None, :])
        if s["bias"] is not None:
            y += s["bias"].double()[None, :]
        return y * 0.5 * torch.erfc(-y / math.sqrt(2)) if case["gelu"] else y
    if kind == "skip_ln":
        v = s["x"].double() + s["skip"].double() + (0 if s["bias"] is None else s["bias"].double())
        y = (v - v.mean(1, keepdim=True)) / torch.sqrt(v.var(1, correction=0, keepdim=True) + EPS) * s["gamma"].double() + s["beta"].double()
        values, step = rounded_rows(y)
        return [y, values, step]
    x = s["logits"].double()
    p = x - x.max(dim=1, keepdim=True).values
    p = p - torch.log(torch.exp(p).sum(dim=1, keepdim=True))
    out = [torch.gather(p, 1, s["ids"].long()), -torch.special.xlogy(torch.exp(p), torch.exp(p)).sum(dim=1)]
    if case["top"]:
        k = min(case["top"], case["vocab"])
        best = torch.full((case["rows"], case["top"]), -1, dtype=torch.int32, device=DEV)
        value = torch.full((case["rows"], case["top"]), -math.inf, dtype=torch.float64, device=DEV)
        for at in range(0, case["rows"], 256):
            v, i = torch.sort(p[at:at + 256], dim=1, descending=True, stable=True)
            value[at:at + 256, :k] = v[:, :k]
            best[at:at + 256, :k] = torch.where(torch.isneginf(v[:, :k]), -1, i[:, :k]).to(torch.int32)
        out += [best, value]
    return out


def work(case):
    kind = case["kind"]
    if kind == "quantize":
        n = case["rows"] * case["width"]
        return {"bytes": n * (SIZE[case["dtype"]] + 4) + 4 * case["rows"], "flops": 3 * n}  # the result as the values it stands for
    if kind == "fc":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + 4 * (m + n + (n if case["bias"] else 0)) + m * n * SIZE[case["out"]], "flops": 2 * m * n * k}
    if kind == "skip_ln":
        n = case["rows"] * case["width"]
        return {"bytes": n * (3 * SIZE[case["dtype"]] + 2) + 4 * case["rows"] + 3 * case["width"] * SIZE[case["dtype"]], "flops": 10 * n}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * SIZE[case["dtype"]] + case["rows"] * (8 * case["tokens"] + 4 + 8 * case["top"]), "flops": 6 * n}
