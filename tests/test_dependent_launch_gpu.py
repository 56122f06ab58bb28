"""Kernels that start before the kernel ahead of them has ended give the bits that they give one after the other (BERT_B200_PDL=0)."""
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parent.parent

SCRIPT = r"""
import sys
sys.path.insert(0, ".")
import torch
import tensorrt_b200 as T
from tensorrt_b200 import synthetic

d = "cuda:0"
out = {}


def several(name, call, calls):
    # each call's results while the ones before are still running, on memory that holds other values
    for i in range(calls):
        out[f"{name} {i}"] = [t.clone() for t in call(i) if t is not None]


for layers, hidden, heads, ffn in ((4, 768, 12, 3072), (3, 1024, 16, 4096), (3, 256, 4, 1024), (2, 512, 8, 2048), (2, 128, 2, 512)):
    p = synthetic.make_params(layers, hidden, heads, ffn, vocab=2000, device=d)
    batches = [synthetic.make_inputs(b, s, vocab=2000, seed=s, min_len=m, device=d) + (s,) for b, s, m in ((1, 37, None), (8, 384, 32), (3, 128, 1), (24, 384, None))]
    fp16 = T.BertEncoder(p, T.FP16, d)
    synthetic.assign_int8_scales(p, fp16.calibrate(*batches[1][:3], batches[1][4]))
    encoders = {"fp16": fp16, "int8": T.BertEncoder(p, T.INT8, d), "rowwise": T.BertEncoder(p, T.INT8, d, rowwise=True)}
    for kind, e in encoders.items():
        several(f"{kind} {hidden}", lambda i: [e.forward(*batches[i % 4][:3], batches[i % 4][4])], 12)
        assert e.status_word() == 0

g = torch.Generator(device=d).manual_seed(0)
rnd = lambda *s: torch.randn(s, device=d, generator=g)
for dtype in (torch.float16, torch.float32):
    for rows in (1, 37, 300, 1700):
        for width in (64, 250, 256, 512, 768, 1024, 1001, 2048, 4096):
            x, w = [rnd(rows, width).to(dtype) for _ in range(4)], 0.05 * rnd(304, width)
            w8, ws = T.quantize_rows(w)
            gamma, beta, bias = (1 + 0.1 * rnd(width)).to(dtype), rnd(width).to(dtype), rnd(width).to(dtype)
            eps = 0.0 if dtype == torch.float16 else 1.1920929e-7
            ids = torch.randint(0, 304, (rows, 2), device=d, generator=g).int()

            def chain(i):
                a = x[i % 4]
                y = T.skip_layer_norm(a, a, gamma, beta, bias)
                y, q, s = T.skip_layer_norm_quantize(y, a, gamma, beta, bias, eps=eps)
                q2, s2 = T.quantize_rows(y)
                z = T.fc_rowwise(q2, s2, w8, ws, None, T.ACT_GELU_ERF, out_dtype=dtype)
                r = T.token_log_probs(z, ids, top_k=4)
                if width % 16 == 0:
                    v = T.fc_rowwise(q, s, w8, ws, out_dtype=torch.float32)
                    return [y, q, s, q2, s2, z, *r, *T.token_log_probs(v, ids, top_k=20)]
                return [y, q, s, q2, s2, z, *r]

            several(f"chain {dtype} {rows} {width}", chain, 6)
    # products in floating point, attention and lengths that the kernels ahead have just written
    for B, S, N in ((1, 37, 4), (6, 200, 4), (3, 130, 8)):
        E = N * 64
        x = [0.3 * rnd(B * S, E).to(dtype) for _ in range(3)]
        wq, wo = (0.05 * rnd(3 * E, E).to(dtype) for _ in range(2))
        mask = torch.ones((S, B), dtype=torch.int32, device=d)
        mask[S // 2:, ::2] = 0

        def layer(i):
            a = x[i % 3]
            qkv = T.fc(a, wq)
            idx = T.compute_mask_idx(mask)
            c = T.mha(qkv.view(S, B, 3 * E), B, S, N, mask_idx=idx)
            y = T.fc(a, wo, None, T.ACT_GELU_ERF)
            return [qkv, idx, c, y, T.skip_layer_norm(y[:, :E].contiguous(), a, wq[0], wq[1])]

        several(f"layer {dtype} {B}", layer, 6)
torch.cuda.synchronize()
torch.save({k: [t.cpu() for t in v] for k, v in out.items()}, sys.argv[1])
"""


def test_starting_early_changes_no_bit(cuda, tmp_path):
    got = {}
    for pdl in ("0", "1"):
        file = tmp_path / f"{pdl}.pt"
        r = subprocess.run([sys.executable, "-c", SCRIPT, str(file)], cwd=ROOT, env={**os.environ, "BERT_B200_PDL": pdl}, capture_output=True, text=True, timeout=600)
        assert r.returncode == 0, r.stderr[-3000:]
        got[pdl] = torch.load(file)
    assert got["0"].keys() == got["1"].keys() and len(got["0"]) > 500
    bits = lambda t: t.view({1: torch.int8, 2: torch.int16, 4: torch.int32}[t.element_size()])
    wrong = [k for k in got["0"] if not all(torch.equal(bits(a), bits(b)) for a, b in zip(got["0"][k], got["1"][k]))]
    assert not wrong, wrong
