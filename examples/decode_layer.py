"""One decoder layer on the GPU, a prompt and then single tokens: attention over the paged cache next to the FFN.

    python examples/decode_layer.py [--tokens 8] [--cache i8|f16|bf16]

The layer is x <- x + O(attention(QKV(norm x))), then x <- x + FFN(norm x), with seeded Q8_0 weights:
the projections run as ``gemv_dev``, keys and values go into the pages with ``kv_append_dev``,
``attn_paged_dev`` reads them, and ``ffn_stack_dev`` is the rest.  Queries, keys and values are
slices of one projection's rows.  At the end the layer is computed again in 64 bits from the
dequantised weights, all tokens at once and without a cache, and the largest deviation is printed.
"""
from __future__ import annotations

import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import hayai_b200 as hb  # noqa: E402

HEADS, KV_HEADS, DIM, D_FF, PAGE = 8, 2, 64, 1024, 16
D_MODEL = HEADS * DIM


def q8_0(rng, m: int, n: int):
    """Seeded Q8_0 blocks (f16 scale, 32 codes) of an m x n matrix, and their values."""
    w = rng.normal(0.0, 0.05, (m * n // 32, 32)).astype(np.float32)
    d = (np.abs(w).max(1) / 127).astype(np.float16)
    codes = np.clip(np.rint(w / d[:, None].astype(np.float32)), -127, 127).astype(np.int8)
    raw = np.concatenate([d.view(np.uint8).reshape(-1, 2), codes.view(np.uint8)], 1)
    return raw, (codes * d[:, None].astype(np.float64)).reshape(m, n)


class Layer:
    """The layer's weights and its cache: one pool of pages that the sequences share."""

    def __init__(self, engine, n_pages: int, cache: str, seed: int = 0):
        rng = np.random.default_rng(seed)
        shapes = {"qkv": ((HEADS + 2 * KV_HEADS) * DIM, D_MODEL), "out": (D_MODEL, HEADS * DIM),
                  "gate": (D_FF, D_MODEL), "up": (D_FF, D_MODEL), "down": (D_MODEL, D_FF)}
        self.engine, self.w, self.exact = engine, {}, {}
        for name, (m, n) in shapes.items():
            raw, self.exact[name] = q8_0(rng, m, n)
            self.w[name] = engine.upload(hb.Q8_0, m, n, raw)
        dtype = {"i8": torch.int8, "f16": torch.float16, "bf16": torch.bfloat16}[cache]
        pool = lambda: torch.zeros(n_pages, KV_HEADS, PAGE, DIM, dtype=dtype, device="cuda")  # noqa: E731
        scale = lambda: torch.zeros(n_pages, KV_HEADS, PAGE, device="cuda") if cache == "i8" else None  # noqa: E731
        self.cache = hb.KvCache(pool(), pool(), scale(), scale())
        self.norm = torch.ones(D_MODEL, device="cuda")

    def step(self, x, batch):
        """x [n_tok][D_MODEL] float32: the batch's new tokens, in place."""
        e, n = self.engine, x.shape[0]
        xn = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-5)
        qkv = torch.empty(n, HEADS + 2 * KV_HEADS, DIM, device="cuda")
        e.gemv_dev(self.w["qkv"], xn, qkv.view(n, -1), nvec=n)
        q, k, v = qkv[:, :HEADS], qkv[:, HEADS:HEADS + KV_HEADS], qkv[:, HEADS + KV_HEADS:]
        e.kv_append_dev(self.cache, batch, k, v)
        att = torch.empty(n, HEADS, DIM, device="cuda")
        e.attn_paged_dev(self.cache, batch, q, att)
        e.gemv_dev(self.w["out"], att.view(n, -1), x, resid=x, nvec=n)
        e.ffn_stack_dev([self.w["gate"]], [self.w["up"]], [self.w["down"]], x, nvec=n, norms=[self.norm])

    def reference(self, x):
        """The layer over the whole sequence x [n][D_MODEL] in 64 bits."""
        w, n = self.exact, x.shape[0]
        norm = lambda t: t / np.sqrt((t * t).mean(-1, keepdims=True) + 1e-5)  # noqa: E731
        qkv = (norm(x) @ w["qkv"].T).reshape(n, -1, DIM)
        q, k, v = qkv[:, :HEADS], qkv[:, HEADS:HEADS + KV_HEADS], qkv[:, HEADS + KV_HEADS:]
        att = np.zeros((n, HEADS, DIM))
        for h in range(HEADS):
            g = h // (HEADS // KV_HEADS)
            s = np.where(np.tri(n, dtype=bool), q[:, h] @ k[:, g].T / np.sqrt(DIM), -np.inf)
            p = np.exp(s - s.max(-1, keepdims=True))
            att[:, h] = p / p.sum(-1, keepdims=True) @ v[:, g]
        x = x + att.reshape(n, -1) @ w["out"].T
        a, u = norm(x) @ w["gate"].T, norm(x) @ w["up"].T
        return x + (a / (1 + np.exp(-a)) * u) @ w["down"].T


def run(tokens: int = 8, cache: str = "i8", prompts=(37, 5, 130)) -> float:
    """Prompts of three sequences in one step, then `tokens` single-token steps; returns the largest
    deviation from the 64-bit layer, relative to the outputs' root mean square."""
    engine = hb.CudaEngine(0)
    engine.set_stream(torch.cuda.current_stream())
    n_seq, most = len(prompts), max(prompts) + tokens
    per_seq = -(-most // PAGE)
    layer = Layer(engine, n_seq * per_seq, cache)
    # the allocator's part: pages in no order
    order = torch.randperm(n_seq * per_seq, generator=torch.Generator().manual_seed(1))
    table = order.view(n_seq, per_seq).to(torch.int32).cuda()
    rng = np.random.default_rng(7)
    inputs = [rng.normal(size=(p + tokens, D_MODEL)) for p in prompts]
    outputs = [[] for _ in prompts]
    done = [0] * n_seq
    for new in [list(prompts)] + [[1] * n_seq] * tokens:
        x = np.concatenate([a[d:d + n] for a, d, n in zip(inputs, done, new)])
        done = [d + n for d, n in zip(done, new)]
        start = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32).cuda()
        batch = hb.KvBatch(table, start, torch.tensor(done, dtype=torch.int32).cuda(), sum(new), max(new))
        xd = torch.from_numpy(x.astype(np.float32)).cuda()
        layer.step(xd, batch)
        engine.sync()
        for out, part in zip(outputs, np.split(xd.double().cpu().numpy(), np.cumsum(new)[:-1])):
            out.append(part)
    worst = 0.0
    for a, out in zip(inputs, outputs):
        ref = layer.reference(a.astype(np.float32).astype(np.float64))
        worst = max(worst, np.abs(np.concatenate(out) - ref).max() / np.sqrt((ref * ref).mean()))
    engine.close()
    return float(worst)


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--tokens", type=int, default=8)
    ap.add_argument("--cache", choices=["i8", "f16", "bf16"], default="i8")
    args = ap.parse_args()
    print(f"largest deviation from the 64-bit layer: {run(args.tokens, args.cache):.2e} of the outputs' rms")
