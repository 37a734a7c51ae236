"""Many continuations of one prompt through a decoder layer's attention, on the GPU.

    python examples/continuations.py [--continuations 6] [--tokens 5] [--cache i8|f16|bf16]

A prompt's queries, keys and values (a seeded Q8_0 projection of its rows) are turned by their positions and
stored (``kv_append_rope_dev``), the prompt is forked (``kv_fork_dev``), and every continuation gets a token a
step: the pool grows (``kv_resize_dev``), the token is turned and stored, and attends with ``attn_shared_dev``,
which may read the prompt once for all of them.  Half way, every other continuation is let go and the pool is
compacted (``kv_compact_dev``).  At the end all of it is computed again in 64 bits, without a cache, and the
largest deviation is printed.
"""
from __future__ import annotations

import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import hayai_b200 as hb  # noqa: E402
from examples.decode_layer import q8_0  # noqa: E402

HEADS, KV_HEADS, DIM, PAGE, BASE = 8, 2, 64, 16, 500000.0
D_MODEL = HEADS * DIM


def ints(v):
    return torch.tensor(v, dtype=torch.int32).cuda()


def exact(x, w):
    """Attention of rows x [n][D_MODEL] over themselves, causal, in 64 bits: [n][HEADS][DIM]."""
    n = len(x)
    qkv = (x @ w.T).reshape(n, -1, DIM)
    angle = np.arange(n)[:, None] * BASE ** (-np.arange(DIM // 2) / (DIM // 2))
    z = (qkv[:, :HEADS + KV_HEADS, :DIM // 2] + 1j * qkv[:, :HEADS + KV_HEADS, DIM // 2:]) * np.exp(1j * angle)[:, None]
    turned = np.concatenate([z.real, z.imag], -1)
    q, k, v = turned[:, :HEADS], turned[:, HEADS:], qkv[:, HEADS + KV_HEADS:]
    out = np.zeros((n, HEADS, DIM))
    for h in range(HEADS):
        g = h // (HEADS // KV_HEADS)
        s = np.where(np.tri(n, dtype=bool), q[:, h] @ k[:, g].T / np.sqrt(DIM), -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        out[:, h] = p / p.sum(-1, keepdims=True) @ v[:, g]
    return out


def run(continuations: int = 6, tokens: int = 5, cache: str = "i8", prompt: int = 77) -> float:
    """Returns the largest deviation from 64 bits, relative to the results' root mean square."""
    engine = hb.CudaEngine(0)
    engine.set_stream(torch.cuda.current_stream())
    rng = np.random.default_rng(3)
    raw, w = q8_0(rng, (HEADS + 2 * KV_HEADS) * DIM, D_MODEL)
    project = engine.upload(hb.Q8_0, *w.shape, raw)
    slots, per_slot = continuations + 1, -(-(prompt + tokens) // PAGE)
    n_pages = slots * per_slot
    dtype = {"i8": torch.int8, "f16": torch.float16, "bf16": torch.bfloat16}[cache]
    pool = lambda: torch.zeros(n_pages, KV_HEADS, PAGE, DIM, dtype=dtype, device="cuda")  # noqa: E731
    scale = lambda: torch.zeros(n_pages, KV_HEADS, PAGE, device="cuda") if cache == "i8" else None  # noqa: E731
    layer = hb.KvCache(pool(), pool(), scale(), scale())
    table, kv_len, refs = (torch.zeros(s, dtype=torch.int32, device="cuda") for s in ((slots, per_slot), slots, n_pages))
    pages = hb.KvPages([layer], table, kv_len, refs)
    rope = hb.Rope(DIM, base=BASE)
    # slot 0 is the prompt, and all slots behind it may continue it
    shared = hb.KvShared(ints([0, slots]), ints([prompt]), least=1)
    rows = [rng.normal(size=(prompt, D_MODEL))] + [None] * continuations
    out = [[] for _ in range(slots)]

    def step(live, new):
        """Tokens new [n][D_MODEL] of every live slot, the same number each."""
        n, each = sum(len(x) for x in new), len(new[0])
        x = torch.from_numpy(np.concatenate(new).astype(np.float32)).cuda()
        engine.kv_resize_dev(pages, ints(live), kv_len[torch.tensor(live).cuda()] + each)
        counts = [each if s in live else 0 for s in range(slots)]
        batch = hb.KvBatch(table, ints(np.concatenate([[0], np.cumsum(counts)])), kv_len, n, each)
        qkv = torch.empty(n, HEADS + 2 * KV_HEADS, DIM, device="cuda")
        engine.gemv_dev(project, x, qkv.view(n, -1), nvec=n)
        q, k, v = qkv[:, :HEADS], qkv[:, HEADS:HEADS + KV_HEADS], qkv[:, HEADS + KV_HEADS:]
        engine.kv_append_rope_dev(layer, batch, rope, q, k, v)
        att = torch.empty(n, HEADS, DIM, device="cuda")
        engine.attn_shared_dev(layer, batch, shared, q, att)
        engine.sync()
        for s, part in zip(live, np.split(att.double().cpu().numpy(), len(live))):
            out[s].append(part)

    step([0], [rows[0]])
    children = list(range(1, slots))
    engine.kv_fork_dev(pages, ints([0] * continuations), ints(children))
    for s in children:
        rows[s], out[s] = rows[0], list(out[0])
    for t in range(tokens):
        if t == tokens // 2 and t:
            engine.kv_resize_dev(pages, ints(children[1::2]), ints([0] * len(children[1::2])))
            engine.kv_compact_dev(pages)
            children = children[::2]
        new = [rng.normal(size=(1, D_MODEL)) for _ in children]
        for s, x in zip(children, new):
            rows[s] = np.concatenate([rows[s], x])
        step(children, new)
    worst = 0.0
    for s in range(slots):
        ref = exact(rows[s].astype(np.float32).astype(np.float64), w)
        worst = max(worst, np.abs(np.concatenate(out[s]) - ref).max() / np.sqrt((ref * ref).mean()))
    project.free()
    engine.close()
    return float(worst)


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--continuations", type=int, default=6)
    ap.add_argument("--tokens", type=int, default=5)
    ap.add_argument("--cache", choices=["i8", "f16", "bf16"], default="i8")
    args = ap.parse_args()
    print(f"largest deviation from 64 bits: {run(args.continuations, args.tokens, args.cache):.2e} of the results' rms")
