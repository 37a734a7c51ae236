"""Cases of the paged key/value cache and of the attention over it, for timing and comparison.

Three operators, each over a batch of sequences of which every one has ``kv`` tokens in the cache,
the last ``new`` of them being the tokens of this step:

  write   store the step's key and value rows in the cache's pages (16-bit, or 8-bit codes with one
          scale for each token and head).  A 16-bit cache is returned as it stands; of an 8-bit one
          the rows just written are read back, so that the values they stand for are returned
  read    gather rows of the cache back into packed rows, as the values that they stand for
  attend  attention of the step's query rows over the cache: causal, with shared heads, and where
          asked with a window of recent tokens and a few first tokens that stay visible

``run`` computes them in elementary torch operations in 32 bits, or, where ``own`` is true, by the
calls that a program makes of hayai_b200.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}


def listed():
    return [
        # One token of one conversation enters a layer's cache (8 kv heads of 128): launch latency.
        dict(name="write-1-f32-bf16", op="write", x="f32", cache="bf16", heads=8, kv_heads=8, dim=128, page=16,
             seqs=1, new_lo=1, new_hi=1, ctx_lo=999, ctx_hi=999, single=0.0, lens=1),
        # A step of a server: decoding sequences beside short prompts, 3 kv heads of 64.
        dict(name="write-ragged-f32-f16", op="write", x="f32", cache="f16", heads=3, kv_heads=3, dim=64, page=16,
             seqs=37, new_lo=1, new_hi=301, ctx_lo=1, ctx_hi=2000, single=0.5, lens=2),
        # 256 decoding sequences, one token each, into an 8-bit cache, and the rows read back.
        dict(name="write-256-f32-i8", op="write", x="f32", cache="i8", heads=8, kv_heads=8, dim=128, page=16,
             seqs=256, new_lo=1, new_hi=1, ctx_lo=30, ctx_hi=1500, single=0.0, lens=3),
        # Nine prompts of a few thousand tokens into an 8-bit cache, and the rows read back.
        dict(name="write-prompts-bf16-i8", op="write", x="bf16", cache="i8", heads=8, kv_heads=8, dim=128, page=64,
             seqs=9, new_lo=2500, new_hi=5000, ctx_lo=1, ctx_hi=500, single=0.0, lens=4),
        # A prefix leaves the cache (moved to another worker, or kept on the host): all its rows.
        dict(name="read-prefix-i8-bf16", op="read", x="bf16", cache="i8", heads=8, kv_heads=8, dim=128, page=64,
             seqs=8, new_lo=2000, new_hi=6000, ctx_lo=0, ctx_hi=0, single=0.0, lens=5),
        # Short pieces of many conversations, 4 kv heads of 128.
        dict(name="read-ragged-bf16-f32", op="read", x="f32", cache="bf16", heads=4, kv_heads=4, dim=128, page=32,
             seqs=19, new_lo=1, new_hi=700, ctx_lo=0, ctx_hi=300, single=0.1, lens=6),
        # One user's next token at a context of a thousand (32 query heads on 8): latency.
        dict(name="decode-1-f32-i8", op="attend", x="f32", cache="i8", heads=32, kv_heads=8, dim=128, page=16,
             seqs=1, new_lo=1, new_hi=1, ctx_lo=1000, ctx_hi=1000, single=0.0, window=0, sink=0, lens=7),
        # A server's decode step: 64 sequences of very different lengths (64 heads on 8), 8-bit cache.
        dict(name="decode-64-bf16-i8", op="attend", x="bf16", cache="i8", heads=64, kv_heads=8, dim=128, page=64,
             seqs=64, new_lo=1, new_hi=1, ctx_lo=300, ctx_hi=12000, single=0.0, window=0, sink=0, lens=8),
        # One very long document: 131071 cached tokens, 32 heads on 4; the work has to be split.
        dict(name="decode-long-f16-f16", op="attend", x="f16", cache="f16", heads=32, kv_heads=4, dim=128, page=64,
             seqs=1, new_lo=1, new_hi=1, ctx_lo=131070, ctx_hi=131070, single=0.0, window=0, sink=0, lens=9),
        # Prompts from their first token on, 32 heads on 8, 16-bit cache: the tensor cores' case.
        dict(name="prompt-4-bf16-bf16", op="attend", x="bf16", cache="bf16", heads=32, kv_heads=8, dim=128, page=64,
             seqs=4, new_lo=2000, new_hi=4100, ctx_lo=0, ctx_hi=0, single=0.0, window=0, sink=0, lens=10),
        # Chunks of long prompts over what is cached of them, 8-bit cache.
        dict(name="chunk-4-f16-i8", op="attend", x="f16", cache="i8", heads=32, kv_heads=8, dim=128, page=32,
             seqs=4, new_lo=512, new_hi=512, ctx_lo=3000, ctx_hi=15000, single=0.0, window=0, sink=0, lens=11),
        # A mixed step in 32 bits, decoding sequences beside chunks, with a window and first tokens
        # kept (9 heads on 3, of 64).
        dict(name="mixed-f32-i8-window", op="attend", x="f32", cache="i8", heads=9, kv_heads=3, dim=64, page=16,
             seqs=24, new_lo=1, new_hi=1500, ctx_lo=1, ctx_hi=9000, single=0.5, window=2048, sink=4, lens=12),
    ]


def _lens(case):
    """(new, kv) of every sequence: the step's tokens, and all tokens with them."""
    r = random.Random(case["lens"])
    new, kv = [], []
    for _ in range(case["seqs"]):
        n = 1 if r.random() < case["single"] else _log(r, case["new_lo"], case["new_hi"])
        c = _log(r, case["ctx_lo"], case["ctx_hi"])
        new.append(n)
        kv.append(n + c)
    return new, kv


def _log(r, lo, hi):
    """A whole number in [lo, hi], spread over the logarithm."""
    return lo if lo == hi else min(hi, int(math.exp(r.uniform(math.log(lo + 1), math.log(hi + 2)))) - 1)


def _visible(new, kv, window, sink):
    """(query, key) pairs of one sequence that attention has to look at, and keys that any query sees."""
    first = kv - new
    if not window:
        return new * first + new * (new + 1) // 2, kv
    pairs, low = 0, max(0, first - window + 1)
    for p in range(first, kv):
        recent = min(p + 1, window)
        pairs += recent + min(sink, p + 1 - recent)
    return pairs, kv - low + min(sink, low)


def work(case):
    new, kv = _lens(case)
    rows, dim, hk = sum(new), case["dim"], case["kv_heads"]
    cached = 2 * hk * (dim * SIZE[case["cache"]] + (4 if case["cache"] == "i8" else 0))  # bytes of a token
    if case["op"] == "write":
        given = rows * 2 * hk * dim * SIZE[case["x"]]
        if case["cache"] == "i8":  # and read back
            return {"bytes": 2 * (given + rows * cached), "flops": 0}
        return {"bytes": given + rows * cached, "flops": 0}
    if case["op"] == "read":
        return {"bytes": rows * (cached + 2 * hk * dim * SIZE[case["x"]]), "flops": 0}
    seen = [_visible(n, k, case["window"], case["sink"]) for n, k in zip(new, kv)]
    heads = case["heads"]
    return {"bytes": sum(k for _, k in seen) * cached + rows * heads * (2 * dim * SIZE[case["x"]] + 4),
            "flops": 4 * dim * heads * sum(p for p, _ in seen)}


def draw(rng):
    op = rng.choice(["write", "read", "attend", "attend", "attend"])
    cache = rng.choice(["f16", "bf16", "i8", "i8"])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 8]) if op == "attend" else 1
    c = dict(op=op, x=rng.choice(["f32", "f16", "bf16"]), cache=cache, heads=kv_heads * group, kv_heads=kv_heads,
             dim=rng.choice([64, 128, 128]), page=rng.choice([16, 16, 24, 32, 64, 100, 128]),
             lens=rng.randrange(1 << 30))
    if op != "attend":
        c |= dict(seqs=_log(rng, 1, 64), new_lo=1, new_hi=_log(rng, 1, 5000), ctx_lo=0, ctx_hi=_log(rng, 1, 2000),
                  single=rng.choice([0.0, 0.5]))
    else:
        kind = rng.choice(["decode", "decode", "chunk", "mixed"])
        c |= dict(window=0, sink=0, single={"decode": 1.0, "chunk": 0.0, "mixed": 0.6}[kind], new_lo=1,
                  seqs=_log(rng, 1, 64) if kind != "chunk" else _log(rng, 1, 6),
                  new_hi=1 if kind == "decode" else _log(rng, 2, 3000 if kind == "chunk" else 400),
                  ctx_lo=0, ctx_hi=_log(rng, 10, 100000 if kind == "decode" else 12000))
        if rng.random() < 0.3:
            c |= dict(window=_log(rng, 16, 4096), sink=rng.choice([0, 1, 4, 100]))
    most = [work(k) for k in listed() if (k["op"] == "attend") == (op == "attend")]
    top = {k: max(m[k] for m in most) for k in ("bytes", "flops")}
    while True:
        w = work(c)
        new, kv = _lens(c)
        padded = c["seqs"] * max(new) * max(kv) * c["heads"]
        if w["bytes"] <= top["bytes"] and w["flops"] <= top["flops"] and (op != "attend" or padded <= 2.5e9) and \
                c["seqs"] * max(kv) * kv_heads * c["dim"] <= 6e8:
            return c
        if c["seqs"] > 1:
            c["seqs"] = c["seqs"] // 2 + c["seqs"] % 2 * (c["seqs"] > 2)
        else:
            c["new_hi"], c["ctx_hi"] = max(1, c["new_hi"] * 3 // 4), max(1, c["ctx_hi"] * 3 // 4)


def prepare(case, seed):
    """The cache's pages, the batch's page table and lengths, and the step's rows, on the GPU."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    new, kv = _lens(case)
    page, hk, dim, rows = case["page"], case["kv_heads"], case["dim"], sum(new)
    need = [-(-k // page) for k in kv]
    n_pages = sum(need) + 3
    order = torch.randperm(n_pages, generator=g, device=DEV, dtype=torch.int32)[:sum(need)]
    table = torch.zeros(len(kv), max(need), dtype=torch.int32, device=DEV)
    at = torch.arange(max(need), device=DEV)[None, :] < torch.tensor(need, device=DEV)[:, None]
    table[at] = order
    s = dict(case=case, table=table, page=page,
             q_start=torch.tensor([0] + new, device=DEV).cumsum(0).to(torch.int32),
             kv_len=torch.tensor(kv, dtype=torch.int32, device=DEV), n_tok=rows, max_new=max(new), max_kv=max(kv))
    pools = {}
    for which in ("k", "v"):
        shape = (n_pages, hk, page, dim)
        if case["op"] == "write":  # rows of earlier steps are not looked at: an empty cache
            pools[which] = torch.zeros(shape, dtype=TYPES[case["cache"]], device=DEV)
            pools[which + "_scale"] = torch.zeros(shape[:3], device=DEV) if case["cache"] == "i8" else None
            continue
        x = torch.randn(shape, generator=g, device=DEV)
        if which == "k":  # keys have a few strong channels
            x[..., :: dim // 4] *= 3.0
        if case["cache"] == "i8":
            pools[which], pools[which + "_scale"] = _quantised(x)
        else:
            pools[which], pools[which + "_scale"] = x.to(TYPES[case["cache"]]), None
    s |= pools
    xt = TYPES[case["x"]]
    if case["op"] == "attend":
        s["q"] = torch.randn(rows, case["heads"], dim, generator=g, device=DEV).to(xt)
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(rows, case["heads"], device=DEV)
    else:
        s["k_rows"], s["v_rows"] = (torch.empty(rows, hk, dim, dtype=xt, device=DEV) for _ in range(2))
        if case["op"] == "write":
            for t in ("k_in", "v_in"):
                s[t] = torch.randn(rows, hk, dim, generator=g, device=DEV).to(xt)
    if own:  # the handles that a program keeps beside its tensors
        s["engine"] = _engine()
        import hayai_b200 as hb
        s["cache"] = hb.KvCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
        s["batch"] = hb.KvBatch(table, s["q_start"], s["kv_len"], rows, s["max_new"])
    return s


_engines = []


def _engine():
    if not _engines:
        import hayai_b200 as hb
        e = hb.CudaEngine(0)
        e.set_stream(torch.cuda.current_stream())
        _engines.append(e)
    return _engines[0]


def run(s):
    if own:
        return _run_own(s)
    op = s["case"]["op"]
    if op == "attend":
        return _attend(s)
    if op == "read":
        return _read(s)
    page, row, _ = _slots(s)
    for x, which in (("k_in", "k"), ("v_in", "v")):
        v = s[x].float()
        if s["case"]["cache"] == "i8":
            codes, scale = _quantised(v)
            s[which][page, :, row] = codes
            s[which + "_scale"][page, :, row] = scale
        else:
            s[which][page, :, row] = v.to(s[which].dtype)
    return _read(s) if s["case"]["cache"] == "i8" else [s["k"], s["v"]]


def _run_own(s):
    e, cache, batch, c = s["engine"], s["cache"], s["batch"], s["case"]
    if c["op"] == "attend":
        e.attn_paged_dev(cache, batch, s["q"], s["out"], window=c["window"], sink=c["sink"], lse=s["lse"])
        return [s["out"], s["lse"]]
    if c["op"] == "write":
        e.kv_append_dev(cache, batch, s["k_in"], s["v_in"])
        if c["cache"] != "i8":
            return [s["k"], s["v"]]
    e.kv_read_dev(cache, batch, s["k_rows"], s["v_rows"])
    return [s["k_rows"], s["v_rows"]]


# ------------------------------------------------------------------ the plain form
def _quantised(x):
    """8-bit codes and the scale of each last-axis row: scale = max|x| / 127, code = x / scale rounded
    to the nearest, ties to even."""
    scale = x.abs().amax(-1) / 127.0
    codes = torch.where(scale[..., None] > 0, (x / scale[..., None]).round().clamp(-127, 127), torch.zeros_like(x))
    return codes.to(torch.int8), scale


def _slots(s):
    """Page, row in the page and sequence of each of the step's tokens."""
    start, kv = s["q_start"].long(), s["kv_len"].long()
    t = torch.arange(s["n_tok"], device=DEV)
    seq = torch.searchsorted(start, t, right=True) - 1
    pos = kv[seq] - start[seq + 1] + t
    return s["table"][seq, pos // s["page"]].long(), pos % s["page"], seq


def _read(s):
    page, row, _ = _slots(s)
    out = []
    for which in ("k", "v"):
        x = s[which][page, :, row].float()
        if s[which + "_scale"] is not None:
            x = x * s[which + "_scale"][page, :, row][..., None]
        out.append(x.to(TYPES[s["case"]["x"]]))
    return out


def _attend(s):
    c = s["case"]
    hk, dim = c["kv_heads"], c["dim"]
    group = c["heads"] // hk
    n, most_q, most_k = len(s["kv_len"]), s["max_new"], s["max_kv"]
    key = torch.arange(most_k, device=DEV)
    page, row = s["table"][:, key // s["page"]].long(), (key % s["page"])[None, :]
    kv = []
    for which in ("k", "v"):
        x = s[which][page, :, row].float()  # [n, most_k, hk, dim]
        if s[which + "_scale"] is not None:
            x = x * s[which + "_scale"][page, :, row][..., None]
        kv.append(x.transpose(1, 2))
    _, _, seq = _slots(s)
    start, length = s["q_start"].long(), s["kv_len"].long()
    t = torch.arange(s["n_tok"], device=DEV)
    at = t - start[seq]
    q = torch.zeros(n, most_q, c["heads"], dim, device=DEV)
    q[seq, at] = s["q"].float()
    q = q.view(n, most_q, hk, group, dim).permute(0, 2, 3, 1, 4).reshape(n, hk, group * most_q, dim)
    scores = torch.matmul(q, kv[0].transpose(2, 3)).mul_(1.0 / math.sqrt(dim)).view(n, hk, group, most_q, most_k)
    where = torch.arange(most_q, device=DEV)[None, :, None] + (length - start.diff())[:, None, None]
    seen = (key <= where) & (key < length[:, None, None])
    if c["window"]:
        seen &= (where - key < c["window"]) | (key < c["sink"])
    seen = seen[:, None, None]
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top > -math.inf, top, torch.zeros_like(top))
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(n, hk, group * most_q, most_k), kv[1]).view(n, hk, group, most_q, dim)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    lse = (top + total.log()).squeeze(-1)
    out = out.permute(0, 3, 1, 2, 4).reshape(n, most_q, c["heads"], dim)[seq, at]
    lse = lse.permute(0, 3, 1, 2).reshape(n, most_q, c["heads"])[seq, at]
    return [out.to(TYPES[c["x"]]), lse]


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """The operators' definition in 64 bits, one sequence (and for attention one kv head) at a time."""
    s = prepare(case, seed)
    new, kv = _lens(case)
    page = case["page"]

    def rows_of(which, i, lo, hi):
        pos = torch.arange(lo, hi, device=DEV)
        p, r = s["table"][i].long()[torch.div(pos, page, rounding_mode="floor")], pos.remainder(page)
        x = s[which][p, :, r].double()
        scale = s[which + "_scale"]
        return x if scale is None else x * scale[p, :, r].double().unsqueeze(-1)

    if case["op"] == "write":
        outs = []
        if case["cache"] == "i8":
            for t in ("k_in", "v_in"):
                x = s[t].double()
                step = x.abs().max(-1, keepdim=True).values / 127
                outs.append(torch.round(x / torch.where(step == 0, 1.0, step)) * step)
            return outs
        for t, which in (("k_in", "k"), ("v_in", "v")):
            pool = s[which].double()
            done = 0
            for i, (n, k) in enumerate(zip(new, kv)):
                pos = torch.arange(k - n, k, device=DEV)
                pool[s["table"][i].long()[pos // page], :, pos % page] = s[t][done:done + n].double()
                done += n
            outs.append(pool)
        return outs
    if case["op"] == "read":
        return [torch.cat([rows_of(w, i, k - n, k) for i, (n, k) in enumerate(zip(new, kv))]) for w in ("k", "v")]
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device=DEV)
    done = 0
    for i, (n, k) in enumerate(zip(new, kv)):
        K, V = rows_of("k", i, 0, k), rows_of("v", i, 0, k)
        i_pos = torch.arange(k - n, k, device=DEV).view(n, 1, 1)
        j_pos = torch.arange(k, device=DEV).view(1, 1, k)
        hidden = j_pos > i_pos
        if case["window"]:
            hidden = hidden | ((j_pos <= i_pos - case["window"]) & (j_pos >= case["sink"]))
        for h in range(case["kv_heads"]):
            q = s["q"][done:done + n, h * group:(h + 1) * group].double()
            a = torch.einsum("ngd,kd->ngk", q, K[:, h]) / math.sqrt(case["dim"])
            a = a.masked_fill(hidden, -math.inf)
            log_sum = torch.logsumexp(a, -1)
            out[done:done + n, h * group:(h + 1) * group] = torch.einsum("ngk,kd->ngd", (a - log_sum[..., None]).exp(), V[:, h])
            lse[done:done + n, h * group:(h + 1) * group] = log_sum
        done += n
    return [out, lse]
