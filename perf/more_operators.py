"""Cases of what many continuations of one prompt need, for timing and comparison: rotary positions, the
cache's pages forked, resized and compacted, and attention that reads a shared prefix once.

  rope     rows of queries or keys turned by their positions
  append   a step's queries and keys turned by the positions that they have in the cache, and the keys
           and values stored in its pages, over a batch of sequences
  fork     the children of last time are let go, the parents forked anew (whole pages shared, the last,
           partly filled one copied for each child, in every layer), and every child grows by its new tokens
  compact  the pages in use move to the lowest numbers, in every layer, and the tables follow
  share    attention of groups of sequences, each group's first tokens being the same pages

``run`` computes them in elementary torch operations in 32 bits (angles in 64), or, where ``own`` is
true, by the calls that a program makes of hayai_b200.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}
PLAIN = dict(base=10000.0, factor=1.0, original=0, low=0.0, high=0.0, amplitude=1.0)


def listed():
    return [
        # 1201 rows of a long document's far positions, half of each head turned in adjacent pairs, context
        # stretched by frequency bands (f32, as the projections give them).
        dict(name="rope-far-f32", op="rope", x="f32", heads=12, dim=128, rot=64, layout="pairs", tokens=1201, far=900000,
             base=500000.0, factor=8.0, original=8192, low=1.0, high=32.0, amplitude=1.2079441541679836, lens=1),
        # The queries of prompts, 32 heads of 128, 9000 tokens.
        dict(name="rope-prompts-bf16", op="rope", x="bf16", heads=32, dim=128, rot=128, layout="half", tokens=9000,
             far=20000, **(PLAIN | dict(base=500000.0)), lens=2),
        # One token of one conversation: 32 query heads, 8 kv heads of 128: launch latency.
        dict(name="append-1-f32-bf16", op="append", x="f32", cache="bf16", heads=32, kv_heads=8, dim=128, rot=128,
             layout="half", page=16, seqs=1, new_lo=1, new_hi=1, ctx_lo=999, ctx_hi=999, single=0.0, **PLAIN, lens=3),
        # Seven prompts of a few thousand tokens into an 8-bit cache (read back, as the values that its codes
        # stand for), with linear scaling.
        dict(name="append-prompts-bf16-i8", op="append", x="bf16", cache="i8", heads=32, kv_heads=8, dim=128, rot=128,
             layout="half", page=64, seqs=7, new_lo=1500, new_hi=4000, ctx_lo=1, ctx_hi=500, single=0.0,
             **(PLAIN | dict(factor=4.0)), lens=4),
        # Four continuations of one short conversation, three layers with 3 kv heads of 64.
        dict(name="fork-4-f16", op="fork", cache="f16", kv_heads=3, dim=64, page=16, layers=3, parents=1, children=4,
             len_lo=203, len_hi=203, grow=3, spare=10, lens=5),
        # A sampling server: 9 prompts, 16 continuations each, 12 layers with 8 kv heads of 128 in 8 bits.
        dict(name="fork-144-i8", op="fork", cache="i8", kv_heads=8, dim=128, page=64, layers=12, parents=9, children=16,
             len_lo=400, len_hi=5000, grow=70, spare=300, lens=6),
        # A few of 40 short conversations have ended: two layers with 4 kv heads of 64.
        dict(name="compact-40-bf16", op="compact", cache="bf16", kv_heads=4, dim=64, page=16, layers=2, seqs=40, len_lo=5,
             len_hi=400, gone=0.3, spare=37, lens=7),
        # Half of 96 long ones have ended: 8 layers with 8 kv heads of 128 in 8 bits.
        dict(name="compact-96-i8", op="compact", cache="i8", kv_heads=8, dim=128, page=64, layers=8, seqs=96, len_lo=300,
             len_hi=6000, gone=0.5, spare=200, lens=8),
        # Four continuations of a conversation's 601 tokens (32 heads on 8), f32 rows on 8-bit pages: latency.
        dict(name="share-4-f32-i8", op="share", x="f32", cache="i8", heads=32, kv_heads=8, dim=128, page=16, groups=1,
             seqs_lo=4, seqs_hi=4, pre_lo=601, pre_hi=601, own_lo=9, own_hi=40, new_lo=1, new_hi=1, lens=9),
        # A server's decode step: 64 conversations behind one instruction of 4100 tokens, 64 heads on 8.
        dict(name="share-64-bf16-i8", op="share", x="bf16", cache="i8", heads=64, kv_heads=8, dim=128, page=64, groups=1,
             seqs_lo=64, seqs_hi=64, pre_lo=4100, pre_hi=4100, own_lo=30, own_hi=1500, new_lo=1, new_hi=1, lens=10),
        # Six groups, of one to forty sequences, with chunks of new tokens behind prefixes of very different
        # lengths (32 heads on 4).
        dict(name="share-groups-f16-f16", op="share", x="f16", cache="f16", heads=32, kv_heads=4, dim=128, page=32,
             groups=6, seqs_lo=1, seqs_hi=40, pre_lo=100, pre_hi=12000, own_lo=0, own_hi=300, new_lo=1, new_hi=60, lens=11),
        # A hundred questions on one document of 60001 tokens (32 heads on 8).
        dict(name="share-100-bf16-bf16", op="share", x="bf16", cache="bf16", heads=32, kv_heads=8, dim=128, page=64, groups=1,
             seqs_lo=100, seqs_hi=100, pre_lo=60001, pre_hi=60001, own_lo=10, own_hi=200, new_lo=1, new_hi=1, lens=12),
    ]


def _log(r, lo, hi):
    """A whole number in [lo, hi], spread over the logarithm."""
    return lo if lo == hi else min(hi, int(math.exp(r.uniform(math.log(lo + 1), math.log(hi + 2)))) - 1)


def _lens(case):
    """append: (new, kv) of every sequence, its step's tokens and all tokens with them."""
    r = random.Random(case["lens"])
    new, kv = [], []
    for _ in range(case["seqs"]):
        n = 1 if r.random() < case["single"] else _log(r, case["new_lo"], case["new_hi"])
        new.append(n)
        kv.append(n + _log(r, case["ctx_lo"], case["ctx_hi"]))
    return new, kv


def _forks(case):
    """The parents' lengths, and what every child grows by."""
    r = random.Random(case["lens"])
    parents = [_log(r, case["len_lo"], case["len_hi"]) for _ in range(case["parents"])]
    return parents, [r.randint(1, case["grow"]) for _ in range(case["parents"] * case["children"])]


def _holes(case):
    """compact: the lengths (0: gone) and pages of every sequence, and the number of pages."""
    r = random.Random(case["lens"])
    lens = [_log(r, case["len_lo"], case["len_hi"]) for _ in range(case["seqs"])]
    need = [-(-n // case["page"]) for n in lens]
    order = list(range(sum(need) + case["spare"]))
    r.shuffle(order)
    pages, at = [], 0
    for n in need:
        pages.append(order[at:at + n])
        at += n
    lens = [0 if r.random() < case["gone"] else n for n in lens]
    return lens, pages, len(order)


def _groups(case):
    """share: of every group (shared tokens, [(new, kv) of every sequence])."""
    r = random.Random(case["lens"])
    got = []
    for _ in range(case["groups"]):
        pre = _log(r, case["pre_lo"], case["pre_hi"])
        seqs = []
        for _ in range(_log(r, case["seqs_lo"], case["seqs_hi"])):
            new = _log(r, case["new_lo"], case["new_hi"])
            seqs.append((new, pre + _log(r, case["own_lo"], case["own_hi"]) + new))
        got.append((pre, seqs))
    return got


def _row_bytes(case):
    """Bytes of a token's key and value in one layer's cache."""
    return 2 * case["kv_heads"] * (case["dim"] * SIZE[case["cache"]] + (4 if case["cache"] == "i8" else 0))


def work(case):
    op = case["op"]
    if op == "rope":
        n = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 2 * n * SIZE[case["x"]] + 4 * case["tokens"], "flops": 3 * n * case["rot"] // case["dim"]}
    if op == "append":
        rows = sum(_lens(case)[0])
        q, kv = (rows * case[h] * case["dim"] * SIZE[case["x"]] for h in ("heads", "kv_heads"))
        again = rows * _row_bytes(case) + 2 * kv if case["cache"] == "i8" else 0  # and read back
        return {"bytes": 2 * q + 2 * kv + rows * _row_bytes(case) + again,
                "flops": 3 * rows * (case["heads"] + case["kv_heads"]) * case["rot"]}
    if op == "fork":
        parents, grow = _forks(case)
        page, kids = case["page"], case["children"]
        rows = sum(n % page for n in parents) * kids * case["layers"]
        entries = sum(-(-(parents[i // kids] + g) // page) for i, g in enumerate(grow))
        return {"bytes": 2 * rows * _row_bytes(case) + 16 * entries, "flops": 0}
    if op == "compact":
        lens, pages, n_pages = _holes(case)
        used = sum(len(p) for n, p in zip(lens, pages) if n)
        moved = sum(q >= used for n, p in zip(lens, pages) if n for q in p)
        return {"bytes": 2 * moved * case["layers"] * case["page"] * _row_bytes(case) + 8 * used + 12 * n_pages, "flops": 0}
    heads, read, pairs, rows = case["heads"], 0, 0, 0
    for pre, seqs in _groups(case):
        read += pre
        for new, kv in seqs:
            rows += new
            read += kv - pre
            pairs += new * (kv - new) + new * (new + 1) // 2
    return {"bytes": read * _row_bytes(case) + rows * heads * (2 * case["dim"] * SIZE[case["x"]] + 4),
            "flops": 4 * case["dim"] * heads * pairs}


def _positions(rng):
    """How a drawn case turns: head size, turned part, layout, base and scaling."""
    dim = rng.choice([64, 128, 128])
    c = dict(dim=dim, rot=rng.choice([dim, dim, dim // 2, 3 * dim // 4]), layout=rng.choice(["half", "pairs"]),
             **(PLAIN | dict(base=rng.choice([10000.0, 500000.0, 1000000.0]))))
    how = rng.choice(["none", "linear", "bands"])
    if how != "none":
        c["factor"] = rng.choice([2.0, 4.0, 7.5, 32.0])
    if how == "bands":
        c |= dict(original=rng.choice([2048, 8192]), low=1.0, high=rng.choice([4.0, 32.0]),
                  amplitude=rng.choice([1.0, 0.1 * math.log(c["factor"]) + 1.0]))
    return c


def draw(rng):
    op = rng.choice(["rope", "append", "append", "fork", "compact", "share", "share", "share"])
    lens = rng.randrange(1 << 30)
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    cache = rng.choice(["f16", "bf16", "i8", "i8"])
    if op == "rope":
        c = dict(op=op, x=rng.choice(["f32", "f16", "bf16"]), heads=rng.choice([1, 3, 8, 12, 32, 40]),
                 tokens=_log(rng, 1, 9000), far=_log(rng, 10, 1000000), lens=lens, **_positions(rng))
    elif op == "append":
        # rows of an 8-bit cache are returned in 16 bits: in 32 a last bit before the codes' rounding would show
        c = dict(op=op, x=rng.choice(["f16", "bf16"] if cache == "i8" else ["f32", "f16", "bf16"]), cache=cache,
                 heads=kv_heads * rng.choice([1, 3, 4, 8]), kv_heads=kv_heads, page=rng.choice([16, 24, 32, 64, 100]),
                 seqs=_log(rng, 1, 64), new_lo=1, new_hi=_log(rng, 1, 3000), ctx_lo=0, ctx_hi=_log(rng, 1, 3000),
                 single=rng.choice([0.0, 0.5]), lens=lens, **_positions(rng))
    elif op == "fork":
        c = dict(op=op, cache=cache, kv_heads=kv_heads, dim=rng.choice([64, 128]), page=rng.choice([16, 24, 32, 64, 100]),
                 layers=_log(rng, 1, 12), parents=_log(rng, 1, 12), children=_log(rng, 1, 20), len_lo=_log(rng, 0, 100),
                 len_hi=_log(rng, 100, 5000), grow=_log(rng, 1, 100), spare=_log(rng, 1, 300), lens=lens)
    elif op == "compact":
        c = dict(op=op, cache=cache, kv_heads=kv_heads, dim=rng.choice([64, 128]), page=rng.choice([16, 24, 32, 64, 100]),
                 layers=_log(rng, 1, 8), seqs=_log(rng, 2, 120), len_lo=1, len_hi=_log(rng, 10, 6000),
                 gone=rng.choice([0.1, 0.3, 0.5, 0.8]), spare=_log(rng, 1, 300), lens=lens)
    else:
        c = dict(op=op, x=rng.choice(["f32", "f16", "bf16", "bf16"]), cache=cache, heads=kv_heads * rng.choice([1, 3, 4, 8]),
                 kv_heads=kv_heads, dim=rng.choice([64, 128, 128]), page=rng.choice([16, 24, 32, 64, 100]),
                 groups=rng.choice([1, 1, 2, 5]), seqs_lo=_log(rng, 1, 8), seqs_hi=0, pre_lo=_log(rng, 16, 2000), pre_hi=0,
                 own_lo=0, own_hi=_log(rng, 1, 1000), new_lo=1, new_hi=rng.choice([1, 1, 5, 60]), lens=lens)
        c["seqs_hi"] = c["seqs_lo"] * rng.choice([1, 2, 12])
        c["pre_hi"] = c["pre_lo"] * rng.choice([1, 3, 30])
    most = [work(k) for k in listed() if k["op"] == op]
    top = {k: max(m[k] for m in most) for k in ("bytes", "flops")}
    if op == "compact":
        pool = _holes(listed()[7])[2] * 8 * 64 * _row_bytes(listed()[7])
    while True:
        w = work(c)
        fits = w["bytes"] <= top["bytes"] and w["flops"] <= top["flops"]
        if op == "compact":
            fits = fits and _holes(c)[2] * c["layers"] * c["page"] * _row_bytes(c) <= pool
        if op == "fork":
            fits = fits and _fork_pages(c) * c["layers"] * c["page"] * _row_bytes(c) <= 4e9
        if op == "share":
            n = sum(len(s) for _, s in _groups(c))
            q = max(a for _, s in _groups(c) for a, _ in s)
            k = max(p for p, _ in _groups(c))
            fits = fits and n * q * c["heads"] * (k + c["own_hi"] + q) <= 6e8
        if fits:
            return c
        for k in ("new_hi", "seqs", "layers", "children", "seqs_hi", "len_hi", "pre_hi", "tokens"):
            if c.get(k, 0) > c.get(k[:-2] + "lo", 1 if k != "seqs" else 2):
                c[k] = max(c.get(k[:-2] + "lo", 1), c[k] * 3 // 4)


def _fork_pages(case):
    """Pages that a fork case's pool has: the parents', the children's new ones, and spare ones."""
    parents, grow = _forks(case)
    page, kids = case["page"], case["children"]
    new = sum(-(-(parents[i // kids] + g) // page) - parents[i // kids] // page for i, g in enumerate(grow))
    return sum(-(-n // page) for n in parents) + new + case["spare"]


def _pools(case, n_pages, g, fill=True):
    """A layer's pages of keys and values, and the scales of 8-bit ones."""
    shape = (n_pages, case["kv_heads"], case["page"], case["dim"])
    i8 = case["cache"] == "i8"
    got = {}
    for which in ("k", "v"):
        if not fill:
            x, scale = torch.zeros(shape, dtype=TYPES[case["cache"]], device=DEV), torch.zeros(shape[:3], device=DEV)
        elif i8:  # codes of rows of normal values: the largest is 127
            x = torch.randint(-127, 128, shape, generator=g, device=DEV, dtype=torch.int8)
            scale = torch.rand(shape[:3], generator=g, device=DEV).mul_(0.02).add_(0.01)
        else:
            x = torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(TYPES[case["cache"]])
        got[which], got[which + "_scale"] = x, scale if i8 else None
    return got


def prepare(case, seed):
    """A step's rows, and the cache's pages and bookkeeping, on the GPU."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = {"rope": _prepare_rope, "append": _prepare_append, "fork": _prepare_fork, "compact": _prepare_compact,
         "share": _prepare_share}[case["op"]](case, g)
    s["case"] = case
    if own:  # the handles that a program keeps beside its tensors
        _describe(s)
    return s


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _rows(case, n, heads, g):
    return torch.randn(n, case[heads], case["dim"], generator=g, device=DEV).to(TYPES[case["x"]])


def _prepare_rope(case, g):
    x = _rows(case, case["tokens"], "heads", g)
    pos = torch.randint(0, case["far"], (case["tokens"],), generator=g, device=DEV, dtype=torch.int32)
    return dict(x=x, out=torch.empty_like(x), pos=pos)


def _prepare_append(case, g):
    new, kv = _lens(case)
    need = [-(-k // case["page"]) for k in kv]
    n_pages = sum(need) + 3
    table = torch.zeros(len(kv), max(need), dtype=torch.int32, device=DEV)
    table[torch.arange(max(need), device=DEV)[None, :] < _ints(need)[:, None]] = torch.randperm(
        n_pages, generator=g, device=DEV, dtype=torch.int32)[:sum(need)]
    s = dict(table=table, q_start=_ints([0] + new).cumsum(0).to(torch.int32), kv_len=_ints(kv), n_tok=sum(new),
             max_new=max(new), layers=[_pools(case, n_pages, g, fill=False)])
    for t, heads in (("q", "heads"), ("k", "kv_heads"), ("v", "kv_heads")):
        s[t] = _rows(case, sum(new), heads, g)
    s |= dict(q_out=torch.empty_like(s["q"]), k_rows=torch.empty_like(s["k"]), v_rows=torch.empty_like(s["v"]))
    return s


def _prepare_fork(case, g):
    parents, grow = _forks(case)
    page, n_pages, kids = case["page"], _fork_pages(case), case["children"]
    need = [-(-n // page) for n in parents]
    slots = len(parents) * (1 + kids)
    most = max(-(-(parents[i // kids] + n) // page) for i, n in enumerate(grow))
    order = torch.randperm(n_pages, generator=g, device=DEV, dtype=torch.int32)[:sum(need)]
    table = torch.zeros(slots, max(need + [most]), dtype=torch.int32, device=DEV)
    table[:len(need)][torch.arange(table.shape[1], device=DEV)[None, :] < _ints(need)[:, None]] = order
    refs = torch.zeros(n_pages, dtype=torch.int32, device=DEV)
    refs[order.long()] = 1
    return dict(table=table, refs=refs, kv_len=_ints(parents + [0] * (slots - len(parents))),
                layers=[_pools(case, n_pages, g) for _ in range(case["layers"])],
                parents=_ints([i // kids for i in range(len(grow))]), children=_ints(list(range(len(parents), slots))),
                none=_ints([0] * len(grow)), then=_ints([parents[i // kids] + n for i, n in enumerate(grow)]))


def _prepare_compact(case, g):
    lens, pages, n_pages = _holes(case)
    table = torch.zeros(len(lens), max(len(p) for p in pages), dtype=torch.int32)
    refs = torch.zeros(n_pages, dtype=torch.int32)
    for i, p in enumerate(pages):
        table[i, :len(p)] = torch.tensor(p, dtype=torch.int32)
        if lens[i]:
            refs[torch.tensor(p, dtype=torch.long)] = 1
    s = dict(table_now=table.to(DEV), refs_now=refs.to(DEV), kv_len=_ints(lens),
             moved=torch.empty(n_pages, dtype=torch.int32, device=DEV),
             layers=[_pools(case, n_pages, g) for _ in range(case["layers"])])
    return s | dict(table=torch.empty_like(s["table_now"]), refs=torch.empty_like(s["refs_now"]))


def _prepare_share(case, g):
    page, groups = case["page"], _groups(case)
    new = [n for _, seqs in groups for n, _ in seqs]
    kv = [k for _, seqs in groups for _, k in seqs]
    # a group's whole pages are one for all its sequences, the rest of the prefix a copy of each
    whole = [pre // page for pre, seqs in groups for _ in seqs]
    first = [i == 0 for _, seqs in groups for i in range(len(seqs))]
    need = [-(-k // page) for k in kv]
    n_pages = sum(n if f else n - w for n, f, w in zip(need, first, whole)) + 3
    order = torch.randperm(n_pages, generator=g, device=DEV, dtype=torch.int32)
    pools = _pools(case, n_pages, g)
    if case["cache"] != "i8":  # keys have a few strong channels
        pools["k"][..., :: case["dim"] // 4] *= 3.0
    table = torch.zeros(len(kv), max(need), dtype=torch.int32, device=DEV)
    at = 0
    starts, i = [0], 0
    for pre, seqs in groups:
        head = i
        for _ in seqs:
            w = 0 if i == head else whole[i]
            table[i, :w] = table[head, :w]
            table[i, w:need[i]] = order[at:at + need[i] - w]
            at += need[i] - w
            if i > head and pre % page:
                for name in ("k", "v", "k_scale", "v_scale"):
                    if pools[name] is not None:
                        pools[name][table[i, w].long(), :, :pre % page] = pools[name][table[head, w].long(), :, :pre % page]
            i += 1
        starts.append(i)
    q = _rows(case, sum(new), "heads", g)
    return dict(layers=[pools], table=table, q_start=_ints([0] + new).cumsum(0).to(torch.int32), kv_len=_ints(kv),
                n_tok=sum(new), max_new=max(new), starts=_ints(starts), shared=_ints([pre for pre, _ in groups]),
                max_group=max(sum(n for n, _ in seqs) for _, seqs in groups), q=q, out=torch.empty_like(q),
                lse=torch.empty(sum(new), case["heads"], device=DEV), most_own=max(k - p for p, t in groups for _, k in t))


# ------------------------------------------------------------------ hayai_b200
_engines = []


def _describe(s):
    import hayai_b200 as hb
    if not _engines:
        _engines.append(hb.CudaEngine(0))
        _engines[0].set_stream(torch.cuda.current_stream())
    c = s["case"]
    s["engine"] = _engines[0]
    if "rot" in c:
        s["rope"] = hb.Rope(c["dim"], c["rot"], base=c["base"], layout=c["layout"], factor=c["factor"],
                            original=c["original"], low=c["low"], high=c["high"], amplitude=c["amplitude"])
    if "layers" in s:
        s["caches"] = [hb.KvCache(p["k"], p["v"], p["k_scale"], p["v_scale"]) for p in s["layers"]]
    if "q_start" in s:
        s["batch"] = hb.KvBatch(s["table"], s["q_start"], s["kv_len"], s["n_tok"], s["max_new"])
    if "refs" in s:
        s["pages"] = hb.KvPages(s["caches"], s["table"], s["kv_len"], s["refs"])
    if "shared" in s:
        s["prefix"] = hb.KvShared(s["starts"], s["shared"], s["max_group"])


def _run_own(s):
    e, op, i8 = s["engine"], s["case"]["op"], s["case"].get("cache") == "i8"
    if op == "rope":
        e.rope_dev(s["rope"], s["pos"], s["x"], s["out"])
        return [s["out"]]
    if op == "append":
        e.kv_append_rope_dev(s["caches"][0], s["batch"], s["rope"], s["q"], s["k"], s["v"], s["q_out"])
        if not i8:
            return [s["q_out"], s["layers"][0]["k"], s["layers"][0]["v"]]
        e.kv_read_dev(s["caches"][0], s["batch"], s["k_rows"], s["v_rows"])
        return [s["q_out"], s["k_rows"], s["v_rows"]]
    if op == "fork":
        e.kv_resize_dev(s["pages"], s["children"], s["none"])
        e.kv_fork_dev(s["pages"], s["parents"], s["children"])
        e.kv_resize_dev(s["pages"], s["children"], s["then"])
        return [s["table"], s["kv_len"], s["refs"], _tensors(s)]
    if op == "compact":
        s["table"].copy_(s["table_now"])  # the bookkeeping as the step finds it
        s["refs"].copy_(s["refs_now"])
        e.kv_compact_dev(s["pages"], s["moved"])
        return [s["table"], s["refs"], s["moved"], _tensors(s)]
    e.attn_shared_dev(s["caches"][0], s["batch"], s["prefix"], s["q"], s["out"], lse=s["lse"])
    return [s["out"], s["lse"]]


def _tensors(s):
    return [t for p in s["layers"] for t in p.values() if t is not None]


def run(s):
    if own:
        return _run_own(s)
    return {"rope": _rope, "append": _append, "fork": _fork, "compact": _compact, "share": _share}[s["case"]["op"]](s)


# ------------------------------------------------------------------ the plain form
def _turned(c, x, pos):
    """Rows x [n][heads][dim] in 32 bits, turned by their positions."""
    rot = c["rot"]
    t = c["base"] ** (torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / -rot)
    if c["original"]:
        keep = ((c["original"] * t / (2 * math.pi) - c["low"]) / (c["high"] - c["low"])).clamp(0, 1)
        t = t * ((1 - keep) / c["factor"] + keep)
    else:
        t = t / c["factor"]
    angle = (pos.double()[:, None] * t)[:, None]
    cos, sin = (angle.cos() * c["amplitude"]).float(), (angle.sin() * c["amplitude"]).float()
    y = x.float()
    if c["layout"] == "half":
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, y[..., rot:]], -1)
    a, b = y[..., :rot:2], y[..., 1:rot:2]
    return torch.cat([torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2), y[..., rot:]], -1)


def _rope(s):
    return [_turned(s["case"], s["x"], s["pos"]).to(s["x"].dtype)]


def _seqs(s):
    """Sequence of each of the step's tokens, and its position there."""
    start = s["q_start"].long()
    t = torch.arange(s["n_tok"], device=DEV)
    seq = torch.searchsorted(start, t, right=True) - 1
    return seq, s["kv_len"].long()[seq] - start[seq + 1] + t


def _append(s):
    c, pool = s["case"], s["layers"][0]
    seq, pos = _seqs(s)
    page, row = s["table"][seq, pos // c["page"]].long(), pos % c["page"]
    out = [_turned(c, s["q"], pos).to(s["q"].dtype)]
    for x, which in ((_turned(c, s["k"], pos), "k"), (s["v"].float(), "v")):
        if c["cache"] == "i8":
            scale = x.abs().amax(-1) / 127.0
            codes = torch.where(scale[..., None] > 0, (x / scale[..., None]).round().clamp(-127, 127), torch.zeros_like(x))
            pool[which][page, :, row] = codes.to(torch.int8)
            pool[which + "_scale"][page, :, row] = scale
            out.append((pool[which][page, :, row].float() * pool[which + "_scale"][page, :, row][..., None]).to(s["k"].dtype))
        else:
            pool[which][page, :, row] = x.to(pool[which].dtype)
            out.append(pool[which])
    return out


def _copied(s, src, dst, rows):
    """The first `rows` rows of pages src to pages dst, in every layer."""
    have = (torch.arange(s["case"]["page"], device=DEV) < rows[:, None])[:, None]
    for t in _tensors(s):
        t[dst] = torch.where(have[..., None] if t.dim() == 4 else have, t[src], t[dst])


def _resized(s, slots, lens):
    page, table, refs, slots = s["case"]["page"], s["table"], s["refs"], slots.long()
    old, new = s["kv_len"][slots].long(), lens.long()
    keep = torch.minimum(old, new)
    had, get = (old + page - 1) // page, (new + page - 1) // page
    last = table[slots, (keep - 1).clamp(min=0) // page].long()
    split = (keep % page > 0) & (refs[last] > 1)  # a page of others' as well: a copy of its rows
    need = (get - had).clamp(min=0) + split
    at = need.cumsum(0) - need
    free = (refs == 0).nonzero().flatten()
    col = torch.arange(table.shape[1], device=DEV)
    gone = (col >= get[:, None]) & (col < had[:, None])
    refs.index_add_(0, table[slots][gone].long(), torch.full_like(table[slots][gone], -1))
    which = split.nonzero().flatten()
    _copied(s, last[which], free[at[which]], keep[which] % page)
    table[slots[which], (keep[which] - 1) // page] = free[at[which]].int()
    refs.index_add_(0, last[which], torch.full_like(which, -1, dtype=torch.int32))
    i, j = ((col >= had[:, None]) & (col < get[:, None])).nonzero(as_tuple=True)
    table[slots[i], j] = free[(at + split)[i] + j - had[i]].int()
    refs[free[:int(need.sum())]] = 1
    s["kv_len"][slots] = lens


def _forked(s, parents, children):
    page, table, refs, parents, children = s["case"]["page"], s["table"], s["refs"], parents.long(), children.long()
    n = s["kv_len"][parents].long()
    col = torch.arange(table.shape[1], device=DEV)
    i, j = (col < (n // page)[:, None]).nonzero(as_tuple=True)
    pages = table[parents[i], j]
    table[children[i], j] = pages
    refs.index_add_(0, pages.long(), torch.ones_like(pages))
    which = (n % page > 0).nonzero().flatten()
    free = (refs == 0).nonzero().flatten()[:len(which)]
    _copied(s, table[parents[which], n[which] // page].long(), free, n[which] % page)
    table[children[which], n[which] // page] = free.int()
    refs[free] = 1
    s["kv_len"][children] = s["kv_len"][parents]


def _fork(s):
    _resized(s, s["children"], s["none"])
    _forked(s, s["parents"], s["children"])
    _resized(s, s["children"], s["then"])
    return [s["table"], s["kv_len"], s["refs"], _tensors(s)]


def _compact(s):
    table, refs, moved = s["table"].copy_(s["table_now"]), s["refs"].copy_(s["refs_now"]), s["moved"]
    used = int((refs > 0).sum())
    src, dst = (refs[used:] > 0).nonzero().flatten() + used, (refs[:used] == 0).nonzero().flatten()
    for t in _tensors(s):
        t[dst] = t[src]
    moved.copy_(torch.arange(len(refs), device=DEV))
    moved[src] = dst.int()
    refs[dst] = refs[src]
    refs[src] = 0
    page = s["case"]["page"]
    live = torch.arange(table.shape[1], device=DEV) < ((s["kv_len"] + page - 1) // page)[:, None]
    table.copy_(torch.where(live, moved[table.long()], table))
    return [table, refs, moved, _tensors(s)]


def _gathered(pool, which, page, row):
    x = pool[which][page, :, row].float()
    scale = pool[which + "_scale"]
    return x if scale is None else x * scale[page, :, row][..., None]


def _share(s):
    c, pool = s["case"], s["layers"][0]
    hk, dim, heads = c["kv_heads"], c["dim"], c["heads"]
    group = heads // hk
    n, most_q, most_k = len(s["kv_len"]), s["max_new"], s["most_own"]
    seq, pos = _seqs(s)
    at = torch.arange(s["n_tok"], device=DEV) - s["q_start"].long()[seq]
    q = torch.zeros(n, most_q, heads, dim, device=DEV)
    q[seq, at] = s["q"].float() * dim ** -0.5
    q = q.view(n, most_q, hk, group, dim).permute(0, 2, 3, 1, 4).reshape(n, hk, group * most_q, dim)
    starts, shared = s["starts"].tolist(), s["shared"].tolist()
    pre = s["shared"].long().repeat_interleave(s["starts"].diff())
    # every sequence's own tokens
    key = pre[:, None] + torch.arange(most_k, device=DEV)
    page = s["table"].gather(1, (key // c["page"]).clamp(max=s["table"].shape[1] - 1)).long()
    k, v = (_gathered(pool, w, page, key % c["page"]).transpose(1, 2) for w in ("k", "v"))
    a = torch.matmul(q, k.transpose(2, 3)).view(n, hk, group, most_q, most_k)
    where = (s["kv_len"] - s["q_start"].diff())[:, None] + torch.arange(most_q, device=DEV)
    a.masked_fill_((key[:, None] > where[..., None])[:, None, None], -math.inf)
    top = a.amax(-1).flatten(2)
    safe = torch.where(top > -math.inf, top, torch.zeros_like(top))
    p = a.flatten(2, 3).sub_(safe[..., None]).exp_()
    total, out = p.sum(-1), torch.matmul(p, v)
    # the groups' shared tokens
    for lo, hi, length in zip(starts[:-1], starts[1:], shared):
        key = torch.arange(length, device=DEV)
        page = s["table"][lo, key // c["page"]].long()
        k, v = (_gathered(pool, w, page, key % c["page"]).transpose(0, 1) for w in ("k", "v"))
        a = torch.matmul(q[lo:hi].transpose(0, 1).reshape(hk, -1, dim), k.transpose(1, 2))
        most = a.amax(-1)
        p = a.sub_(most[..., None]).exp_()
        back = lambda t: t.view(hk, hi - lo, group * most_q, *t.shape[2:]).transpose(0, 1)  # noqa: E731
        m, t, o = back(most), back(p.sum(-1)), back(torch.matmul(p, v))
        new = torch.maximum(m, top[lo:hi])
        f, g = (m - new).exp(), (top[lo:hi] - new).exp()
        out[lo:hi] = out[lo:hi] * g[..., None] + o * f[..., None]
        total[lo:hi] = total[lo:hi] * g + t * f
        top[lo:hi] = new
    out, lse = out / total[..., None], top + total.log()
    out = out.view(n, hk, group, most_q, dim).permute(0, 3, 1, 2, 4).reshape(n, most_q, heads, dim)[seq, at]
    lse = lse.view(n, hk, group, most_q).permute(0, 3, 1, 2).reshape(n, most_q, heads)[seq, at]
    return [out.to(TYPES[c["x"]]), lse]


# ------------------------------------------------------------------ the definition
def _exact_turn(case, x, pos):
    """Rows x, turned as complex numbers in 64 bits."""
    half = case["rot"] // 2
    t = []
    for i in range(half):
        f = 1.0 / case["base"] ** (i / half)
        if case["original"]:
            turns = case["original"] * f / math.tau
            g = min(1.0, max(0.0, (turns - case["low"]) / (case["high"] - case["low"])))
            t.append(f / case["factor"] * (1.0 - g) + f * g)
        else:
            t.append(f / case["factor"])
    by = torch.polar(torch.tensor(case["amplitude"], dtype=torch.float64, device=DEV),
                     torch.outer(pos.double(), torch.tensor(t, dtype=torch.float64, device=DEV))).unsqueeze(1)
    y = x.double()
    part = y[..., :2 * half]
    z = torch.complex(part[..., :half], part[..., half:]) if case["layout"] == "half" else torch.complex(
        part[..., 0::2], part[..., 1::2])
    z = z * by
    y[..., :2 * half] = torch.cat([z.real, z.imag], -1) if case["layout"] == "half" else torch.view_as_real(z).flatten(-2)
    return y


def exact(case, seed):
    """The operators' definition, in 64 bits or whole numbers, one sequence or page at a time."""
    s = prepare(case, seed)
    return {"rope": lambda: [_exact_turn(case, s["x"], s["pos"])], "append": lambda: _exact_append(case, s),
            "fork": lambda: _exact_fork(case, s), "compact": lambda: _exact_compact(case, s),
            "share": lambda: _exact_share(case, s)}[case["op"]]()


def _exact_append(case, s):
    new, kv = _lens(case)
    pos = torch.cat([torch.arange(k - n, k, device=DEV) for n, k in zip(new, kv)])
    rows = [_exact_turn(case, s["k"], pos), s["v"].double()]
    outs = [_exact_turn(case, s["q"], pos)]
    if case["cache"] == "i8":
        for x in rows:
            step = x.abs().max(-1, keepdim=True).values / 127
            outs.append(torch.round(x / torch.where(step == 0, 1.0, step)) * step)
        return outs
    for x, which in zip(rows, ("k", "v")):
        pool, done = s["layers"][0][which].double(), 0
        for i, (n, k) in enumerate(zip(new, kv)):
            p = torch.arange(k - n, k, device=DEV)
            pool[s["table"][i].long()[p // case["page"]], :, p % case["page"]] = x[done:done + n]
            done += n
        outs.append(pool)
    return outs


def _exact_fork(case, s):
    page = case["page"]
    table, refs, kv = s["table"].tolist(), s["refs"].tolist(), s["kv_len"].tolist()

    def take():
        p = refs.index(0)
        refs[p] = 1
        return p

    # the children hold nothing yet, so that letting them go is nothing
    for a, b in zip(s["parents"].tolist(), s["children"].tolist()):
        whole, rest = divmod(kv[a], page)
        for j in range(whole):
            table[b][j] = table[a][j]
            refs[table[a][j]] += 1
        if rest:
            table[b][whole] = take()
            for t in _tensors(s):
                t[table[b][whole], :, :rest] = t[table[a][whole], :, :rest]
        kv[b] = kv[a]
    for b, n in zip(s["children"].tolist(), s["then"].tolist()):
        for j in range(-(-kv[b] // page), -(-n // page)):
            table[b][j] = take()
        kv[b] = n
    return [_ints(table), _ints(kv), _ints(refs), _tensors(s)]


def _exact_compact(case, s):
    table, refs, kv = s["table_now"].tolist(), s["refs_now"].tolist(), s["kv_len"].tolist()
    used = sum(r > 0 for r in refs)
    to = list(range(len(refs)))
    hole = 0
    for p in range(used, len(refs)):
        if refs[p] == 0:
            continue
        hole = refs.index(0, hole)
        to[p], refs[hole], refs[p] = hole, refs[p], 0
        for t in _tensors(s):
            t[hole] = t[p]
    for row, n in zip(table, kv):
        for j in range(-(-n // case["page"])):
            row[j] = to[row[j]]
    return [_ints(table), _ints(refs), _ints(to), _tensors(s)]


def _exact_share(case, s):
    page, group = case["page"], case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device=DEV)

    def rows_of(which, i, lo, hi):
        pos = torch.arange(lo, hi, device=DEV)
        p = s["table"][i].long()[torch.div(pos, page, rounding_mode="floor")]
        x = s["layers"][0][which][p, :, pos.remainder(page)].double()
        scale = s["layers"][0][which + "_scale"]
        return x if scale is None else x * scale[p, :, pos.remainder(page)].double().unsqueeze(-1)

    done = i = 0
    for _, seqs in _groups(case):
        for new, kv in seqs:  # every sequence by its own pages
            K, V = rows_of("k", i, 0, kv), rows_of("v", i, 0, kv)
            hidden = torch.arange(kv, device=DEV)[None, :] > torch.arange(kv - new, kv, device=DEV)[:, None]
            q = s["q"][done:done + new].double().view(new, case["kv_heads"], group, case["dim"])
            a = torch.einsum("nhgd,khd->hgnk", q, K) / math.sqrt(case["dim"])
            a = a.masked_fill(hidden, -math.inf)
            log_sum = torch.logsumexp(a, -1)
            o = torch.einsum("hgnk,khd->nhgd", (a - log_sum[..., None]).exp(), V)
            out[done:done + new] = o.reshape(new, case["heads"], case["dim"])
            lse[done:done + new] = log_sum.permute(2, 0, 1).reshape(new, case["heads"])
            done += new
            i += 1
    return [out, lse]
