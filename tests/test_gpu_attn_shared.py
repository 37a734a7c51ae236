"""GPU tests of attention over shared prefixes (attn_shared_dev) against its definition in 64 bits: what every
sequence sees by its own pages.

Tolerances as for attn_paged_dev (tests/test_gpu_kv.py): A_i = sum_j p_ij |v_j|; 16-bit weights and results 2^-8
(A + |out|), f16 on f16 2^-10, f32 results 2^-13 elementwise and 1e-5 in the 2-norm.  Joining the prefix with a
sequence's own tokens adds a few roundings of 32 bits (2^-22), far below these."""
import math

import pytest
import torch

import hayai_b200 as hb

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}


@pytest.fixture(autouse=True)
def _stream(engine):
    engine.set_stream(torch.cuda.current_stream())
    yield
    engine.sync()
    engine.set_stream(None)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


class Groups:
    """groups: [(shared, [(new, own)])], own counted from the prefix's end, the new tokens included (of an
    empty sequence: 0, 0).  Whole pages of a prefix are shared, the rest copied; slots that no token has hold
    NaN (16-bit) or NaN scales."""

    def __init__(self, groups, kv_heads, dim, page, cache, seed=1, spread=1.0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.page, self.kv_heads, self.dim, self.type, self.groups = page, kv_heads, dim, cache, groups
        self.new = [n for _, seqs in groups for n, _ in seqs]
        self.kv = [p + own for p, seqs in groups for _, own in seqs]
        need = [-(-k // page) for k in self.kv]
        lists, fresh, i, starts, copies = [], 0, 0, [0], []
        for p, seqs in groups:
            for j in range(len(seqs)):
                whole = p // page if j else 0
                own = list(range(fresh, fresh + need[i] - whole))
                fresh += len(own)
                lists.append((lists[i - j][:whole] if j else []) + own)
                if j and p % page:
                    copies.append((lists[i - j][whole], lists[i][whole], p % page))
                i += 1
            starts.append(i)
        n_pages = fresh + 2
        perm = torch.randperm(n_pages, generator=g, device=DEV, dtype=torch.int32)
        self.table = torch.full((len(lists), max(need + [1])), -7, dtype=torch.int32, device=DEV)
        used = torch.zeros(n_pages, page, dtype=torch.bool, device=DEV)
        for i, l in enumerate(lists):
            if l:
                self.table[i, :len(l)] = perm[torch.tensor(l, device=DEV)]
                pos = torch.arange(self.kv[i], device=DEV)
                used[self.table[i].long()[pos // page], pos % page] = True
        shape = (n_pages, kv_heads, page, dim)
        self.pool, self.scale = [], []
        for _ in range(2):
            x = torch.randn(shape, generator=g, device=DEV) * spread
            if cache == "i8":
                s = x.abs().amax(-1) / 127
                c = (x / s[..., None]).round().to(torch.int8)
                s[~used[:, None].expand(s.shape)] = math.nan
            else:
                s, c = None, x.to(T[cache])
                c[~used[:, None, :, None].expand(c.shape)] = math.nan
            for a, b, rows in copies:
                for t in (c, s):
                    if t is not None:
                        t[perm[b].long(), :, :rows] = t[perm[a].long(), :, :rows]
            self.pool.append(c)
            self.scale.append(s)
        self.q_start, self.kv_len = ints([0] + self.new).cumsum(0).to(torch.int32), ints(self.kv)
        self.rows, self.g = sum(self.new), g
        self.cache = hb.KvCache(*self.pool, *self.scale)
        self.batch = hb.KvBatch(self.table, self.q_start, self.kv_len, self.rows, max(self.new))
        self.starts, self.length = ints(starts), ints([p for p, _ in groups])
        self.shared = hb.KvShared(self.starts, self.length, max(sum(n for n, _ in s) for _, s in groups), 1)

    def q(self, heads, dtype, scale=1.0):
        return (torch.randn(self.rows, heads, self.dim, generator=self.g, device=DEV) * scale).to(T[dtype])

    def values(self, w, i):
        pos = torch.arange(self.kv[i], device=DEV)
        p, r = self.table[i].long()[pos // self.page], pos % self.page
        x = self.pool[w][p, :, r].double()
        return x if self.scale[w] is None else x * self.scale[w][p, :, r].double()[..., None]

    def attention(self, q, scale=None):
        scale = self.dim ** -0.5 if scale is None else scale
        heads = q.shape[1]
        out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
        amp, lse = torch.zeros_like(out), torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=DEV)
        done = 0
        for i, (n, k) in enumerate(zip(self.new, self.kv)):
            if n and k:
                K, V = (self.values(w, i).repeat_interleave(heads // self.kv_heads, 1) for w in range(2))
                see = torch.arange(k, device=DEV)[None] <= torch.arange(k - n, k, device=DEV)[:, None]
                s = torch.einsum("nhd,khd->hnk", q[done:done + n].double(), K) * scale
                s = s.masked_fill(~see, -math.inf)
                l = torch.logsumexp(s, -1)
                p = torch.where(see, (s - l.masked_fill(l == -math.inf, 0)[..., None]).exp(), 0.0)
                out[done:done + n] = torch.einsum("hnk,khd->nhd", p, V)
                amp[done:done + n] = torch.einsum("hnk,khd->nhd", p, V.abs())
                lse[done:done + n] = l.T
            done += n
        return out, lse, amp


def close(s, dtype, out, lse, want):
    ref, ref_lse, amp = want
    got = out.double()
    assert torch.isfinite(got).all()
    c = 2.0 ** -13 if dtype == "f32" else 2.0 ** -10 if dtype == s.type == "f16" else 2.0 ** -8
    worst = ((got - ref).abs() - c * (amp + ref.abs())).max().item()
    assert worst <= 1e-30, f"off by {worst} more than its bound"
    if dtype == "f32":
        assert ((got - ref).norm() / ref.norm()).item() <= 1e-5
    none = ref_lse == -math.inf
    assert torch.equal(lse == -math.inf, none) and (got[none] == 0).all()
    assert ((lse.double() - ref_lse)[~none].abs() <= 2.0 ** -12 + ref_lse[~none].abs() * 2.0 ** -20).all()


def check(engine, s, heads, dtype, q=None, scale=None, shared=None):
    q = s.q(heads, dtype) if q is None else q
    out, lse = torch.full_like(q, math.nan), torch.full(q.shape[:2], math.nan, device=DEV)
    engine.attn_shared_dev(s.cache, s.batch, shared or s.shared, q, out, scale=scale, lse=lse)
    engine.sync()
    close(s, dtype, out, lse, s.attention(q, scale))
    return out, lse


ONE = [(1, 1)]
CASES = {
    "two": [(5, ONE * 2)],
    "whole pages": [(64, [(1, 1), (1, 20), (1, 33)])],
    "ragged": [(37, [(1, 1), (2, 3), (1, 40)]), (0, [(1, 4), (1, 1)]), (200, [(1, 9)]), (1, ONE * 3), (129, [(5, 5), (1, 100)])],
    "chunks": [(130, [(7, 7), (20, 31), (1, 1)]), (16, [(40, 40), (3, 50)])],
    "empty ones": [(50, [(1, 1), (0, 0), (1, 7)]), (20, [(0, 3), (0, 0)]), (30, [(0, 0), (2, 2), (2, 5)])],
    "many": [(300, ONE * 20 + [(1, 60)] * 20)],
}


@pytest.mark.parametrize("case", list(CASES))
@pytest.mark.parametrize("cache", ["i8", "f16", "bf16"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(8, 2, 64, 16), (3, 3, 128, 24), (16, 2, 128, 100)])
def test_groups(engine, case, cache, dtype, heads, kv_heads, dim, page):
    check(engine, Groups(CASES[case], kv_heads, dim, page, cache), heads, dtype)


@pytest.mark.parametrize("cache,dtype", [("i8", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("i8", "f32"), ("bf16", "f16")])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("groups", [[(5000, [(1, 30)] * 33)], [(20011, [(1, 700), (1, 1), (1, 2000)])], [(3000, [(60, 90)] * 9), (70, [(1, 5000)] * 5)],
                                    [(9001, [(1, 3)] * 150)]])
def test_long_prefixes(engine, cache, dtype, dim, groups):
    check(engine, Groups(groups, 2, dim, 64, cache), 16, dtype)


@pytest.mark.parametrize("rows", [15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300])
@pytest.mark.parametrize("cache,dtype", [("i8", "f16"), ("bf16", "bf16")])
def test_rows_at_the_tiles_edges(engine, rows, cache, dtype):
    check(engine, Groups([(777, ONE * rows)], 1, 128, 32, cache), 1, dtype)


@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 127, 128, 129, 255, 256, 257, 383, 384, 385, 1000])
@pytest.mark.parametrize("cache,dtype", [("i8", "f16"), ("f16", "f16"), ("bf16", "f32")])
def test_lengths_at_the_units_edges(engine, length, cache, dtype):
    check(engine, Groups([(length, [(1, 2)] * 20)], 1, 64, 16, cache), 4, dtype)


@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("f32", "i8")])
def test_lengths_are_cut_to_what_all_new_tokens_see(engine, dtype, cache):
    """A shared length that reaches into the new tokens of a sequence, or past its end, is shared as far as it goes:
    page by page of one sequence's own, which has all that is cut."""
    s = Groups([(100, [(3, 3), (1, 40), (5, 60)]), (60, [(1, 1), (2, 2)])], 2, 64, 16, cache)
    want = check(engine, s, 4, dtype, q=(q := s.q(4, dtype)))
    s.length.copy_(ints([95, 44]))
    close(s, dtype, *check(engine, s, 4, dtype, q=q), s.attention(q))
    s.length.copy_(ints([105, 62]))  # sequences of one group agree on the first 100 and 60 tokens: so much is shared
    got = check(engine, s, 4, dtype, q=q)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("cache,dtype", [("i8", "bf16"), ("f16", "f16"), ("bf16", "f32")])
@pytest.mark.parametrize("new", [1, 40])
def test_sequences_that_have_gone(engine, cache, dtype, new):
    """A group is read by the pages of one that is there: those without new tokens may hold nothing."""
    s = Groups([(200, [(0, 0), (0, 0), (new, 90), (0, 0), (new, 60)]), (90, [(0, 0), (new, 70), (new, 70)])], 2, 64, 16, cache)
    for i in (0, 1, 3, 5):
        s.table[i], s.kv_len[i] = -1, 0
    check(engine, s, 8, dtype)


def test_sequences_outside_the_groups(engine):
    s = Groups(CASES["ragged"], 2, 64, 16, "f16")
    n = len(s.new)
    check(engine, s, 8, "f16", shared=hb.KvShared(ints([3, 5, 6]), ints([0, 200]), 0, 1))
    check(engine, s, 8, "f16", shared=hb.KvShared(ints([0, 3]), ints([37]), 4, 1))
    check(engine, s, 8, "f16", shared=hb.KvShared(ints([n, n]), ints([37]), 0, 1))
    check(engine, s, 8, "f16", shared=hb.KvShared(ints([0]), ints([]), 0, 1))


def test_without_hints_and_with_wrong_ones(engine):
    s = Groups(CASES["chunks"], 2, 128, 16, "bf16")
    for most in (0, 1, 10**9):
        check(engine, s, 16, "bf16", shared=hb.KvShared(s.starts, s.length, most, 1))
    s.batch = hb.KvBatch(s.table, s.q_start, s.kv_len, s.rows)
    check(engine, s, 16, "bf16")


@pytest.mark.parametrize("dtype,cache", [("f32", "f16"), ("bf16", "i8"), ("f16", "f16")])
@pytest.mark.parametrize("strength", [0.0, 4.0, -4.0])
def test_weights_on_one_side(engine, dtype, cache, strength):
    """Queries along the prefix's keys, or against them: all weight in the prefix, or none."""
    s = Groups([(300, [(1, 20)] * 12)], 1, 64, 16, cache)
    K = s.values(0, 0)[:300, 0]
    q = (K.mean(0) / K.mean(0).norm() * strength * 8).float().expand(s.rows, 2, 64) + 0.1 * s.q(2, "f32")
    check(engine, s, 2, dtype, q=q.to(T[dtype]).contiguous())


def test_scale_and_strided_rows(engine):
    s = Groups(CASES["chunks"], 2, 64, 16, "f16")
    buf = torch.randn(s.rows, 3, 8, 64, generator=s.g, device=DEV).half()
    q, out = buf[:, 1], torch.full((s.rows, 2, 8, 64), 7.0, device=DEV).half()
    lse = torch.empty(s.rows, 8, device=DEV)
    for scale in (0.3, -0.2, 0.0):
        engine.attn_shared_dev(s.cache, s.batch, s.shared, q, out[:, 1], scale=scale, lse=lse)
        engine.sync()
        close(s, "f16", out[:, 1], lse, s.attention(q, scale))
        assert (out[:, 0] == 7).all()
    engine.attn_shared_dev(s.cache, s.batch, s.shared, q, out[:, 1])  # no lse
    engine.sync()


@pytest.mark.parametrize("dtype,cache", [("f32", "i8"), ("bf16", "bf16"), ("f16", "i8")])
@pytest.mark.parametrize("at", ["prefix", "own"])
def test_not_finite(engine, dtype, cache, at):
    """A value that is not finite reaches the rows that see it, and no others."""
    s = Groups([(40, [(1, 20)] * 3), (50, [(1, 9)] * 2)], 1, 64, 16, cache)
    page = s.table[0, 1] if at == "prefix" else s.table[1, 3]
    if cache == "i8":
        s.scale[1][page.long(), 0, 2] = math.inf
    else:
        s.pool[1][page.long(), 0, 2, :] = math.inf
    q = s.q(4, dtype)
    out = torch.zeros_like(q)
    engine.attn_shared_dev(s.cache, s.batch, s.shared, q, out)
    engine.sync()
    bad = ~out.isfinite().all(-1).all(-1)
    assert bad.tolist() == ([True] * 3 if at == "prefix" else [False, True, False]) + [False, False]


@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "i8"), ("bf16", "f16"), ("f32", "f16")])
@pytest.mark.parametrize("new,own", [(40, 40), (70, 200), (3, 300)])
@pytest.mark.parametrize("heads", [1, 4, 16])
def test_not_finite_where_some_rows_do_not_see_it(engine, dtype, cache, new, own, heads):
    """Infinities among a chunk's own tokens reach its later tokens, and leave the earlier ones what they were."""
    s = Groups([(90, [(new, own), (2, 30), (1, 1)])], 1, 64, 16, cache)
    q = s.q(heads, dtype)
    clean, lse = check(engine, s, heads, dtype, q=q)
    at = s.kv[0] - 2  # the chunk's last token but one
    page, row = s.table[0, at // 16].long(), at % 16
    if cache == "i8":
        s.scale[1][page, 0, row] = math.nan
    else:
        s.pool[1][page, 0, row, 5] = math.inf
        s.pool[1][page, 0, row, 6] = math.nan
    out = torch.zeros_like(q)
    engine.attn_shared_dev(s.cache, s.batch, s.shared, q, out)
    engine.sync()
    bad = ~out.isfinite().all(-1).all(-1)
    assert bad.nonzero().flatten().tolist() == [new - 2, new - 1]
    c = 2.0 ** -13 if dtype == "f32" else 2.0 ** -10 if dtype == cache == "f16" else 2.0 ** -8
    most = s.values(1, 1).abs().max().item()
    keep = ~bad
    # both are within c (A + |out|) of the definition, and |out| <= A <= the largest value
    most = max(most, clean.abs().max().item(), 6.0)
    assert (out[keep].double() - clean[keep].double()).abs().max().item() <= 4 * c * most


@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("f16", "i8"), ("f32", "bf16")])
def test_tokens_before_the_first_position_see_nothing(engine, dtype, cache):
    """A sequence with more new tokens than tokens shares nothing with its group, and its first ones get zeros."""
    s = Groups([(40, [(1, 5), (1, 9)]), (0, [(30, 12), (5, 2)])], 2, 64, 16, cache)
    out, lse = check(engine, s, 8, dtype)
    assert (lse[2:20] == -math.inf).all() and (out[2:20] == 0).all() and (lse[20:32] > -math.inf).all()


@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("f16", "i8"), ("bf16", "f16")])
@pytest.mark.parametrize("dim", [64, 128])
def test_chunks_of_many_tiles(engine, dtype, cache, dim):
    """Chunks whose rows are several tiles with ends of their own, beside single tokens, behind a long prefix."""
    check(engine, Groups([(2050, [(130, 130), (1, 700), (257, 900), (16, 16), (1, 1)]), (0, [(300, 300)])], 1, dim, 24, cache), 4, dtype)


@pytest.mark.parametrize("dtype,cache", [("bf16", "i8"), ("f32", "f16")])
def test_as_many_sequences_as_a_batch_takes(engine, dtype, cache):
    """2048 sequences in 1024 groups of two, and in one group, tables wider than they need be."""
    s = Groups([(20 + i % 7, ONE * 2) for i in range(1024)], 1, 64, 16, cache)
    wide = torch.full((2048, 5), -1, dtype=torch.int32, device=DEV)
    wide[:, 1:1 + s.table.shape[1]] = s.table
    s.batch = hb.KvBatch(wide[:, 1:3], s.q_start, s.kv_len, s.rows, 1)
    check(engine, s, 2, dtype)
    check(engine, Groups([(333, [(1, 1 + i % 3) for i in range(2048)])], 1, 64, 16, cache), 2, dtype)


def test_the_same_bits_every_time(engine):
    s = Groups([(3000, [(1, 50)] * 40), (500, [(3, 30)] * 7)], 2, 128, 64, "bf16")
    q = s.q(8, "bf16")
    first = None
    for _ in range(5):
        out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device=DEV)
        engine.attn_shared_dev(s.cache, s.batch, s.shared, q, out, lse=lse)
        engine.sync()
        first = first or (out, lse)
        assert torch.equal(out, first[0]) and torch.equal(lse, first[1])


def test_forked_pages(engine):
    """As a server uses them together: a prompt goes in, is forked, every continuation gets a token (turned and
    stored), and attends; then one is dropped, the pool compacted, and they go on."""
    page, heads, kv_heads, dim, n_slots = 16, 8, 2, 64, 6
    g = torch.Generator(device=DEV).manual_seed(3)
    pool = [torch.zeros(64, kv_heads, page, dim, device=DEV, dtype=torch.float16) for _ in range(2)]
    cache = hb.KvCache(*pool)
    table, kv_len, refs = (torch.zeros(n, dtype=torch.int32, device=DEV) for n in ((n_slots, 10), n_slots, 64))
    pages = hb.KvPages([cache], table, kv_len, refs)
    rope = hb.Rope(dim, base=1000.0)
    engine.kv_resize_dev(pages, ints([5, 0]), ints([40, 101]))  # a conversation that will end, and the prompt

    def rows(n, h):
        return torch.randn(n, h, dim, generator=g, device=DEV)

    def step(new, shared):
        n = sum(new)
        batch = hb.KvBatch(table, ints([0] + new).cumsum(0).to(torch.int32), kv_len, n)
        q, k, v = rows(n, heads), rows(n, kv_heads), rows(n, kv_heads)
        qt = torch.empty_like(q)
        engine.kv_append_rope_dev(cache, batch, rope, q, k, v, qt)
        a, b = torch.empty_like(q), torch.empty_like(q)
        engine.attn_shared_dev(cache, batch, shared, qt, a)
        engine.attn_paged_dev(cache, batch, qt, b)
        engine.sync()
        # both are within 2^-13 (A + |out|) of the definition, and |out| <= A <= the largest value there
        most = max(p.abs().max().item() for p in pool)
        assert (a - b).abs().max().item() <= 4 * 2.0 ** -13 * most
        return a

    nobody = hb.KvShared(ints([0]), ints([]))
    step([101, 0, 0, 0, 0, 40], nobody)
    engine.kv_fork_dev(pages, ints([0] * 4), ints([1, 2, 3, 4]))
    family = hb.KvShared(ints([0, 5]), ints([101]), least=1)
    for _ in range(3):
        engine.kv_resize_dev(pages, ints([0, 1, 2, 3, 4]), kv_len[:5] + 1)
        step([1] * 5 + [0], family)
    before = [pool[0][table[2, p // page].long(), :, p % page].clone() for p in range(104)]
    engine.kv_resize_dev(pages, ints([5, 3]), ints([0, 0]))
    engine.kv_compact_dev(pages)
    engine.sync()
    used = int((refs > 0).sum())
    assert used == 6 + 4 and not refs[used:].any()
    assert all(torch.equal(before[p], pool[0][table[2, p // page].long(), :, p % page]) for p in range(104))
    engine.kv_resize_dev(pages, ints([0, 1, 2, 4]), kv_len[:5][torch.tensor([0, 1, 2, 4], device=DEV)] + 1)
    step([1, 1, 1, 0, 1, 0], family)


def test_streams_and_captured_graphs(engine):
    """A captured call follows lengths that change, its workspace is its own: direct calls, larger ones on the same
    stream and on another, and a larger capture between replays do not reach it."""
    small, large = Groups([(200, [(1, 30)] * 10)], 2, 64, 16, "bf16"), Groups([(900, [(4, 40)] * 60)], 2, 64, 16, "bf16", seed=2)
    q, Q = small.q(8, "bf16"), large.q(8, "bf16")
    out, big, aside = torch.empty_like(q), torch.empty_like(Q), torch.empty_like(Q)
    stream, other = torch.cuda.Stream(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs = []
    for s, x, y in ((small, q, out), (large, Q, big)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            engine.set_stream(torch.cuda.current_stream())
            engine.attn_shared_dev(s.cache, s.batch, s.shared, x, y)
        graphs.append(graph)
    expect = [s.attention(x) for s, x in ((small, q), (large, Q))]
    lse = torch.empty(Q.shape[:2], device=DEV)
    for _ in range(3):
        for graph, y in zip(graphs, (out, big)):
            y.fill_(math.nan)
            aside.fill_(math.nan)
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                graph.replay()
            engine.set_stream(other)
            engine.attn_shared_dev(large.cache, large.batch, large.shared, Q, aside, lse=lse)
            torch.cuda.synchronize()
            close(large, "bf16", aside, lse, expect[1])
        for y, want in zip((out, big), expect):
            assert ((y.double() - want[0]).abs() <= 2.0 ** -8 * (want[2] + want[0].abs())).all()
    small.kv_len -= 5
    small.kv = [k - 5 for k in small.kv]
    graphs[0].replay()
    torch.cuda.synchronize()
    want = small.attention(q)
    assert ((out.double() - want[0]).abs() <= 2.0 ** -8 * (want[2] + want[0].abs())).all()
    engine.set_stream(torch.cuda.current_stream())


@pytest.mark.parametrize("starts,length", [([0, 9, 10], [5, 5]), ([-1, 2, 5], [5, 5]), ([3, 2, 5], [5, 5]), ([0, 3, 5], [-1, 5]),
                                           ([0, 3, 5], [5, 2**31 - 1]), ([0, 2**31 - 1, -2**31], [5, 5])])
def test_groups_out_of_range_are_reported(engine, starts, length):
    s = Groups([(37, [(1, 1), (2, 3), (1, 40)]), (20, [(1, 4), (1, 1)])], 2, 64, 16, "f16")
    q = s.q(4, "f16")
    out = torch.empty_like(q)
    engine.attn_shared_dev(s.cache, s.batch, hb.KvShared(ints(starts), ints(length), 0, 1), q, out)
    with pytest.raises(hb.CudaError, match="out of range"):
        engine.sync()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_what_sharing_has_to_save(engine, dtype):
    """Two groups of five save 4 * 300 + 4 * 100 tokens: up to there it is made, past it not; by the library's rule it is
    not.  All are the same results, and bit for bit where nothing is shared."""
    s = Groups([(300, [(1, 30)] * 5), (100, [(2, 9)] * 5)], 2, 64, 16, "bf16")
    q = s.q(8, dtype)
    plain, lse = torch.empty_like(q), torch.empty(q.shape[:2], device=DEV)
    engine.attn_paged_dev(s.cache, s.batch, q, plain, lse=lse)
    got = [check(engine, s, 8, dtype, q=q, shared=hb.KvShared(s.starts, s.length, least=n))[0] for n in (1, 1600, 1601, 10**30, 0)]
    assert torch.equal(got[0], got[1]) and not torch.equal(got[1], got[2])
    assert all(torch.equal(g, plain) for g in got[2:])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("page", [-1, 10**6, 2**31 - 1, -2**31])
@pytest.mark.parametrize("where", ["prefix", "own"])
def test_pages_out_of_range_are_reported(engine, dtype, page, where):
    s = Groups([(64, [(1, 20)] * 20)], 2, 64, 16, "bf16")
    s.table[0 if where == "prefix" else 3, 1 if where == "prefix" else 4] = page
    q = s.q(4, dtype)
    engine.attn_shared_dev(s.cache, s.batch, s.shared, q, torch.empty_like(q))
    with pytest.raises(hb.CudaError, match="out of range"):
        engine.sync()


def test_shared_refusals(engine):
    s = Groups(CASES["two"], 2, 64, 16, "f16")
    q = s.q(4, "f16")
    out = torch.empty_like(q)
    with pytest.raises(ValueError, match="one type"):
        engine.attn_shared_dev(s.cache, s.batch, s.shared, q, out.float())
    with pytest.raises(hb.CudaError, match="query heads"):
        engine.attn_shared_dev(s.cache, s.batch, s.shared, q[:, :3], out[:, :3])
    with pytest.raises(hb.CudaError, match="finite"):
        engine.attn_shared_dev(s.cache, s.batch, s.shared, q, out, scale=math.inf)
    with pytest.raises(ValueError, match="lse"):
        engine.attn_shared_dev(s.cache, s.batch, s.shared, q, out, lse=torch.empty(2, 3, device=DEV))
    with pytest.raises(ValueError, match="n_groups"):
        hb.KvShared(s.starts, s.starts)
    with pytest.raises(ValueError, match="int32"):
        hb.KvShared(s.starts.long(), s.length)
    with pytest.raises(hb.CudaError, match="2049 groups"):
        engine.attn_shared_dev(s.cache, s.batch, hb.KvShared(ints([0] * 2050), ints([0] * 2049)), q, out)
    empty = hb.KvBatch(s.table[:0], s.q_start[:1], s.kv_len[:0], 0)
    engine.attn_shared_dev(s.cache, empty, hb.KvShared(ints([0]), ints([])), q[:0], out[:0])
    engine.sync()


@pytest.mark.parametrize("dtype,cache", [("f32", "f16"), ("bf16", "bf16"), ("f16", "i8")])
@pytest.mark.parametrize("new", [[2, 0, 2, 1], [100, 0, 100, 3], [7, 0, 1, 60]])
def test_offsets_that_do_not_ascend_are_reported(engine, dtype, cache, new):
    """A group whose sequences have rows before its first one's shares nothing: rows are those of the sequences by
    themselves, and no others are written."""
    s = Groups([(300, [(n, n + 5) for n in new])], 2, 64, 16, cache)
    q = s.q(8, dtype)
    first = sum(new) - new[0] - new[3]
    starts = [first, first + new[0], 0, new[2], new[2]]  # the first sequence's rows lie behind the third's; the last has none
    batch = hb.KvBatch(s.table, ints(starts), s.kv_len, s.rows, max(new))
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device=DEV)
    engine.attn_shared_dev(s.cache, batch, s.shared, q, out, lse=lse)
    with pytest.raises(hb.CudaError, match="out of range"):
        engine.sync()
    order = torch.cat([torch.arange(first, first + new[0]), torch.arange(new[2])]).to(DEV)
    s.new = [new[0], 0, new[2], 0]
    close(s, dtype, out[order], lse[order], s.attention(q[order]))
    assert (out[first + new[0]:] == 7).all() and (lse[first + new[0]:] == 7).all()


@pytest.mark.parametrize("dtype,hint", [("f32", 0), ("bf16", 1)])
def test_a_long_chunk_beside_single_tokens(engine, dtype, hint):
    """Rows behind the prefixes that go to the kernel for few rows, of a long sequence and of short ones (16-bit rows
    where the hint says single tokens): all of them are joined."""
    for kv_heads, heads in ((2, 8), (32, 32)):
        s = Groups([(70, ONE * 3 + [(700, 720)] + [(1, 30)] * 5), (40, [(333, 333), (1, 1)]), (0, [(90, 90)])], kv_heads, 64, 16, "f16")
        s.batch = hb.KvBatch(s.table, s.q_start, s.kv_len, s.rows, hint)
        check(engine, s, heads, dtype, shared=hb.KvShared(s.starts, s.length, least=1))


def test_a_chunk_of_millions_of_rows_beside_as_many_sequences_as_there_can_be(engine):
    """2048 sequences, one of them of 8192 tokens: 1024 heads make 2^23 rows of that one alone.  Every row is written, and
    as the paged attention has it: both are within 2^-13 (A + |out|) of the definition, and |out| <= A <= the largest value."""
    s = Groups([(20, ONE * 2047 + [(8192, 8192)])], 1, 64, 64, "f16")
    q = s.q(1024, "f32", scale=0.5)
    out, plain = torch.full_like(q, math.nan), torch.empty_like(q)
    lse, plain_lse = (torch.full(q.shape[:2], math.nan, device=DEV) for _ in range(2))
    engine.attn_shared_dev(s.cache, s.batch, s.shared, q, out, lse=lse)
    engine.attn_paged_dev(s.cache, s.batch, q, plain, lse=plain_lse)
    engine.sync()
    most = s.pool[1].nan_to_num().abs().max().item()
    assert ((out - plain).abs() <= 4 * 2.0 ** -13 * most).all()
    assert ((lse - plain_lse).abs() <= 2 * (2.0 ** -12 + plain_lse.abs() * 2.0 ** -20)).all()


@pytest.mark.parametrize("captured", [False, True])
def test_without_room_for_its_parts_nothing_is_shared(engine, captured):
    """Where the workspace cannot be had the call is the paged attention's, bit for bit; once there is room it shares."""
    s = Groups([(200, [(2, 30)] * 2048)], 4, 64, 16, "f16")
    q = s.q(256, "f16")
    assert q.shape[0] * 256 * 2 * 66 * 4 > 500 << 20  # two results and sums of a row, at least
    out, plain = torch.empty_like(q), torch.empty_like(q)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    engine.set_stream(stream)

    def call():
        if not captured:
            engine.attn_shared_dev(s.cache, s.batch, s.shared, q, out)
            return None
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            engine.attn_shared_dev(s.cache, s.batch, s.shared, q, out)
        graph.replay()
        return graph

    engine.attn_paged_dev(s.cache, s.batch, q, plain)  # its code is there, and the part of the workspace that both have
    small = Groups([(200, [(2, 30)] * 2)], 4, 64, 16, "f16")
    x = small.q(4, "f16")
    engine.attn_shared_dev(small.cache, small.batch, small.shared, x, torch.empty_like(x))
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    filler = torch.empty(torch.cuda.mem_get_info()[0] - (400 << 20), dtype=torch.uint8, device=DEV)
    graph = call()
    torch.cuda.synchronize()
    assert torch.equal(out, plain)
    del filler, graph
    torch.cuda.empty_cache()
    graph = call()
    torch.cuda.synchronize()
    assert not torch.equal(out, plain)
    most = s.pool[1].nan_to_num().abs().max().item()
    assert ((out.double() - plain.double()).abs() <= 4 * 2.0 ** -10 * most).all()
    del graph
    engine.sync()
    engine.set_stream(torch.cuda.current_stream())


@pytest.mark.parametrize("dtype,cache,new", [("f16", "i8", 1), ("bf16", "bf16", 3), ("f32", "f16", 2)])
@pytest.mark.parametrize("heads,dim", [(64, 64), (512, 128)])
def test_the_workspace_is_as_large_as_it_is_said_to_be(engine, dtype, cache, new, heads, dim):
    s = Groups([(500, [(new, 9)] * 700)], 2, dim, 16, cache)
    q = s.q(heads, dtype)
    out = torch.empty_like(q)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    engine.set_stream(stream)
    engine.attn_paged_dev(s.cache, s.batch, q, out)
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    engine.attn_shared_dev(s.cache, s.batch, s.shared, q, out)
    torch.cuda.synchronize()
    took = before - torch.cuda.mem_get_info()[0]
    most = (4.5 if dtype == "bf16" else 3.5) * s.rows * heads * (dim + 2) * 4 + (21 << 20)
    least = 1 << 20
    while least < most:
        least *= 2
    if least > 256 << 20:
        least = min(n for n in range(4, 9) if n * least / 8 >= most) * least // 8
    assert took <= least + (2 << 20)  # the driver's pages
    engine.set_stream(torch.cuda.current_stream())


def laid_out(x, order, fill):
    """The same pool [page][head][row][dim] in memory of another order or with room between its parts."""
    n, h, r, d = x.shape
    if order == "rows of all heads":  # [page][row][head]
        return x.transpose(1, 2).contiguous().transpose(1, 2)
    if order == "heads apart":  # [head][page][row]
        return x.transpose(0, 1).contiguous().transpose(0, 1)
    shape, at = {"rows apart": ((n, h, r, 2 * d), (slice(None),) * 3 + (slice(d),)),
                 "pages and heads apart": ((2 * n, h + 1, r, d), (slice(1, None, 2), slice(1, None)))}[order]
    big = torch.full(shape, fill, dtype=x.dtype, device=DEV)
    big[at] = x
    return big[at]


ORDERS = ["rows of all heads", "heads apart", "rows apart", "pages and heads apart"]


@pytest.mark.parametrize("order", ORDERS)
@pytest.mark.parametrize("cache,dtype", [("i8", "bf16"), ("i8", "f16"), ("i8", "f32"), ("bf16", "bf16"), ("f16", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("dim,page,kv_heads", [(64, 16, 2), (128, 24, 2), (64, 1, 64), (128, 300, 2), (128, 20, 64)])
def test_pools_of_other_orders(engine, order, cache, dtype, dim, page, kv_heads):
    """Bit for bit what the contiguous pool gives: chunks and single tokens, prefixes of several units and pages."""
    heads = max(kv_heads, 8)
    s = Groups([(333, [(1, 1), (9, 40), (1, 150)]), (130, [(2, 2), (60, 70)])], kv_heads, dim, page, cache)
    q = s.q(heads, dtype)
    for hint in (0, 1):  # 1: what is behind the prefixes goes to the kernel for few rows
        s.batch = hb.KvBatch(s.table, s.q_start, s.kv_len, s.rows, hint)
        plain = s.cache
        want = check(engine, s, heads, dtype, q=q)
        scale = []
        for x in s.scale:
            if x is not None:
                wide = torch.full((x.shape[0], x[0].numel() + 5), math.nan, device=DEV)
                wide[:, 3:-2] = x.flatten(1)
                x = wide[:, 3:-2].unflatten(1, x.shape[1:])
            scale.append(x)
        s.cache = hb.KvCache(*(laid_out(x, order, 77 if cache == "i8" else math.nan) for x in s.pool), *scale)
        got = check(engine, s, heads, dtype, q=q)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        s.cache = plain


@pytest.mark.parametrize("dtype,cache,groups,hint,made", [
    ("bf16", "bf16", [(16384, [(256, 356)] * 8)], 0, False),  # full tiles: nothing but reading from L2 to save
    ("bf16", "bf16", [(16384, [(17, 117)] * 8)], 0, True),
    ("bf16", "bf16", [(2048, [(17, 117)] * 4)], 0, False),
    ("bf16", "i8", [(65536, [(1, 101)] * 4)], 1, False),  # the prefix's units cost more than three readings
    ("bf16", "i8", [(65536, [(1, 101)] * 8)], 1, True),
    ("f16", "f16", [(16384, [(1, 101)] * 4)], 1, False),
    ("f16", "f16", [(16384, [(1, 101)] * 16)], 1, True),
    ("f32", "bf16", [(16384, [(16, 116)] * 16)], 16, False),  # 64 rows each: as many tiles of 16 together
    ("f32", "bf16", [(16384, [(1, 101)] * 16)], 1, True),
    ("f32", "i8", [(16384, [(5, 105)] * 8)], 5, True)])
def test_the_rule_on_what_is_shared(engine, dtype, cache, groups, hint, made):
    """Sharing is left where it would be slower, and made on the other side of the rule: the paged attention's bits tell."""
    s = Groups(groups, 8, 128, 64, cache)
    s.batch = hb.KvBatch(s.table, s.q_start, s.kv_len, s.rows, hint)
    q = s.q(32, dtype)
    out, plain = torch.empty_like(q), torch.empty_like(q)
    engine.attn_shared_dev(s.cache, s.batch, hb.KvShared(s.starts, s.length), q, out)
    engine.attn_paged_dev(s.cache, s.batch, q, plain)
    engine.sync()
    assert torch.equal(out, plain) != made
    c = 2.0 ** -13 if dtype == "f32" else 2.0 ** -10 if dtype == cache == "f16" else 2.0 ** -8
    v = s.pool[1].float() if cache != "i8" else s.pool[1].float() * s.scale[1][..., None]
    assert ((out.double() - plain.double()).abs() <= 4 * c * v.nan_to_num().abs().max().item()).all()


@pytest.mark.parametrize("dtype,cache,hint", [("f32", "i8", 0), ("f32", "bf16", 1), ("bf16", "i8", 1), ("f16", "f16", 1), ("bf16", "bf16", 0)])
@pytest.mark.parametrize("heads,kv_heads", [(6, 2), (4, 4), (64, 64), (96, 48)])
def test_scale_and_strided_rows_of_the_other_kernels(engine, dtype, cache, hint, heads, kv_heads):
    """f32 rows, and single tokens behind prefixes: rows apart, any scale, with a log-sum-exp and without."""
    s = Groups([(90, ONE * 4 + [(1, 33), (3, 20)]), (0, [(2, 9)]), (160, [(1, 1), (1, 70)])], kv_heads, 64, 16, cache)
    s.batch = hb.KvBatch(s.table, s.q_start, s.kv_len, s.rows, hint)
    buf = torch.randn(s.rows, 3, heads, 64, generator=s.g, device=DEV).to(T[dtype])
    q = buf[:, 1]
    for scale in (0.3, -0.2, 0.0, None):
        out, lse = torch.full((s.rows, 2, heads, 64), 7.0, device=DEV).to(T[dtype]), torch.empty(s.rows, heads, device=DEV)
        engine.attn_shared_dev(s.cache, s.batch, s.shared, q, out[:, 1], scale=scale, lse=lse)
        engine.sync()
        close(s, dtype, out[:, 1], lse, s.attention(q, scale))
        again = torch.empty_like(out)
        engine.attn_shared_dev(s.cache, s.batch, s.shared, q, again[:, 1], scale=scale)
        engine.sync()
        assert (out[:, 0] == 7).all() and torch.equal(again[:, 1], out[:, 1])


@pytest.mark.parametrize("dtype,cache,hint", [("f32", "i8", 0), ("bf16", "i8", 1), ("f16", "f16", 0)])
def test_one_graph_through_sharing_and_none(engine, dtype, cache, hint):
    """A captured call whose lengths change between replays: groups that share, that share nothing any more, sequences that
    go; two streams' direct calls between them."""
    s = Groups([(300, [(1, 40)] * 9), (64, [(1, 8), (1, 30)])], 2, 64, 16, cache)
    s.batch = hb.KvBatch(s.table, s.q_start, s.kv_len, s.rows, hint)
    shared = hb.KvShared(s.starts, s.length, least=500)
    q = s.q(8, dtype)
    out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device=DEV)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        engine.set_stream(torch.cuda.current_stream())
        engine.attn_shared_dev(s.cache, s.batch, shared, q, out, lse=lse)
    kv = list(s.kv)
    for lengths, cut in (([300, 64], 0), ([50, 0], 0), ([300, 64], 30), ([0, 0], 0), ([300, 64], 0)):
        s.length.copy_(ints(lengths))
        s.kv = [k - cut if i else k for i, k in enumerate(kv)]
        s.kv = [max(k, 1) for k in s.kv]
        s.kv_len.copy_(ints(s.kv))
        out.fill_(math.nan), lse.fill_(math.nan)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        close(s, dtype, out, lse, s.attention(q))
        first = out.clone()
        for st in (torch.cuda.Stream(), torch.cuda.Stream()):
            engine.set_stream(st)
            direct = torch.empty_like(q)
            torch.cuda.synchronize()
            engine.attn_shared_dev(s.cache, s.batch, shared, q, direct)
            torch.cuda.synchronize()
            assert torch.equal(direct, first)
    engine.set_stream(torch.cuda.current_stream())


@pytest.mark.parametrize("case", list(CASES))
@pytest.mark.parametrize("cache,dtype", [("i8", "bf16"), ("i8", "f16"), ("f16", "f16"), ("f16", "bf16"), ("bf16", "bf16")])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(96, 96, 64, 16), (180, 60, 64, 24), (64, 64, 128, 100)])
def test_groups_of_more_tiles_than_blocks(engine, case, cache, dtype, heads, kv_heads, dim, page):
    """So many kv heads that what is behind the prefixes goes to the kernel for few rows, whatever sequences have more."""
    s = Groups(CASES[case], kv_heads, dim, page, cache)
    s.batch = hb.KvBatch(s.table, s.q_start, s.kv_len, s.rows, 1)
    check(engine, s, heads, dtype)


@pytest.mark.parametrize("dtype,cache", [("bf16", "i8"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("at", ["prefix", "own"])
def test_not_finite_behind_many_tiles(engine, dtype, cache, at):
    s = Groups([(40, [(1, 20)] * 3), (50, [(1, 9)] * 2)], 64, 64, 16, cache)
    page = s.table[0, 1] if at == "prefix" else s.table[1, 3]
    if cache == "i8":
        s.scale[1][page.long(), 0, 2] = math.inf
    else:
        s.pool[1][page.long(), 0, 2, :] = math.inf
    q = s.q(64, dtype)
    out = torch.zeros_like(q)
    engine.attn_shared_dev(s.cache, s.batch, s.shared, q, out)
    engine.sync()
    bad = ~out.isfinite().all(-1)
    assert bad[:, 0].tolist() == ([True] * 3 if at == "prefix" else [False, True, False]) + [False, False]
    assert not bad[:, 1:].any()
