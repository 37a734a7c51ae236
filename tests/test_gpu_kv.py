"""GPU tests of the paged key/value cache (kv_append_dev, kv_read_dev) and of the attention over it
(attn_paged_dev) against their definitions in 64 bits.

Tolerances, from the number formats alone (u = half a unit in the last place, A_i = sum_j p_ij |v_j|,
which every rounding of a weight p_ij or of a product is relative to):
  * cache: codes and scales exactly; values read back exactly (one rounding of code * scale);
  * attention in 16 bits: the weights are rounded to at most 8 significant bits (u = 2^-9), the
    result to its type (2^-9 or 2^-12): |err| <= 2^-8 (A + |out|); where both the cache and the rows
    are float16 the weights keep 11 bits: 2^-10 (A + |out|);
  * attention in 32 bits: weights of at least 16 bits (2^-17), scores of 22 bits or more with f32
    sums of up to 128 products (128 * 2^-24 of sum |q k| scale, about 16 here): 2^-13 (A + |out|)
    holds elementwise at worst, 1e-5 in the 2-norm, where errors of random sign average out;
  * lse: the scores' error, 128 * 2^-24 * 16 < 2^-12, and f32's own of |lse|.
"""
import math

import pytest
import torch

import hayai_b200 as hb
from hayai_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}


@pytest.fixture(autouse=True)
def _stream(engine):
    engine.set_stream(torch.cuda.current_stream())
    yield
    engine.sync()
    engine.set_stream(None)


def quantised(x):
    scale = x.abs().amax(-1) / 127.0
    codes = torch.where(scale[..., None] > 0, (x / scale[..., None]).round().clamp(-127, 127), torch.zeros_like(x))
    return codes.to(torch.int8), scale


class Setup:
    """A pool with shuffled pages, of which the slots that no token has hold NaN (16-bit) or NaN scales."""

    def __init__(self, lens, kv_heads, dim, page, cache, seed=1, order="phrd", extra=2, spread=1.0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.new, self.kv = [a for a, _ in lens], [b for _, b in lens]
        self.page, self.kv_heads, self.dim, self.type = page, kv_heads, dim, cache
        need = [-(-max(k, 0) // page) for k in self.kv]
        self.n_pages = sum(need) + extra
        perm = torch.randperm(self.n_pages, generator=g, device=DEV, dtype=torch.int32)
        self.table = torch.full((len(lens), max(need + [1])), -7, dtype=torch.int32, device=DEV)
        used = torch.zeros(self.n_pages, page, dtype=torch.bool, device=DEV)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = perm[at:at + n]
            pos = torch.arange(max(self.kv[i], 0), device=DEV)
            used[self.table[i].long()[pos // page], pos % page] = True
            at += n
        shape = (self.n_pages, kv_heads, page, dim)
        self.pool, self.scale = [], []
        for w in range(2):
            x = torch.randn(shape, generator=g, device=DEV) * spread
            if cache == "i8":
                c, s = quantised(x)
                s[~used[:, None].expand(s.shape)] = math.nan
            else:
                c, s = x.to(T[cache]), None
                c[~used[:, None, :, None].expand(c.shape)] = math.nan
            if order == "prhd":  # rows of all heads together
                c = c.transpose(1, 2).contiguous().transpose(1, 2)
            elif order == "both":  # k and v of a page side by side, in a pool of three layers
                big = torch.zeros((self.n_pages, 3, 2) + shape[1:], dtype=c.dtype, device=DEV)
                big[:, 1, w] = c
                c = big[:, 1, w]
            self.pool.append(c)
            self.scale.append(s)
        self.q_start = torch.tensor([0] + self.new, device=DEV).cumsum(0).to(torch.int32)
        self.kv_len = torch.tensor(self.kv, dtype=torch.int32, device=DEV)
        self.rows = sum(self.new)
        self.g = g
        self.cache = hb.KvCache(*self.pool, *self.scale)
        self.batch = hb.KvBatch(self.table, self.q_start, self.kv_len, self.rows, max(self.new + [0]))

    def q(self, heads, dtype, scale=1.0):
        return (torch.randn(self.rows, heads, self.dim, generator=self.g, device=DEV) * scale).to(T[dtype])

    def values(self, w, i, lo, hi):
        pos = torch.arange(lo, hi, device=DEV)
        p, r = self.table[i].long()[pos // self.page], pos % self.page
        x = self.pool[w][p, :, r].double()
        return x if self.scale[w] is None else x * self.scale[w][p, :, r].double()[..., None]

    def attention(self, q, scale=None, causal=True, window=0, sink=0):
        """(out, lse, A) in 64 bits."""
        scale = self.dim ** -0.5 if scale is None else scale
        heads = q.shape[1]
        group = heads // self.kv_heads
        out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
        amp = torch.zeros_like(out)
        lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=DEV)
        done = 0
        for i, (n, k) in enumerate(zip(self.new, self.kv)):
            if n and k > 0:
                K, V = self.values(0, i, 0, k), self.values(1, i, 0, k)
                ip = torch.arange(k - n, k, device=DEV).view(n, 1)
                jp = torch.arange(k, device=DEV).view(1, k)
                see = (jp <= ip) if causal else torch.ones(n, k, dtype=torch.bool, device=DEV)
                if window:
                    see = see & ((ip - jp < window) | (jp < sink))
                for h in range(heads):
                    s = (q[done:done + n, h].double() @ K[:, h // group].T) * scale
                    s = torch.where(see, s, -math.inf)
                    m = s.amax(-1, keepdim=True)
                    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
                    p = torch.where(see, (s - m).exp(), torch.zeros_like(s))
                    tot = p.sum(-1, keepdim=True)
                    w = torch.where(tot > 0, p / tot, torch.zeros_like(p))
                    vis = see.any(0)  # a value that no row sees is not looked at
                    v = torch.where(vis[:, None], V[:, h // group], torch.zeros_like(V[:, 0]))
                    out[done:done + n, h] = w @ v
                    amp[done:done + n, h] = w @ v.abs()
                    lse[done:done + n, h] = (m + tot.log()).squeeze(-1)
            done += n
        return out, lse, amp


def check(engine, s, heads, dtype, q=None, **kw):
    q = s.q(heads, dtype) if q is None else q
    out = torch.full_like(q, math.nan)
    lse = torch.full(q.shape[:2], math.nan, device=DEV)
    engine.attn_paged_dev(s.cache, s.batch, q, out, lse=lse, **kw)
    engine.sync()
    ref, ref_lse, amp = s.attention(q, **kw)
    got = out.double()
    c = 2.0 ** -13 if dtype == "f32" else 2.0 ** -10 if dtype == s.type == "f16" else 2.0 ** -8
    assert torch.isfinite(got).all()
    worst = ((got - ref).abs() - c * (amp + ref.abs())).max().item() if got.numel() else 0.0
    assert worst <= 1e-30, f"off by {worst} more than its bound"
    if dtype == "f32" and got.numel():
        rel = ((got - ref).norm() / ref.norm().clamp_min(1e-300)).item()
        assert rel <= 1e-5, rel
    none = ref_lse == -math.inf
    assert torch.equal(lse == -math.inf, none) and (got[none] == 0).all()
    off = (lse.double() - ref_lse)[~none].abs() - 2.0 ** -12 - ref_lse[~none].abs() * 2.0 ** -20
    assert not off.numel() or off.max().item() <= 0, off.max().item()
    return out, lse


# ------------------------------------------------------------------ the cache
LENS = [(1, 1), (3, 3), (0, 0), (1, 40), (17, 100), (0, 9), (5, 5)]


@pytest.mark.parametrize("cache", ["i8", "f16", "bf16"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,kv_heads,page,order", [(64, 3, 16, "phrd"), (128, 8, 24, "prhd"), (128, 1, 1, "phrd"),
                                                     (64, 5, 100, "both")])
def test_append_then_read(engine, cache, dtype, dim, kv_heads, page, order):
    s = Setup(LENS, kv_heads, dim, page, cache, order=order)
    before = [p.clone() for p in s.pool]
    x = [(torch.randn(s.rows, kv_heads, dim, generator=s.g, device=DEV) * 10 ** w).to(T[dtype]) for w in (0, 1)]
    x[0][2] = 0  # a row of zeros
    if dtype == "f32":
        x[1][4, 0] = 1e-44  # a scale that is not a normal number
    engine.kv_append_dev(s.cache, s.batch, *x)
    back = [torch.full_like(t, math.nan) for t in x]
    engine.kv_read_dev(s.cache, s.batch, *back)
    engine.sync()
    written = torch.zeros(s.n_pages, page, dtype=torch.bool, device=DEV)
    done = 0
    for i, (n, k) in enumerate(zip(s.new, s.kv)):
        pos = torch.arange(k - n, k, device=DEV)
        p, r = s.table[i].long()[pos // page], pos % page
        written[p, r] = True
        for w in range(2):
            v = x[w][done:done + n].float()
            if cache == "i8":
                codes, scale = quantised(v)
                assert torch.equal(s.pool[w][p, :, r], codes) and torch.equal(s.scale[w][p, :, r], scale)
                v = codes.float() * scale[..., None]
            else:
                v = v.to(T[cache])
                assert torch.equal(s.pool[w][p, :, r], v)
            assert torch.equal(back[w][done:done + n], v.float().to(T[dtype]))
        done += n
    for w in range(2):  # nothing else is touched
        rest = ~written[:, None, :, None].expand(before[w].shape)
        a, b = s.pool[w][rest].float(), before[w][rest].float()
        assert torch.equal(a.nan_to_num(7e4), b.nan_to_num(7e4))


def test_rows_that_are_not_finite_read_back_as_nan(engine):
    s = Setup([(4, 4)], 2, 64, 16, "i8")
    x = s.q(2, "f32")
    x[1, 0, 3], x[2, 1, 9] = math.nan, -math.inf
    engine.kv_append_dev(s.cache, s.batch, x, x)
    back = [torch.zeros_like(x) for _ in range(2)]
    engine.kv_read_dev(s.cache, s.batch, *back)
    engine.sync()
    bad = torch.zeros(4, 2, dtype=torch.bool, device=DEV)
    bad[1, 0] = bad[2, 1] = True
    for b in back:
        assert b[bad].isnan().all() and b[~bad].isfinite().all()


def test_packed_projection_rows(engine):
    """q, k and v as slices of one projection's rows [n_tok][(heads + 2 kv_heads) * dim]."""
    s = Setup([(5, 70), (2, 2)], 2, 64, 16, "i8", extra=3)
    qkv = torch.randn(s.rows, 8, 64, generator=s.g, device=DEV)
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    engine.kv_append_dev(s.cache, s.batch, k, v)
    wide = torch.full((s.rows, 6, 64), math.nan, device=DEV)
    ref, _, amp = s.attention(q)
    engine.attn_paged_dev(s.cache, s.batch, q, wide[:, 1:5])
    engine.sync()
    assert ((wide[:, 1:5].double() - ref).abs() <= 2.0 ** -13 * (amp + ref.abs()) + 1e-30).all()
    assert wide[:, 0].isnan().all() and wide[:, 5].isnan().all()


# ------------------------------------------------------------------ attention
ODD = [(1, n) for n in (1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1000)] + [(0, 0), (0, 5)]


@pytest.mark.parametrize("cache", ["i8", "f16", "bf16"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(9, 3, 64, 16), (32, 8, 128, 16), (16, 2, 128, 64), (5, 1, 128, 1),
                                                     (2, 2, 64, 100), (40, 2, 64, 24)])
def test_single_tokens(engine, cache, dtype, heads, kv_heads, dim, page):
    check(engine, Setup(ODD, kv_heads, dim, page, cache), heads, dtype)


CHUNKS = {"one": [(130, 130)], "tail": [(64, 500), (1, 300), (0, 0), (257, 1000)], "few": [(2, 40), (5, 600), (9, 9), (3, 129)],
          "mixed": [(1, 77), (300, 300), (1, 1), (33, 2000), (1, 700), (128, 128), (129, 385)]}


@pytest.mark.parametrize("cache", ["i8", "f16", "bf16"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens", list(CHUNKS))
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 1, 128, 16), (6, 2, 64, 24), (8, 8, 128, 64)])
def test_chunks(engine, cache, dtype, lens, heads, kv_heads, dim, page):
    check(engine, Setup(CHUNKS[lens], kv_heads, dim, page, cache), heads, dtype)


@pytest.mark.parametrize("cache,dtype", [("i8", "f32"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("window,sink", [(1, 0), (16, 4), (100, 1), (128, 130), (5000, 3), (37, 10000)])
@pytest.mark.parametrize("dim", [64, 128])
def test_window_and_first_tokens(engine, cache, dtype, window, sink, dim):
    check(engine, Setup(CHUNKS["mixed"] + [(1, 1500), (4, 260)], 2, dim, 16, cache), 8, dtype, window=window, sink=sink)


@pytest.mark.parametrize("cache,dtype", [("i8", "f16"), ("f16", "f32"), ("bf16", "bf16")])
def test_every_position_seen(engine, cache, dtype):
    check(engine, Setup(CHUNKS["mixed"], 2, 128, 32, cache), 4, dtype, causal=False)


@pytest.mark.parametrize("cache,dtype", [("i8", "f32"), ("bf16", "f32"), ("f16", "f16"), ("i8", "bf16")])
def test_tokens_before_the_first_position_see_nothing(engine, cache, dtype):
    """More new tokens than the sequence holds: the first ones have no position, and rows 0 / -inf."""
    out, lse = check(engine, Setup([(6, 2), (140, 10), (3, 0), (1, 5)], 2, 64, 16, cache), 4, dtype)
    assert (lse[:4] == -math.inf).all() and (out[:4] == 0).all()


@pytest.mark.parametrize("cache,dtype", [("i8", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("i8", "bf16")])
@pytest.mark.parametrize("lens", [[(1, 20000)], [(40, 9001)], [(1, 5), (1, 30011), (1, 64)]])
def test_long_and_split(engine, cache, dtype, lens):
    s = Setup(lens, 2, 128, 64, cache)
    q = s.q(8, dtype)
    a = check(engine, s, 8, dtype, q=q)
    b = check(engine, s, 8, dtype, q=q)  # the same bits again
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("lens", [[(1, 3000)], [(200, 3000)]])
def test_scores_that_rise_and_fall(engine, lens):
    """Scores over hundreds, the largest late: the running maximum moves often, weights underflow."""
    for cache, dtype in (("i8", "f32"), ("f16", "f16"), ("bf16", "bf16")):
        s = Setup(lens, 1, 64, 16, cache)
        ramp = torch.linspace(0.01, 6.0, 3000, device=DEV)
        pos = torch.arange(3000, device=DEV)
        p, r = s.table[0].long()[pos // 16], pos % 16
        if cache == "i8":
            s.scale[0][p, :, r] *= ramp[:, None]
        else:
            s.pool[0][p, :, r] = (s.pool[0][p, :, r].float() * ramp[:, None, None]).to(T[cache])
        q = s.q(4, dtype)
        out = torch.empty_like(q)
        engine.attn_paged_dev(s.cache, s.batch, q, out, scale=2.0)
        ref, _, amp = s.attention(q, scale=2.0)
        # scores up to 800: 128 * 2^-24 * sum |q k| scale is up to 2^-17 * 2500 in a weight's exponent;
        # weights under f32's smallest normal (and so results made of them alone) may be flushed
        c = 2.0 ** -8 + 2500 * 2.0 ** -17
        assert ((out.double() - ref).abs() <= c * (amp + ref.abs()) + 1e-30).all(), cache


@pytest.mark.parametrize("small", [1e-6, 1e6])
def test_values_of_any_size(engine, small):
    """8-bit values whose scales differ by many orders between tokens."""
    for lens, dtype in (([(1, 700)], "f32"), ([(1, 700)], "bf16"), ([(150, 700)], "bf16"), ([(150, 700)], "f32")):
        s = Setup(lens, 2, 128, 16, "i8")
        pos = torch.arange(0, 700, 2, device=DEV)
        s.scale[1][s.table[0].long()[pos // 16], :, pos % 16] *= small
        check(engine, s, 4, dtype)


@pytest.mark.parametrize("lens", [[(5, 100)], [(130, 300)]])
@pytest.mark.parametrize("cache,dtype", [("f16", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("i8", "bf16")])
def test_not_finite_where_masked(engine, lens, cache, dtype):
    """A later new token's key and value are not finite: the tokens before it do not see them, and
    those from it on get NaN."""
    s = Setup(lens, 2, 128, 16, cache)
    n, k = lens[0]
    at = k - 3
    p, r = int(s.table[0, at // 16]), at % 16
    clean = s.attention(s.q(4, dtype))  # advances the generator alike
    s.g.manual_seed(5)
    q = s.q(4, dtype)
    ref, _, amp = s.attention(q)
    for w, bad in ((0, math.nan), (1, math.inf)):
        if cache == "i8":
            s.scale[w][p, :, r] = bad
        else:
            s.pool[w][p, :, r, ::3] = bad
    out = torch.empty_like(q)
    engine.attn_paged_dev(s.cache, s.batch, q, out)
    engine.sync()
    assert clean is not None and torch.isfinite(out[:n - 3]).all()
    assert ((out.double() - ref).abs()[:n - 3] <= (2.0 ** -8 * (amp + ref.abs()))[:n - 3]).all()
    assert out[n - 3:].isnan().any(-1).all()


@pytest.mark.parametrize("window", [70, 300])
@pytest.mark.parametrize("at", [610, 650, 767, 768])
@pytest.mark.parametrize("cache,dtype", [("f16", "f16"), ("bf16", "bf16"), ("i8", "bf16")])
def test_not_finite_outside_a_window(engine, cache, dtype, at, window):
    """One value that is not finite among units that rows see in part, one after the other: the rows
    whose window does not reach it are as without it."""
    s = Setup([(300, 900)], 2, 128, 16, cache)
    q = s.q(4, dtype)
    ref, _, amp = s.attention(q, window=window)
    p, r = int(s.table[0, at // 16]), at % 16
    if cache == "i8":
        s.scale[1][p, :, r] = math.inf
    else:
        s.pool[1][p, :, r, 5] = math.inf
    out = torch.empty_like(q)
    for _ in range(3):
        engine.attn_paged_dev(s.cache, s.batch, q, out, window=window)
        engine.sync()
        pos = torch.arange(600, 900, device=DEV)
        sees = (pos >= at) & (pos - at < window)
        assert ((out.double() - ref).abs()[~sees] <= (2.0 ** -8 * (amp + ref.abs()))[~sees]).all()
        assert not torch.isfinite(out[sees][..., 5]).any()


@pytest.mark.parametrize("order", ["prhd", "both"])
@pytest.mark.parametrize("cache,dtype", [("i8", "f32"), ("bf16", "bf16")])
def test_orders_of_the_pool(engine, order, cache, dtype):
    check(engine, Setup(CHUNKS["mixed"], 2, 64, 16, cache, order=order), 4, dtype)


def test_offsets_past_32_bits(engine):
    """A pool of 6 GiB codes: the sequence's pages lie past 4 GiB."""
    n_pages, page = 6 << 30 >> 13, 64
    k = torch.zeros(n_pages, 1, page, 128, dtype=torch.int8, device=DEV)
    sc = torch.zeros(n_pages, 1, page, device=DEV)
    table = torch.arange(n_pages - 9, n_pages, dtype=torch.int32, device=DEV).flip(0)[None]
    q_start = torch.tensor([0, 550], dtype=torch.int32, device=DEV)
    kv_len = torch.tensor([550], dtype=torch.int32, device=DEV)
    cache, batch = hb.KvCache(k, k, sc, sc), hb.KvBatch(table, q_start, kv_len, 550, 550)
    x = torch.randn(550, 1, 128, device=DEV, generator=torch.Generator(device=DEV).manual_seed(3))
    engine.kv_append_dev(cache, batch, x, x)
    back = [torch.empty_like(x) for _ in range(2)]
    engine.kv_read_dev(cache, batch, *back)
    codes, scale = quantised(x)
    v = codes.float() * scale[..., None]
    assert torch.equal(back[0], v) and torch.equal(back[1], v)
    for lo in (0, 549):
        b = hb.KvBatch(table, torch.tensor([0, 550 - lo], dtype=torch.int32, device=DEV), kv_len, 550 - lo)
        q, out = x[lo:], torch.empty_like(x[lo:])
        engine.attn_paged_dev(cache, b, q, out)
        s = (q[:, 0].double() @ v[:, 0].double().T) * 128 ** -0.5
        s = s.masked_fill(torch.arange(550, device=DEV)[None] > torch.arange(lo, 550, device=DEV)[:, None], -math.inf)
        ref = s.softmax(-1) @ v[:, 0].double()
        assert ((out[:, 0].double() - ref).norm() / ref.norm()).item() <= 1e-5


def test_another_stream_and_a_captured_graph(engine):
    """The calls run on the engine's stream, and a captured graph follows lengths changed in place."""
    s = Setup([(1, 600), (1, 90)], 2, 128, 16, "i8")
    q, out = s.q(8, "bf16"), torch.empty(2, 8, 128, dtype=torch.bfloat16, device=DEV)
    engine.attn_paged_dev(s.cache, s.batch, q, out)  # workspaces exist before the capture
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    engine.set_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        engine.attn_paged_dev(s.cache, s.batch, q, out)
    for kv in ([600, 90], [1, 33], [599, 0]):
        s.kv_len.copy_(torch.tensor(kv, dtype=torch.int32))
        s.kv = kv
        ref, _, amp = s.attention(q)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert ((out.double() - ref).abs() <= 2.0 ** -8 * (amp + ref.abs())).all()


@pytest.mark.parametrize("what", ["page", "len", "q_start"])
@pytest.mark.parametrize("new", [1, 150])
def test_device_values_out_of_range_are_reported(engine, what, new):
    s = Setup([(new, 200), (new, 250)], 2, 64, 16, "i8")
    {"page": s.table, "len": s.kv_len, "q_start": s.q_start}[what].view(-1)[1] = {"page": 1 << 20, "len": 100000,
                                                                                 "q_start": 1 << 20}[what]
    q = s.q(4, "f16")
    with pytest.raises(hb.CudaError) as e:
        engine.attn_paged_dev(s.cache, s.batch, q, torch.empty_like(q))
        engine.sync()
    assert e.value.code == _lib.HC_ERR_INVALID
    engine.sync()  # reported once


def test_empty_batches(engine):
    s = Setup([(0, 4), (0, 0)], 1, 64, 16, "f16")
    q = s.q(2, "f16")
    engine.attn_paged_dev(s.cache, s.batch, q, q)
    engine.kv_append_dev(s.cache, s.batch, q[:, :1], q[:, :1])
    none = hb.KvBatch(s.table[:0], s.q_start[:1], s.kv_len[:0], 0)
    engine.attn_paged_dev(s.cache, none, q, q)


def test_rows_of_no_sequence_are_left_alone(engine):
    s = Setup([(2, 50), (3, 80)], 1, 64, 16, "f16")
    batch = hb.KvBatch(s.table, s.q_start + 1, s.kv_len, 8, 3)
    q = torch.randn(8, 4, 64, device=DEV).half()
    out = torch.full_like(q, 7.0)
    engine.attn_paged_dev(s.cache, batch, q, out)
    ref, _, amp = s.attention(q[1:6])
    assert (out[0] == 7).all() and (out[6:] == 7).all()
    assert ((out[1:6].double() - ref).abs() <= 2.0 ** -10 * (amp + ref.abs())).all()


# ------------------------------------------------------------------ refusals
def test_refusals(engine):
    s = Setup([(2, 50)], 2, 64, 16, "i8")
    q, out, kv = s.q(4, "f16"), torch.empty(2, 4, 64, dtype=torch.float16, device=DEV), s.q(2, "f16")
    k, ks = s.pool[0], s.scale[0]
    bad = [
        lambda: hb.KvCache(k.float(), k.float()), lambda: hb.KvCache(k, k), lambda: hb.KvCache(k.half(), k.half(), ks, ks),
        lambda: hb.KvCache(k.cpu(), k.cpu(), ks, ks), lambda: hb.KvCache(k[0], k[0], ks[0], ks[0]),
        lambda: hb.KvCache(k.transpose(2, 3), k.transpose(2, 3), ks, ks),
        lambda: hb.KvBatch(s.table.long(), s.q_start, s.kv_len, 2), lambda: hb.KvBatch(s.table, s.q_start[:1], s.kv_len, 2),
        lambda: hb.KvBatch(s.table, s.q_start, s.kv_len, -1),
        lambda: engine.attn_paged_dev(s.cache, s.batch, q[:1], out[:1]),
        lambda: engine.attn_paged_dev(s.cache, s.batch, q, out.float()),
        lambda: engine.attn_paged_dev(s.cache, s.batch, q.double(), out.double()),
        lambda: engine.attn_paged_dev(s.cache, s.batch, q.cpu(), out),
        lambda: engine.attn_paged_dev(s.cache, s.batch, q, out, lse=torch.empty(2, 3, device=DEV)),
        lambda: engine.attn_paged_dev(s.cache, s.batch, q.transpose(1, 2).contiguous().transpose(1, 2), out),
        lambda: engine.kv_append_dev(s.cache, s.batch, q, q), lambda: engine.kv_read_dev(s.cache, s.batch, kv, kv.float()),
    ]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    odd = s.q(3, "f16")
    native = [
        (lambda: engine.attn_paged_dev(s.cache, s.batch, odd, torch.empty_like(odd)), _lib.HC_ERR_INVALID),
        (lambda: engine.attn_paged_dev(s.cache, s.batch, q, out, window=-1), _lib.HC_ERR_INVALID),
        (lambda: engine.attn_paged_dev(s.cache, s.batch, q, out, window=8, causal=False), _lib.HC_ERR_INVALID),
        (lambda: engine.attn_paged_dev(s.cache, s.batch, q, out, scale=math.inf), _lib.HC_ERR_INVALID),
    ]
    for dim in (32, 96, 256):
        x = torch.zeros(3, 2, 16, dim, dtype=torch.float16, device=DEV)
        c, y = hb.KvCache(x, x), torch.zeros(2, 2, dim, dtype=torch.float16, device=DEV)
        native.append((lambda c=c, y=y: engine.attn_paged_dev(c, s.batch, y, y), _lib.HC_ERR_UNSUPPORTED))
    flat = torch.zeros(1 << 16, dtype=torch.float16, device=DEV)
    c = hb.KvCache(*[flat.as_strided((3, 2, 16, 64), (4096, 2048, 72, 1))] * 2)  # rows 144 bytes apart
    native.append((lambda: engine.kv_append_dev(c, s.batch, kv, kv), _lib.HC_ERR_INVALID))
    many = hb.KvBatch(torch.zeros(5000, 1, dtype=torch.int32, device=DEV), torch.zeros(5001, dtype=torch.int32, device=DEV),
                      torch.zeros(5000, dtype=torch.int32, device=DEV), 2)
    native.append((lambda: engine.kv_append_dev(s.cache, many, kv, kv), _lib.HC_ERR_INVALID))
    skew = torch.zeros(2 * 4 * 64 + 1, dtype=torch.float16, device=DEV)[1:].view(2, 4, 64)
    native.append((lambda: engine.attn_paged_dev(s.cache, s.batch, skew, out), _lib.HC_ERR_INVALID))
    for f, code in native:
        with pytest.raises(hb.CudaError) as e:
            f()
        assert e.value.code == code, str(e.value)
    engine.sync()


@pytest.mark.parametrize("cache,dtype", [("f16", "f16"), ("bf16", "bf16"), ("f16", "bf16")])
@pytest.mark.parametrize("dim,group", [(64, 1), (128, 1), (128, 3)])
def test_not_finite_in_a_tile_after_short_ones(engine, cache, dtype, dim, group):
    """Tiles of at most 128 rows and several units, which half of a block's row threads pass over, and
    next to them tiles whose second half has rows that must not see a value that is not finite."""
    lens = [(260 // group + 13 * i % 110 // group, 520 + 37 * i % 480) for i in range(40)]
    s = Setup(lens, 4, dim, 16, cache)
    q = s.q(4 * group, dtype)
    ref, _, amp = s.attention(q)
    sees = torch.zeros(s.rows, dtype=torch.bool, device=DEV)
    done = 0
    for i, (n, k) in enumerate(lens):
        at = k - n + 250 // group  # its row is the 250th of the sequence's first tile, or near it
        s.pool[1][int(s.table[i, at // 16]), :, at % 16, 7] = math.inf
        sees[done + at - (k - n):done + n] = True
        done += n
    first = None
    for _ in range(4):
        out = torch.full_like(q, 5.0)
        engine.attn_paged_dev(s.cache, s.batch, q, out)
        engine.sync()
        assert ((out.double() - ref).abs()[~sees] <= (2.0 ** -8 * (amp + ref.abs()))[~sees]).all()
        assert not torch.isfinite(out[sees][..., 7]).any()
        assert first is None or torch.equal(out.view(torch.int16), first)
        first = out.view(torch.int16).clone()


def places(s, pos, i=0):
    return s.table[i].long()[pos // s.page], pos % s.page


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("lens,zero", [((150, 700), (0, 128)), ((150, 700), (128, 256)), ((150, 700), (0, 300)), ((150, 700), (0, 700)),
                                       ((40, 9001), (0, 4000)), ((40, 9001), (0, 9001)), ((150, 20000), (3000, 16000))])
def test_values_of_zero(engine, dtype, lens, zero):
    """Rows of zeros have scale 0: whole units of them, a block's share, a split tile, all values."""
    s = Setup([lens], 2, 128, 16, "i8")
    pos = torch.arange(*zero, device=DEV)
    p, r = places(s, pos)
    s.pool[1][p, :, r] = 0
    s.scale[1][p, :, r] = 0.0
    check(engine, s, 8, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("sizes", [(0.0, 1e-38, 1e-20, 1.0), (1e-38, 1e-38, 0.0, 1e-38), (0.0, 1e-35, 1e-30, 1e-38)])
def test_values_with_scales_near_zero(engine, dtype, sizes):
    """Scales from zero to f32's smallest, mixed in a unit; what they leave is under the bound's floor or
    beside ordinary values."""
    for lens in ((150, 700), (40, 9001)):
        s = Setup([lens], 2, 128, 16, "i8")
        for i, size in enumerate(sizes):
            pos = torch.arange(i, lens[1], len(sizes), device=DEV)
            p, r = places(s, pos)
            s.scale[1][p, :, r] *= size
        check(engine, s, 8, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("large", [2.0 ** 20, 2.0 ** 30])
@pytest.mark.parametrize("where", ["seen", "masked"])
def test_large_values_with_no_weight(engine, dtype, large, where):
    """A token that has nearly all weight beside one of a far larger value that has next to none of it (a weight
    of e^-56); and one of a far larger value that all rows but the last are masked from."""
    s = Setup([(150, 700)], 2, 128, 16, "i8")
    q = s.q(8, dtype)
    q[..., 0] = 8.0
    for at, key in ((600, 40.0), (603, -40.0)) if where == "seen" else ((699, -40.0),):
        p, r = int(s.table[0, at // 16]), at % 16
        s.pool[0][p, :, r] = 0
        s.pool[0][p, :, r, 0] = 127 if key > 0 else -127
        s.scale[0][p, :, r] = abs(key) / 127
        if key < 0:
            s.scale[1][p, :, r] *= large
    check(engine, s, 8, dtype, q=q)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_a_strong_token_without_a_value(engine, dtype):
    """A first token with 2^30 times the weight of any other and a value of zero: the results are the
    others' (bound by their own sizes, as the zero adds nothing)."""
    s = Setup([(150, 700)], 2, 128, 16, "i8")
    p = int(s.table[0, 0])
    s.pool[0][p, :, 0] = 0
    s.pool[0][p, :, 0, 0] = 127
    s.scale[0][p, :, 0] = 30 * math.log(2.0) * 128 ** 0.5 / 8.0 / 127
    s.pool[1][p, :, 0], s.scale[1][p, :, 0] = 0, 0.0
    q = s.q(8, dtype) * 0.1
    q[..., 0] = 8.0
    out = torch.empty_like(q)
    # results near 2^-30 * 700: under f16's range, so the others' values are made as large
    pos = torch.arange(1, 700, device=DEV)
    pp, r = places(s, pos)
    s.scale[1][pp, :, r] *= 2.0 ** 24
    engine.attn_paged_dev(s.cache, s.batch, q, out)
    engine.sync()
    ref, _, amp = s.attention(q)
    assert ((out.double() - ref).abs() <= 2.0 ** -8 * (amp + ref.abs())).all()


def strong_token(engine, dtype, new, tokens, bits):
    """The first token has 2^bits times the weight of any other and a small value, so that results are made
    of the others' weights.  In the 2-norm: f32 as everywhere; 16-bit results have their own rounding and that of
    weights to 11 bits, each 2^-12 (bf16: 2^-9 and 2^-12) at most and of random sign."""
    s = Setup([(new, tokens)], 1, 128, 64, "f16")
    pos = torch.arange(tokens, device=DEV)
    p, r = places(s, pos)
    s.pool[0][p, :, r] *= 0.1
    s.pool[0][p, :, r, 0] = 0
    s.pool[0][p[0], :, r[0]] = 0
    s.pool[0][p[0], :, r[0], 0] = bits * math.log(2.0) * 128 ** 0.5 / 4.0
    s.pool[1][p[0], :, r[0]] = 1e-3
    q = s.q(4, dtype)
    q[..., 0] = 4.0
    out = torch.empty_like(q)
    lse = torch.empty(q.shape[:2], device=DEV)
    engine.attn_paged_dev(s.cache, s.batch, q, out, lse=lse)
    engine.sync()
    ref, ref_lse, _ = s.attention(q)
    rel = ((out.double() - ref).norm() / ref.norm()).item()
    assert rel <= {"f32": 1e-5, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype], rel
    assert ((lse.double() - ref_lse).abs() <= 2.0 ** -12 + ref_lse.abs() * 2.0 ** -20).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tokens,bits", [(1000, 10), (8000, 14), (131071, 18)])
def test_one_strong_token(engine, dtype, tokens, bits):
    strong_token(engine, dtype, 1, tokens, bits)


@pytest.mark.parametrize("tokens,bits", [(1000, 10), (8000, 14), (20000, 18)])
def test_one_strong_token_before_f32_rows(engine, tokens, bits):
    strong_token(engine, "f32", 64, tokens, bits)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_one_strong_token_in_many_sequences(engine, dtype):
    """The same for single tokens, where each warp streams a thousand positions: 600 sequences of the same 3000
    positions, the first with 2^18 times the weight of any other and no value."""
    s = Setup([(600, 3000)], 1, 128, 64, "f16")
    pos = torch.arange(3000, device=DEV)
    p, r = places(s, pos)
    s.pool[0][p, :, r] *= 0.1
    s.pool[0][p, :, r, 0] = 0
    s.pool[0][p[0], :, r[0]] = 0
    s.pool[0][p[0], :, r[0], 0] = 18 * math.log(2.0) * 128 ** 0.5 / 4.0
    s.pool[1][p[0], :, r[0]] = 0
    q = s.q(4, dtype)
    q[..., 0] = 4.0
    batch = hb.KvBatch(s.table.repeat(600, 1), torch.arange(601, dtype=torch.int32, device=DEV),
                       torch.full((600,), 3000, dtype=torch.int32, device=DEV), 600, 1)
    out = torch.empty_like(q)
    engine.attn_paged_dev(s.cache, batch, q, out)
    engine.sync()
    ref, _, _ = s.attention(q, causal=False)
    rel = ((out.double() - ref).norm() / ref.norm()).item()
    assert rel <= {"f32": 1e-5, "f16": 2.0 ** -11}[dtype], rel


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("tokens,bits", [(1000, 10), (8000, 14), (131071, 18)])
def test_one_strong_token_before_a_chunk(engine, dtype, tokens, bits):
    strong_token(engine, dtype, 64, tokens, bits)


@pytest.mark.parametrize("cache,dtype", [("f16", "f32"), ("i8", "f32"), ("f16", "bf16"), ("i8", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("new", [1, 150])
def test_queries_of_uneven_size(engine, cache, dtype, new):
    """One element of every query is 2^20 (f16: 2^14) times the others and meets keys of zero: the scores are
    made of the others, which keep their bits (f32: 2^-19 of them)."""
    s = Setup([(new, 400)], 2, 128, 16, cache)
    s.pool[0][..., 5] = 0
    q = s.q(8, dtype)
    q[..., 5] = 2.0 ** (14 if dtype == "f16" else 20)
    check(engine, s, 8, dtype, q=q)


@pytest.mark.parametrize("window", [1 << 30, (1 << 31) - 1, 1 << 31, (1 << 32) + 5])
@pytest.mark.parametrize("cache,dtype", [("i8", "f32"), ("f16", "f16"), ("i8", "bf16")])
def test_windows_longer_than_any_sequence(engine, window, cache, dtype):
    """Also with tokens before the first position, from whose place such a window starts far below zero."""
    check(engine, Setup([(6, 2), (140, 10), (3, 0), (1, 5), (40, 300)], 2, 64, 16, cache), 4, dtype, window=window)


@pytest.mark.parametrize("page", [-1, -(1 << 31), 5000])
@pytest.mark.parametrize("cache,dtype", [("i8", "f32"), ("i8", "f16"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("new", [1, 150])
def test_pages_out_of_range_are_reported(engine, page, cache, dtype, new):
    """Every number outside the pool, -1 (a page that is not mapped) among them, where a token sees it; and
    none where no token does."""
    s = Setup([(new, 200), (new, 250)], 2, 64, 16, cache)
    q = s.q(4, dtype)
    out = torch.empty_like(q)
    s.table[0, 13:] = page  # past the first sequence's 200 tokens
    engine.attn_paged_dev(s.cache, s.batch, q, out)
    engine.sync()
    s.table[0, 5] = page
    with pytest.raises(hb.CudaError) as e:
        engine.attn_paged_dev(s.cache, s.batch, q, out)
        engine.sync()
    assert e.value.code == _lib.HC_ERR_INVALID
    engine.sync()


@pytest.mark.parametrize("what,at,value", [("table", 0, -1), ("table", 0, 1 << 20), ("kv_len", 1, -5), ("kv_len", 0, 100000),
                                           ("q_start", 0, -3), ("q_start", 1, 0x7fffffff), ("q_start", 2, 1 << 20), ("q_start", 1, -1)])
@pytest.mark.parametrize("call", ["append", "read", "attend"])
@pytest.mark.parametrize("cache", ["i8", "f16"])
def test_every_call_reports_values_out_of_range(engine, call, what, at, value, cache):
    s = Setup([(40, 200), (40, 250)], 2, 64, 16, cache)
    getattr(s, what).view(-1)[at] = value
    if what == "table":
        s.table[:] = value
    x, q = s.q(2, "f16"), s.q(4, "f16")
    with pytest.raises(hb.CudaError) as e:
        if call == "attend":
            engine.attn_paged_dev(s.cache, s.batch, q, torch.empty_like(q))
        else:
            (engine.kv_append_dev if call == "append" else engine.kv_read_dev)(s.cache, s.batch, x, x.clone())
        engine.sync()
    assert e.value.code == _lib.HC_ERR_INVALID
    engine.sync()  # reported once


@pytest.mark.parametrize("call", ["append", "read"])
def test_sequences_that_fit_are_not_reported(engine, call):
    """Tokens before the first position, sequences without tokens or new ones, rows of no sequence."""
    s = Setup([(6, 2), (0, 0), (3, 0), (0, 9), (1, 5)], 2, 64, 16, "f16")
    batch = hb.KvBatch(s.table, s.q_start + 1, s.kv_len, s.rows + 4, 6)
    x = torch.randn(s.rows + 4, 2, 64, device=DEV).half()
    (engine.kv_append_dev if call == "append" else engine.kv_read_dev)(s.cache, batch, x, x.clone())
    engine.sync()


def split_work(seed):
    """A batch whose sequences are split over blocks, its queries, and their results alone."""
    s = Setup([(1, 9000 + 37 * seed), (1, 3), (90, 5000 + 11 * seed)], 2, 128, 16, "i8", seed=seed)
    return s, s.q(8, "f16")


def test_two_streams_at_once(engine):
    """Calls on two streams are in flight together, and a graph captured on one of them beside both: each has
    partial results of its own, so that all get the bits that they get alone."""
    work = [split_work(i) for i in (1, 2, 3)]
    alone = []
    for s, q in work:
        alone.append(torch.empty_like(q))
        engine.attn_paged_dev(s.cache, s.batch, q, alone[-1])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = [[torch.zeros_like(q) for _ in range(20)] for _, q in work]
    g = torch.cuda.CUDAGraph()
    engine.set_stream(streams[0])
    with torch.cuda.graph(g, stream=streams[0]):  # the stream's first call, in a capture
        for o in outs[2]:
            engine.attn_paged_dev(work[2][0].cache, work[2][0].batch, work[2][1], o)
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(streams[2]):
            g.replay()
        for i in range(20):
            for k in range(2):
                engine.set_stream(streams[k])
                engine.attn_paged_dev(work[k][0].cache, work[k][0].batch, work[k][1], outs[k][i])
        torch.cuda.synchronize()
        for k in range(3):
            for o in outs[k]:
                assert torch.equal(o, alone[k]), k
                o.zero_()
    engine.sync()


# ------------------------------------------------------------------ sizes of prompts
@pytest.mark.parametrize("cache", ["i8", "f16", "bf16"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,kv_heads,page", [(128, 8, 64), (64, 5, 24), (128, 3, 100)])
def test_append_then_read_prompts(engine, cache, dtype, dim, kv_heads, page):
    """More rows than threads at once: several rows to a thread, and heads that they do not divide."""
    s = Setup([(6000, 6100), (1, 7), (4003, 4003)], kv_heads, dim, page, cache)
    x = [s.q(kv_heads, dtype) for _ in range(2)]
    engine.kv_append_dev(s.cache, s.batch, *x)
    back = [torch.full_like(t, math.nan) for t in x]
    engine.kv_read_dev(s.cache, s.batch, *back)
    engine.sync()
    for w in range(2):
        v = x[w].float()
        if cache == "i8":
            codes, scale = quantised(v)
            v = codes.float() * scale[..., None]
        assert torch.equal(back[w], v.to(T[cache]).float().to(T[dtype]) if cache != "i8" else v.to(T[dtype]))


@pytest.mark.parametrize("cache,dtype", [("i8", "f32"), ("bf16", "f32"), ("f16", "f32"), ("bf16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("dim", [64, 128])
def test_prompts_of_thousands(engine, cache, dtype, dim):
    check(engine, Setup([(2500, 2500), (700, 3001), (1, 40)], 1, dim, 64, cache), 4, dtype)


@pytest.mark.parametrize("cache,dtype", [("i8", "f16"), ("f16", "f16"), ("bf16", "bf16")])
def test_a_tile_in_more_than_64_pieces(engine, cache, dtype):
    """One long sequence beside short ones: nearly all blocks have a piece of its one tile."""
    s = Setup([(40, 300000)] + [(40, 60 + i) for i in range(9)], 1, 64, 64, cache)
    q = s.q(4, dtype)
    a, b = check(engine, s, 4, dtype, q=q), check(engine, s, 4, dtype, q=q)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_lse_where_values_are_not_finite(engine, dtype, bad):
    """V scales that are not finite, over a whole unit: the results that see them are not finite, the scores'
    log-sum-exp is as without them."""
    s = Setup([(150, 700), (1, 300)], 2, 128, 16, "i8")
    for i in range(2):
        p, r = places(s, torch.arange(130, device=DEV), i)
        s.scale[1][p, :, r] = bad
    q = s.q(8, dtype)
    out, lse = torch.zeros_like(q), torch.zeros(q.shape[:2], device=DEV)
    engine.attn_paged_dev(s.cache, s.batch, q, out, lse=lse)
    engine.sync()
    _, ref_lse, _ = s.attention(q)
    assert not torch.isfinite(out).any()
    assert ((lse.double() - ref_lse).abs() <= 2.0 ** -12 + ref_lse.abs() * 2.0 ** -20).all()
