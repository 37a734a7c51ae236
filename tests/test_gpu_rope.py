"""GPU tests of rotary positions (rope_dev, kv_append_rope_dev) against their definition in long doubles.

Tolerances: an angle is off by at most 2^-33 of a turn from the fixed point, and 2^-25 of half a turn from the
argument's rounding to f32, in all below 2^-23 rad; cos and sin by two units of f32 (2^-23); the amplitude, two
products and a sum round four times (2^-24 each): |err| <= (|a| + |b|) amplitude 2^-21 holds, and the result's
rounding to its type adds half a step of it.  An 8-bit cache adds half a code."""
import math

import numpy as np
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


def turned(rope, x, pos):
    """(rows turned, |a| + |b| of every value's pair) in long doubles; the frequencies are the rope's own."""
    half, dim = rope.rot_dim // 2, rope.head_dim
    v = x.double().cpu().numpy().astype(np.longdouble)
    f = np.array(rope.struct.turns[:half], dtype=np.uint64).astype(np.longdouble) / np.longdouble(2) ** 64
    t = pos.cpu().numpy().astype(np.longdouble)[:, None] * f
    angle = (t - np.floor(t)) * (8 * np.arctan(np.longdouble(1)))
    amp = np.longdouble(rope.struct.amplitude)
    c, s = (np.cos(angle) * amp)[:, None], (np.sin(angle) * amp)[:, None]
    ia, ib = (np.arange(half), np.arange(half) + half) if rope.struct.layout == 0 else (2 * np.arange(half), 2 * np.arange(half) + 1)
    y, size = v.copy(), np.zeros_like(v)
    y[..., ia], y[..., ib] = v[..., ia] * c - v[..., ib] * s, v[..., ia] * s + v[..., ib] * c
    size[..., ia] = size[..., ib] = (np.abs(v[..., ia]) + np.abs(v[..., ib])) * np.abs(amp)
    return y, size


def near(got, want, size, dtype, extra=0.0):
    off = np.abs(got.double().cpu().numpy().astype(np.longdouble) - want)
    least = 2.0 ** -25 if dtype == "f16" else 0.0  # half the smallest step
    bound = size * 2.0 ** -21 + (np.abs(want) + size * 2.0 ** -21) * (torch.finfo(T[dtype]).eps / 2) + least + extra
    assert (off <= bound).all(), float((off - bound).max())


POS = [0, 1, -1, 2, 4095, 131072, 1000003, 2**30, 2**31 - 1, -2**31, 77, -12345]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,rot,layout,heads", [(128, 0, "half", 5), (128, 0, "pairs", 3), (64, 32, "half", 1), (64, 24, "pairs", 8),
                                                  (256, 256, "half", 2), (96, 48, "half", 4), (80, 20, "half", 3), (128, 10, "pairs", 9),
                                                  (6, 4, "half", 2), (2, 2, "pairs", 1), (128, 112, "half", 33)])
def test_rows(engine, dtype, dim, rot, layout, heads):
    g = torch.Generator(device=DEV).manual_seed(dim + rot)
    rope = hb.Rope(dim, rot, base=500000.0, layout=layout, factor=8.0, original=8192, low=1.0, high=4.0, amplitude=1.25)
    pos = torch.tensor(POS, dtype=torch.int32, device=DEV)
    x = torch.randn(len(POS), heads, dim, generator=g, device=DEV).to(T[dtype])
    out = torch.full_like(x, math.nan)
    engine.rope_dev(rope, pos, x, out)
    engine.sync()
    want, size = turned(rope, x, pos)
    near(out, want, size, dtype)
    rest = x[..., rope.rot_dim:]
    assert torch.equal(out[..., rope.rot_dim:], rest)
    assert torch.equal(out[0, :, :rope.rot_dim].double(), (x[0, :, :rope.rot_dim].float() * 1.25).to(T[dtype]).double())  # position 0
    again = x.clone()
    engine.rope_dev(rope, pos, again)  # in place
    engine.sync()
    assert torch.equal(again, out)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,heads", [(1, 1), (1, 40), (3, 7), (700, 1), (2500, 32)])
def test_sizes(engine, dtype, n, heads):
    g = torch.Generator(device=DEV).manual_seed(n)
    rope = hb.Rope(128)
    pos = torch.randint(0, 1 << 20, (n,), generator=g, device=DEV, dtype=torch.int32)
    x = torch.randn(n, heads, 128, generator=g, device=DEV).to(T[dtype])
    out = torch.full_like(x, math.nan)
    engine.rope_dev(rope, pos, x, out)
    engine.sync()
    near(out, *turned(rope, x, pos), dtype)


@pytest.mark.parametrize("off,pad", [(0, 0), (8, 0), (1, 3), (4, 8)])
def test_slices_of_a_projection_in_place(engine, off, pad):
    """Queries and keys turned where a projection left them, at any alignment; what lies around them stays."""
    g = torch.Generator(device=DEV).manual_seed(off)
    rope = hb.Rope(64, layout="pairs")
    n, heads = 33, 5
    buf = torch.randn(n, off + heads * 64 + pad + 64, generator=g, device=DEV).half()
    before = buf.clone()
    x = buf[:, off:off + heads * 64].unflatten(1, (heads, 64))
    pos = torch.arange(n, dtype=torch.int32, device=DEV) * 1000
    engine.rope_dev(rope, pos, x)
    engine.sync()
    near(x, *turned(rope, before[:, off:off + heads * 64].unflatten(1, (heads, 64)), pos), "f16")
    buf[:, off:off + heads * 64] = before[:, off:off + heads * 64]
    assert torch.equal(buf, before)


def test_turning_back(engine):
    """A negative position undoes a positive one: two turns' bounds."""
    g = torch.Generator(device=DEV).manual_seed(5)
    rope = hb.Rope(128, 64)
    pos = torch.randint(0, 1 << 30, (50,), generator=g, device=DEV, dtype=torch.int32)
    x = torch.randn(50, 4, 128, generator=g, device=DEV)
    y = x.clone()
    engine.rope_dev(rope, pos, y)
    engine.rope_dev(rope, -pos, y)
    engine.sync()
    a, b = x[..., :32].abs(), x[..., 32:64].abs()
    assert ((y - x)[..., :64].abs() <= 2.0 ** -21 * 3 * torch.cat([a + b, a + b], -1)).all()
    assert torch.equal(y[..., 64:], x[..., 64:])


def test_values_that_are_not_finite_stay_in_their_pair(engine):
    rope = hb.Rope(64)
    x = torch.ones(1, 2, 64, device=DEV)
    x[0, 1, 3] = math.inf
    x[0, 1, 40] = math.nan
    out = torch.empty_like(x)
    engine.rope_dev(rope, torch.tensor([5], dtype=torch.int32, device=DEV), x, out)
    engine.sync()
    bad = ~out.isfinite()
    assert bad[0, 1].nonzero().flatten().tolist() == [3, 8, 35, 40] and not bad[0, 0].any()


def test_rope_refusals(engine):
    rope = hb.Rope(64)
    pos = torch.zeros(4, dtype=torch.int32, device=DEV)
    x = torch.zeros(4, 2, 64, device=DEV)
    for bad, what in ((lambda: engine.rope_dev(rope, pos[:3], x), "n_tok"), (lambda: engine.rope_dev(rope, pos, x.double()), "float32"),
                      (lambda: engine.rope_dev(rope, pos, x[..., :32]), "head_dim"), (lambda: engine.rope_dev(rope, pos, x, x.half()), "type"),
                      (lambda: engine.rope_dev(rope, pos, x.transpose(0, 1).contiguous().transpose(0, 1)), "contiguous"),
                      (lambda: engine.rope_dev(rope, pos.long(), x), "int32"), (lambda: engine.rope_dev(rope, pos[::2], x[:2]), "contiguous"),
                      (lambda: engine.rope_dev(rope, pos, x.cpu()), "device")):
        with pytest.raises(ValueError, match=what):
            bad()
    buf = torch.zeros(5, 128, device=DEV)
    with pytest.raises(hb.CudaError, match="overlap"):
        engine.rope_dev(rope, pos, buf[:4].view(4, 2, 64), buf[1:].view(4, 2, 64))
    wide = torch.zeros(4, 256, device=DEV)  # halves of one array's rows: apart
    engine.rope_dev(rope, pos, wide[:, :128].unflatten(1, (2, 64)), wide[:, 128:].unflatten(1, (2, 64)))
    with pytest.raises(hb.CudaError, match="overlap"):
        engine.rope_dev(rope, pos, wide[:, :128].unflatten(1, (2, 64)), wide[:, 64:192].unflatten(1, (2, 64)))
    engine.rope_dev(rope, pos[:0], x[:0])
    engine.sync()


# ------------------------------------------------------------------ together with the cache
class Step:
    """A batch's pages (shuffled, one pool) and its rows."""

    def __init__(self, lens, heads, kv_heads, dim, page, cache, dtype, seed=1, pad=0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.new, self.kv, self.cache_type, self.dtype = [a for a, _ in lens], [b for _, b in lens], cache, dtype
        need = [-(-max(k, 0) // page) for k in self.kv]
        n_pages = sum(need) + 2
        perm = torch.randperm(n_pages, generator=g, device=DEV, dtype=torch.int32)
        self.table = torch.full((len(lens), max(need + [1])), -7, dtype=torch.int32, device=DEV)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = perm[at:at + n]
            at += n
        self.shape = (n_pages, kv_heads, page, dim)
        self.q_start = torch.tensor([0] + self.new, device=DEV).cumsum(0).to(torch.int32)
        self.kv_len = torch.tensor(self.kv, dtype=torch.int32, device=DEV)
        self.rows = sum(self.new)
        self.batch = hb.KvBatch(self.table, self.q_start, self.kv_len, self.rows, max(self.new))
        width = (heads + 2 * kv_heads) * dim + pad
        self.buf = torch.randn(self.rows, width, generator=g, device=DEV).to(T[dtype])
        part = self.buf[:, :width - pad].unflatten(1, (heads + 2 * kv_heads, dim))
        self.q, self.k, self.v = part[:, :heads], part[:, heads:heads + kv_heads], part[:, heads + kv_heads:]
        self.pos = torch.cat([torch.arange(k - n, k, device=DEV) for n, k in zip(self.new, self.kv)]).to(torch.int32)

    def pools(self):
        fill = lambda: torch.full(self.shape, 5, dtype=T[self.cache_type], device=DEV)  # noqa: E731
        scale = lambda: torch.full(self.shape[:3], 3.0, device=DEV) if self.cache_type == "i8" else None  # noqa: E731
        return [fill(), fill(), scale(), scale()]


LENS = [(1, 1), (3, 3), (0, 0), (1, 40), (17, 100), (0, 9), (5, 5), (1, 1000000)]
SHORT = LENS[:-1]


@pytest.mark.parametrize("cache", ["i8", "f16", "bf16"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,rot,layout,heads,kv_heads,page", [(64, 32, "half", 9, 3, 16), (128, 128, "pairs", 8, 8, 24), (128, 96, "half", 4, 1, 1),
                                                                (64, 24, "pairs", 1, 1, 100), (128, 128, "half", 32, 8, 64)])
def test_append(engine, cache, dtype, dim, rot, layout, heads, kv_heads, page):
    s = Step(SHORT, heads, kv_heads, dim, page, cache, dtype, pad=16)
    rope = hb.Rope(dim, rot, layout=layout, base=1000.0, factor=2.0, amplitude=0.75)
    pools, plain = s.pools(), s.pools()
    q_out = torch.full((s.rows, heads, dim), math.nan, device=DEV).to(T[dtype])
    engine.kv_append_rope_dev(hb.KvCache(*pools), s.batch, rope, s.q, s.k, s.v, q_out)
    # queries as rope_dev turns them, values as kv_append_dev stores them, bit for bit; f32 keys as both in turn
    want = torch.empty_like(q_out)
    engine.rope_dev(rope, s.pos, s.q, want)
    keys = s.k.clone()
    engine.rope_dev(rope, s.pos, keys)
    engine.kv_append_dev(hb.KvCache(*plain), s.batch, keys, s.v)
    back = [torch.empty_like(s.k.contiguous()).float() for _ in range(2)]
    engine.kv_read_dev(hb.KvCache(*pools), s.batch, *back)
    engine.sync()
    assert torch.equal(q_out, want)
    near(q_out, *turned(rope, s.q, s.pos), dtype)
    for i in (1, 3):
        assert pools[i] is None or torch.equal(pools[i], plain[i])
    if dtype == "f32":
        assert all(a is None or torch.equal(a, b) for a, b in zip(pools, plain))
    exact, size = turned(rope, s.k, s.pos)
    if cache == "i8":
        step = np.abs(exact).max(-1, keepdims=True) / 127
        near(back[0], exact, size, "f32", extra=step * (0.5 + 2.0 ** -14))
    else:
        near(back[0], exact, size, cache)


def test_in_place_far_positions_and_many_tokens(engine):
    """A long step beside a token at position 999999, in place in a projection's rows."""
    s = Step([(1, 1000000), (5000, 5001), (1, 7)], 8, 2, 64, 128, "bf16", "bf16", pad=8)
    rope = hb.Rope(64, base=500000.0)
    pools = s.pools()
    before = s.buf.clone()
    want = torch.empty(s.rows, 8, 64, dtype=torch.bfloat16, device=DEV)
    engine.rope_dev(rope, s.pos, s.q, want)
    engine.kv_append_rope_dev(hb.KvCache(*pools), s.batch, rope, s.q, s.k, s.v)
    engine.sync()
    assert torch.equal(s.q, want) and torch.equal(s.buf[:, 512:], before[:, 512:])
    k = torch.empty(s.rows, 2, 64, dtype=torch.float32, device=DEV)
    engine.kv_read_dev(hb.KvCache(*pools), s.batch, k, torch.empty_like(k))
    engine.sync()
    near(k, *turned(rope, s.k, s.pos), "bf16")


def test_rows_of_no_sequence_and_before_the_first_position(engine):
    """They are left alone, queries and pages, and so are pages that no token has."""
    s = Step([(2, 2), (3, 9)], 4, 2, 64, 16, "f16", "f32")
    s.q_start += 2  # rows 0 and 1 are nobody's, and the last two fall off the end
    q_start = torch.tensor([2, 4, 5], dtype=torch.int32, device=DEV)
    kv_len = torch.tensor([1, 9], dtype=torch.int32, device=DEV)  # the first one's first new token lies before position 0
    batch = hb.KvBatch(s.table, q_start, kv_len, 5)
    pools = s.pools()
    out = torch.full((5, 4, 64), 9.0, device=DEV)
    engine.kv_append_rope_dev(hb.KvCache(*pools), batch, hb.Rope(64), s.q, s.k, s.v, out)
    engine.sync()
    assert (out[:3] == 9).all() and not (out[3:] == 9).any()
    rows = (pools[0] != 5).any(-1).any(1).sum().item()
    assert rows == 2


def test_keys_that_are_not_finite_read_back_as_nan(engine):
    s = Step([(3, 3)], 1, 1, 64, 16, "i8", "f32")
    s.k[1, 0, 5] = math.inf
    pools = s.pools()
    engine.kv_append_rope_dev(hb.KvCache(*pools), s.batch, hb.Rope(64), s.q, s.k, s.v, torch.empty_like(s.q))
    back = [torch.empty(3, 1, 64, device=DEV) for _ in range(2)]
    engine.kv_read_dev(hb.KvCache(*pools), s.batch, *back)
    engine.sync()
    assert back[0][1].isnan().all() and back[0][0].isfinite().all() and back[0][2].isfinite().all()


def test_a_captured_step_follows_its_lengths(engine):
    s = Step([(1, 5), (1, 20)], 4, 2, 64, 16, "bf16", "f32")
    rope = hb.Rope(64)
    pools, out = s.pools(), torch.empty(2, 4, 64, device=DEV)
    cache = hb.KvCache(*pools)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        engine.set_stream(torch.cuda.current_stream())
        engine.kv_append_rope_dev(cache, s.batch, rope, s.q, s.k, s.v, out)
    engine.set_stream(torch.cuda.current_stream())
    for step in range(3):
        graph.replay()
        near(out, *turned(rope, s.q, s.kv_len - 1), "f32")
        s.kv_len += 1
    torch.cuda.synchronize()


def test_append_refusals(engine):
    s = Step([(1, 5), (1, 20)], 4, 2, 64, 16, "bf16", "f32")
    cache, rope = hb.KvCache(*s.pools()), hb.Rope(64)
    for kw, what in ((dict(rope=hb.Rope(128)), "head_dim"), (dict(q=s.q.half()), "one type"), (dict(q=s.q[:1]), "n_tok"),
                     (dict(k=s.q), "heads"), (dict(q_out=s.q.half()), "one type")):
        args = dict(rope=rope, q=s.q, k=s.k, v=s.v, q_out=None) | kw
        with pytest.raises((ValueError, hb.CudaError), match=what):
            engine.kv_append_rope_dev(cache, s.batch, *args.values())
    for odd in (hb.Rope(64, 24), hb.Rope(64, 12, layout="pairs")):
        with pytest.raises(hb.CudaError, match="rot_dim"):
            engine.kv_append_rope_dev(cache, s.batch, odd, s.q, s.k, s.v)
    with pytest.raises(hb.CudaError, match="overlap"):  # queries over the keys
        engine.kv_append_rope_dev(cache, s.batch, rope, s.q.clone(), s.k, s.v, s.buf[:, 128:384].unflatten(1, (4, 64)))
    empty = hb.KvBatch(s.table[:0], s.q_start[:1], s.kv_len[:0], 0)
    engine.kv_append_rope_dev(cache, empty, rope, s.q[:0], s.k[:0], s.v[:0])
    engine.sync()


def test_one_row_in_place_whatever_its_leading_dimensions(engine):
    """A single row has no next one: in place is the same address."""
    from hayai_b200 import _lib
    x = torch.randn(1, 2, 64, device=DEV)
    pos, rope = torch.tensor([7], dtype=torch.int32, device=DEV), hb.Rope(64)
    want = torch.empty_like(x)
    engine.rope_dev(rope, pos, x, want)
    assert _lib.lib().hc_rope_dev(engine.handle, rope.ref, 0, 1, 2, pos.data_ptr(), x.data_ptr(), 128, x.data_ptr(), 256) == _lib.HC_OK
    engine.sync()
    assert torch.equal(x, want)
    two = torch.randn(2, 2, 64, device=DEV)
    assert _lib.lib().hc_rope_dev(engine.handle, rope.ref, 0, 2, 2, pos.data_ptr(), two.data_ptr(), 128, two.data_ptr(),
                                  256) == _lib.HC_ERR_INVALID
    s = Step([(1, 5)], 4, 2, 64, 16, "bf16", "f32")
    q, q_want = s.q.clone(), torch.empty_like(s.q)
    cache = hb.KvCache(*s.pools())
    engine.kv_append_rope_dev(cache, s.batch, rope, s.q, s.k, s.v, q_want)
    assert _lib.lib().hc_kv_append_rope_dev(engine.handle, cache.ref, s.batch.ref, rope.ref, 0, 4, q.data_ptr(), 256, q.data_ptr(), 512,
                                            s.k.data_ptr(), 512, s.v.data_ptr(), 512) == _lib.HC_OK
    engine.sync()
    assert torch.equal(q, q_want)


@pytest.mark.parametrize("order", ["rows of all heads", "heads apart", "rows apart", "pages and heads apart"])
@pytest.mark.parametrize("cache,dtype", [("i8", "bf16"), ("i8", "f32"), ("bf16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 1)])
def test_append_to_pools_of_other_orders(engine, order, cache, dtype, dim, page):
    """Bit for bit the rows that a contiguous pool gets, and nothing between them."""
    s = Step(SHORT, 8, 2, dim, page, cache, dtype)
    rope = hb.Rope(dim, base=1000.0)
    plain = s.pools()
    out, want = torch.empty_like(s.q), torch.empty_like(s.q)
    engine.kv_append_rope_dev(hb.KvCache(*plain), s.batch, rope, s.q, s.k, s.v, want)
    n, h, r, d = s.shape
    whole, parts = [], []
    for x in plain[:2]:
        shape, perm, at = {"rows of all heads": ((n, r, h, d), (0, 2, 1, 3), ()), "heads apart": ((h, n, r, d), (1, 0, 2, 3), ()),
                           "rows apart": ((n, h, r, 2 * d), (0, 1, 2, 3), (slice(None),) * 3 + (slice(d),)),
                           "pages and heads apart": ((2 * n, h + 1, r, d), (0, 1, 2, 3), (slice(1, None, 2), slice(1, None)))}[order]
        whole.append(torch.full(shape, 5, dtype=x.dtype, device=DEV))
        parts.append(whole[-1].permute(perm)[at])
    for x in plain[2:]:
        if x is None:
            parts.append(None)
            continue
        whole.append(torch.full((n, h * r + 5), 3.0, device=DEV))
        parts.append(whole[-1][:, 2:-3].unflatten(1, (h, r)))
    engine.kv_append_rope_dev(hb.KvCache(*parts), s.batch, rope, s.q, s.k, s.v, out)
    engine.sync()
    assert torch.equal(out, want)
    assert all(a is None or torch.equal(a, b) for a, b in zip(parts, plain))
    for x, fill in zip(parts, (5, 5, 3, 3)):
        if x is not None:
            x.fill_(fill)
    assert all((w == f).all() for w, f in zip(whole, (5, 5, 3, 3)))
