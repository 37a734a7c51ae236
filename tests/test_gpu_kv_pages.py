"""GPU tests of the cache's bookkeeping (kv_fork_dev, kv_resize_dev, kv_compact_dev) against a model that does one
item after the other in Python.  Everything is whole numbers and copied bits: results are equal."""
import random

import pytest
import torch

import hayai_b200 as hb

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
T = {"f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}


@pytest.fixture(autouse=True)
def _stream(engine):
    engine.set_stream(torch.cuda.current_stream())
    yield
    engine.set_stream(None)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


class Pool:
    """Layers' pools of random bits, tables and holders on the GPU, and the same in Python lists."""

    def __init__(self, n_pages=40, slots=12, page=16, layers=2, heads=3, dim=64, cache="f16", order="phrd", max_pages=None, seed=0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.page, self.n_pages, self.slots = page, n_pages, slots
        self.max_pages = max_pages or n_pages
        raw = torch.int8 if cache == "i8" else torch.int16
        shape = (n_pages, heads, page, dim)
        self.bits = []  # every tensor of every layer, as integers
        caches = []
        for _ in range(layers):
            args = []
            for _ in range(2):
                x = torch.randint(-128 if cache == "i8" else -32768, 128 if cache == "i8" else 32768, shape, generator=g,
                                  device=DEV, dtype=torch.int32).to(raw)
                if order == "prhd":
                    x = x.transpose(1, 2).contiguous().transpose(1, 2)
                self.bits.append(x)
                args.append(x if cache == "i8" else x.view(T[cache]))
            for _ in range(2):
                if cache == "i8":
                    x = torch.randint(-2**31, 2**31, shape[:3], generator=g, device=DEV).to(torch.int32)
                    self.bits.append(x)
                    args.append(x.view(torch.float32))
            caches.append(hb.KvCache(*args))
        self.table = torch.full((slots, self.max_pages), -3, dtype=torch.int32, device=DEV)
        self.kv_len, self.refs = torch.zeros(slots, dtype=torch.int32, device=DEV), torch.zeros(n_pages, dtype=torch.int32, device=DEV)
        self.pages = hb.KvPages(caches, self.table, self.kv_len, self.refs)
        self.m_table, self.m_len, self.m_refs = self.table.tolist(), [0] * slots, [0] * n_pages
        self.m_bits = [b.clone() for b in self.bits]

    # ---- the model: items in order; free pages are those that were free before the call
    def copy(self, src, dst, rows):
        for t in self.m_bits:
            t[dst, :, :rows] = t[src, :, :rows]

    def resize(self, slots, lens):
        """Returns whether all was in order."""
        free = [p for p, r in enumerate(self.m_refs) if r <= 0]
        taken, ok, full, seen = 0, True, False, set()
        refs = list(self.m_refs)  # as they stand at the start
        old_bits = self.m_bits
        self.m_bits = [b.clone() for b in old_bits]
        for s, n in zip(slots, lens):
            if not (0 <= s < self.slots and 0 <= n <= self.max_pages * self.page) or s in seen:
                ok = False
                continue
            seen.add(s)
            old = self.m_len[s]
            keep = min(old, n)
            had, get = -(-old // self.page), -(-n // self.page)
            whole, rest = divmod(keep, self.page)
            part = rest > 0 and refs[self.m_table[s][whole]] > 1
            need = max(get - had, 0) + part
            taken += need
            if need and taken > len(free):
                ok = False
                continue
            at = taken - need
            if part:
                p = self.m_table[s][whole]
                for t, o in zip(self.m_bits, old_bits):
                    t[free[at], :, :rest] = o[p, :, :rest]
                self.m_table[s][whole] = free[at]
                self.m_refs[free[at]] = 1
                self.m_refs[p] -= 1
                at += 1
            for j in range(had, get):
                self.m_table[s][j] = free[at + j - had]
                self.m_refs[free[at + j - had]] = 1
            for j in range(get, had):
                self.m_refs[self.m_table[s][j]] -= 1
            self.m_len[s] = n
        return ok

    def fork(self, parents, children):
        free = [p for p, r in enumerate(self.m_refs) if r <= 0]
        taken, ok, seen, lens = 0, True, set(), list(self.m_len)
        for a, b in zip(parents, children):
            if not (0 <= a < self.slots and 0 <= b < self.slots) or b in seen:
                ok = False
                continue
            seen.add(b)
            if lens[b]:
                ok = False
                continue
            whole, rest = divmod(lens[a], self.page)
            taken += rest > 0
            if rest and taken > len(free):
                ok = False
                continue
            for j in range(whole):
                self.m_table[b][j] = self.m_table[a][j]
                self.m_refs[self.m_table[a][j]] += 1
            if rest:
                self.copy(self.m_table[a][whole], free[taken - 1], rest)
                self.m_table[b][whole] = free[taken - 1]
                self.m_refs[free[taken - 1]] = 1
            self.m_len[b] = lens[a]
        return ok

    def compact(self):
        used = sum(r > 0 for r in self.m_refs)
        to, holes = list(range(self.n_pages)), [p for p in range(used) if self.m_refs[p] <= 0]
        for src, dst in zip([p for p in range(used, self.n_pages) if self.m_refs[p] > 0], holes):
            self.copy(src, dst, self.page)
            to[src], self.m_refs[dst], self.m_refs[src] = dst, self.m_refs[src], 0
        for s in range(self.slots):
            for j in range(-(-self.m_len[s] // self.page)):
                self.m_table[s][j] = to[self.m_table[s][j]]
        return to

    def same(self):
        assert self.kv_len.tolist() == self.m_len
        assert self.refs.tolist() == self.m_refs
        assert self.table.tolist() == self.m_table
        assert all(torch.equal(a, b) for a, b in zip(self.bits, self.m_bits))

    def held(self):
        """The holders are the table entries in use."""
        n = [0] * self.n_pages
        for s in range(self.slots):
            for j in range(-(-self.m_len[s] // self.page)):
                n[self.m_table[s][j]] += 1
        assert n == self.m_refs

    def do(self, engine, call, *args, ok=None):
        """One call, on the GPU and in the model; what the model finds out of order is reported."""
        if call == "compact":
            moved = torch.full((self.n_pages,), -9, dtype=torch.int32, device=DEV)
            engine.kv_compact_dev(self.pages, moved)
            good = True
            assert self.compact() == moved.tolist()
        else:
            good = getattr(self, call)(*args)
            getattr(engine, f"kv_{call}_dev")(self.pages, *map(ints, args))
        if good:
            engine.sync()
        else:
            with pytest.raises(hb.CudaError):
                engine.sync()
        assert ok is None or good == ok
        self.same()
        self.held()


SHAPES = [dict(), dict(page=1, n_pages=300, slots=5, dim=128, heads=1), dict(page=24, cache="i8", order="prhd", heads=2),
          dict(page=100, cache="bf16", layers=1, dim=128, slots=30), dict(cache="i8", layers=3, page=64, dim=128, n_pages=25),
          dict(layers=70, n_pages=12, heads=1, page=16), dict(n_pages=9000, page=16, layers=1, heads=1, slots=40, max_pages=700)]


@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_a_few_steps(engine, shape):
    p = Pool(**SHAPES[shape])
    n = min(p.max_pages, p.n_pages // 4) * p.page
    p.do(engine, "resize", [0, 2, 1], [n // 2 + 1, 1, n // 3], ok=True)
    p.do(engine, "fork", [0, 0, 1], [3, 4, p.slots - 1] if p.slots > 5 else [3, 4, 2][:3], ok=p.slots > 5)
    p.do(engine, "resize", [3, 4, 0], [n // 2 + 1 + p.page, n // 4 + 1, 0], ok=True)  # grows, is cut inside a shared page, goes
    p.do(engine, "compact")
    p.do(engine, "resize", [0, 3], [p.page, 0])
    p.do(engine, "compact")
    p.do(engine, "resize", list(range(p.slots)), [0] * p.slots, ok=True)
    assert not any(p.m_refs)
    p.do(engine, "compact")


@pytest.mark.parametrize("seed", range(6))
def test_random_steps(engine, seed):
    """Forty calls in a row, of slots that are used or not, until and past a full pool; out of order ones among them."""
    r = random.Random(seed)
    p = Pool(n_pages=r.choice([13, 60, 200]), slots=r.choice([3, 10, 40]), page=r.choice([3, 16, 24]), layers=r.choice([1, 2]),
             heads=r.choice([1, 4]), cache=r.choice(["f16", "i8"]), max_pages=9, seed=seed)
    for _ in range(40):
        call = r.choice(["resize", "resize", "fork", "compact"])
        n = r.randint(1, p.slots)
        if call == "resize":
            slots = r.sample(range(p.slots), n)
            if r.random() < 0.1:
                slots[-1] = r.choice([-1, p.slots, slots[0], 2**31 - 1, -2**31])
            p.do(engine, call, slots, [r.choice([0, r.randint(0, 9 * p.page + (r.random() < 0.05)), min(9 * p.page, p.m_len[s % p.slots] + 1)])
                                       for s in slots])
        elif call == "fork":
            free = [s for s in range(p.slots) if not p.m_len[s]]
            if r.random() < 0.1:
                free = list(range(p.slots))
            if free:
                kids = r.sample(free, min(len(free), n))
                if r.random() < 0.1:
                    kids[-1] = r.choice([-1, p.slots, kids[0]])
                p.do(engine, call, [r.randrange(p.slots) for _ in kids], kids)
        else:
            p.do(engine, call)


def test_a_slice_of_a_wider_table(engine):
    """Page tables and pools that are views: what lies around them stays."""
    p = Pool(n_pages=30, slots=5, page=16, max_pages=6)
    wide = torch.full((5, 9), 77, dtype=torch.int32, device=DEV)
    wide[:, 2:8] = p.table
    p.table = wide[:, 2:8]
    p.pages = hb.KvPages(p.pages._keep[0], p.table, p.kv_len, p.refs)
    p.do(engine, "resize", [0, 4], [90, 33], ok=True)
    p.do(engine, "fork", [0, 4], [1, 2], ok=True)
    p.do(engine, "resize", [0], [0], ok=True)
    p.do(engine, "compact")
    assert (wide[:, :2] == 77).all() and (wide[:, 8] == 77).all()


def test_lengths_from_the_lengths_themselves(engine):
    """kv_len as the new lengths: nothing changes, but partly filled pages that are shared become the slots' own."""
    p = Pool(page=16)
    p.do(engine, "resize", [0, 1], [40, 7], ok=True)
    engine.kv_resize_dev(p.pages, ints(list(range(p.slots))), p.kv_len)
    engine.sync()
    assert p.resize(list(range(p.slots)), list(p.m_len))
    p.same()


def test_two_thousand_items(engine):
    """As many as a call takes: 2048 children of one parent, one new page each, and all of them let go."""
    p = Pool(n_pages=2200, slots=2049, page=16, layers=1, heads=1, max_pages=9)
    p.do(engine, "resize", [2048], [40], ok=True)
    p.do(engine, "fork", [2048] * 2048, list(range(2048))[::-1], ok=True)
    p.do(engine, "resize", list(range(2048)), [0] * 2048, ok=True)
    with pytest.raises(hb.CudaError, match="2049"):
        engine.kv_resize_dev(p.pages, ints([0] * 2049), ints([0] * 2049))


def test_a_full_pool(engine):
    """Items that no page is left for stay as they were, with those behind them that take pages; the report says so."""
    p = Pool(n_pages=5, slots=4, page=16)
    p.do(engine, "resize", [0, 1, 2, 3], [48, 49, 1, 0], ok=False)
    assert p.m_len == [48, 0, 0, 0]
    engine.kv_resize_dev(p.pages, ints([1, 0]), ints([49, 8]))  # 1 still finds no room, 0 gives pages back all the same
    with pytest.raises(hb.CudaError, match="free page"):
        engine.sync()
    p.resize([1, 0], [49, 8])
    p.same()
    p.do(engine, "resize", [1], [49], ok=True)
    p.do(engine, "fork", [0, 1], [2, 3], ok=False)
    p.do(engine, "resize", [1], [48], ok=True)
    p.do(engine, "fork", [1, 0], [3, 2], ok=True)


def test_both_of_two_are_cut_inside_a_shared_page(engine):
    """Each gets a copy of its own, and the page that they shared is free."""
    p = Pool(page=16)
    p.do(engine, "resize", [0], [32], ok=True)
    p.do(engine, "fork", [0], [1], ok=True)
    p.do(engine, "resize", [0, 1], [20, 25], ok=True)
    assert p.m_refs.count(1) == 2 and p.m_refs.count(2) == 1


def test_a_captured_step(engine):
    """Fork, grow and let go inside a graph, replayed: the children are the same pages every time."""
    p = Pool(n_pages=60, slots=8, page=16)
    p.do(engine, "resize", [0, 1], [37, 100], ok=True)
    kids, parents, then, none = ints([2, 3, 4, 5]), ints([0, 0, 1, 1]), ints([38, 60, 112, 113]), ints([0] * 4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        engine.set_stream(torch.cuda.current_stream())
        engine.kv_resize_dev(p.pages, kids, none)
        engine.kv_fork_dev(p.pages, parents, kids)
        engine.kv_resize_dev(p.pages, kids, then)
        engine.kv_compact_dev(p.pages)
    engine.set_stream(torch.cuda.current_stream())
    for _ in range(3):
        graph.replay()
        engine.sync()
        p.resize(kids.tolist(), [0] * 4)
        p.fork(parents.tolist(), kids.tolist())
        p.resize(kids.tolist(), then.tolist())
        p.compact()
        p.same()


@pytest.mark.parametrize("what", ["page", "negative", "length", "long", "nobody"])
def test_bad_bookkeeping_is_reported(engine, what):
    """Page numbers and lengths out of range touch nothing outside, and counts do not fall below zero."""
    p = Pool(page=16, max_pages=5)
    p.do(engine, "resize", [0, 1], [40, 50], ok=True)
    if what in ("page", "negative"):
        p.table[0, 1] = 40 if what == "page" else -1
    elif what == "nobody":
        p.refs[int(p.table[0, 1])] = 0
    else:
        p.kv_len[0] = -5 if what == "length" else 81
    for call in (lambda: engine.kv_fork_dev(p.pages, ints([0]), ints([5])), lambda: engine.kv_compact_dev(p.pages),
                 lambda: engine.kv_resize_dev(p.pages, ints([0]), ints([0]))):
        if what == "nobody" and call.__code__.co_names[0:1] != ("kv_resize_dev",) and "kv_resize_dev" not in call.__code__.co_names:
            continue
        call()
        with pytest.raises(hb.CudaError):
            engine.sync()
    assert (p.refs >= 0).all()


def test_pages_refusals(engine):
    p = Pool()
    other = Pool(page=24)
    caches = [c for c in p.pages._keep[0]]
    with pytest.raises(ValueError, match="refs"):
        hb.KvPages(caches, p.table, p.kv_len, p.refs[:-1])
    with pytest.raises(ValueError, match="int32"):
        hb.KvPages(caches, p.table.long(), p.kv_len, p.refs)
    mixed = hb.KvPages([caches[0], other.pages._keep[0][0]], p.table, p.kv_len, p.refs)
    with pytest.raises(hb.CudaError, match="shape"):
        engine.kv_compact_dev(mixed)
    many = hb.KvPages(caches * 200, p.table, p.kv_len, p.refs)
    with pytest.raises(hb.CudaError, match="256"):
        engine.kv_compact_dev(many)
    for a, b in ((ints([0]), ints([0, 1])), (ints([0]).long(), ints([0])), (ints([0, 1, 2])[::2], ints([0, 1]))):
        with pytest.raises(ValueError, match="int32"):
            engine.kv_fork_dev(p.pages, a, b)
    with pytest.raises(ValueError, match="moved"):
        engine.kv_compact_dev(p.pages, torch.zeros(3, dtype=torch.int32, device=DEV))
    engine.kv_resize_dev(p.pages, ints([]), ints([]))
    engine.kv_fork_dev(p.pages, ints([]), ints([]))
    empty = hb.KvPages(caches, p.table[:0], p.kv_len[:0], p.refs)
    engine.kv_compact_dev(empty)
    engine.sync()
    p.same()


def test_pools_past_32_bits(engine):
    """Pages behind the first 4 GB of a pool are copied as the others."""
    n, page = 2100, 128  # 2 MB a page
    big = torch.zeros(n, 64, page, 128, dtype=torch.float16, device=DEV)
    big[n - 1] = torch.randn(64, page, 128, device=DEV).half()
    big[n - 2, :, :5] = 2.0
    small = big  # keys and values in one pool will do
    table, kv_len, refs = ints([[n - 1, n - 2, 0], [0, 0, 0]]), ints([page + 5, 0]), ints([0] * (n - 2) + [1, 1])
    pages = hb.KvPages([hb.KvCache(big, small)], table, kv_len, refs)
    engine.kv_fork_dev(pages, ints([0]), ints([1]))
    engine.sync()
    assert table[1].tolist() == [n - 1, 0, 0] and (big[0, :, :5] == 2).all() and not big[0, :, 5:].any()
    engine.kv_compact_dev(pages)
    engine.sync()
    assert table[:, :2].tolist() == [[2, 1], [2, 0]] and torch.equal(big[2], big[n - 1]) and (big[1, :, :5] == 2).all()


@pytest.mark.parametrize("page", [-1, 40, 2**31 - 1, -2**31])
@pytest.mark.parametrize("grow", [0, 1, 30])
def test_a_partly_filled_page_out_of_range(engine, page, grow):
    """Items that would keep it are left out, whatever an earlier use left in the child's table; others are done."""
    p = Pool(page=16, max_pages=5)
    p.do(engine, "resize", [0, 1, 5], [40, 50, 48], ok=True)
    p.do(engine, "resize", [5], [0], ok=True)
    p.do(engine, "resize", [2], [48], ok=True)  # slot 5's table still names pages that slot 2 has now
    assert p.m_table[5][2] in p.m_table[2][:3]
    mine = p.m_table[0][2]
    p.table[0, 2] = p.m_table[0][2] = page
    engine.kv_fork_dev(p.pages, ints([0, 1]), ints([5, 6]))
    with pytest.raises(hb.CudaError, match="out of range"):
        engine.sync()
    p.fork([1], [6])
    p.same()
    engine.kv_resize_dev(p.pages, ints([0, 1]), ints([40 + grow, 33]))  # keeps its bad page
    with pytest.raises(hb.CudaError, match="out of range"):
        engine.sync()
    p.resize([1], [33])
    p.same()
    p.table[0, 2] = p.m_table[0][2] = mine
    p.do(engine, "resize", [0, 1, 2, 6], [0] * 4, ok=True)


@pytest.mark.parametrize("page", [-1, 40])
def test_a_whole_page_out_of_range_goes_to_the_child(engine, page):
    """Reported, counted for nobody, and named by nobody else than parent and child."""
    p = Pool(page=16, max_pages=5)
    p.do(engine, "resize", [0], [40], ok=True)
    lost = p.m_table[0][1]
    p.table[0, 1] = page
    engine.kv_fork_dev(p.pages, ints([0]), ints([5]))
    with pytest.raises(hb.CudaError, match="out of range"):
        engine.sync()
    assert p.kv_len.tolist()[5] == 40 and p.table[5, :2].tolist() == [p.m_table[0][0], page]
    assert p.refs[p.m_table[0][0]] == 2 and p.refs[lost] == 1
    engine.kv_resize_dev(p.pages, ints([0, 5]), ints([0, 0]))
    with pytest.raises(hb.CudaError, match="out of range"):
        engine.sync()
    assert p.refs.sum() == 1 and p.refs[lost] == 1 and not p.kv_len.any()


@pytest.mark.parametrize("bad", [-5, 81, 2**31 - 1, -2**31])
def test_slots_with_lengths_out_of_range(engine, bad):
    """They are not forked, forked into or resized; items beside them are done."""
    p = Pool(page=16, max_pages=5)
    p.do(engine, "resize", [0, 1], [40, 50], ok=True)
    p.kv_len[0] = p.m_len[0] = bad
    for call, a, b, done in (("fork", [0, 1], [5, 6], ([1], [6])), ("fork", [1, 1], [0, 7], ([1], [7])),
                             ("resize", [0, 1], [16, 70], ([1], [70])), ("resize", [0, 6], [0, 3], ([6], [3]))):
        getattr(engine, f"kv_{call}_dev")(p.pages, ints(a), ints(b))
        with pytest.raises(hb.CudaError, match="out of range"):
            engine.sync()
        getattr(p, call)(*done)
        p.same()


def test_holders_and_free_pages_are_those_before_the_call(engine):
    """In a pool with one page left: of two that cut inside the page they share, the second finds none; one that cuts
    inside a page whose other holder goes in the same call takes a copy, and what the other gives back is free after it."""
    p = Pool(n_pages=4, slots=3, page=16, max_pages=4)
    p.do(engine, "resize", [0], [48], ok=True)
    p.do(engine, "fork", [0], [1], ok=True)
    p.do(engine, "resize", [0, 1], [40, 40], ok=False)
    assert p.m_len[:2] == [40, 48] and p.m_table[0][2] == 3
    p.do(engine, "resize", [0], [0], ok=True)
    assert p.m_refs == [1, 1, 1, 0]
    p.do(engine, "fork", [1], [0], ok=True)
    p.do(engine, "resize", [0, 1], [0, 20], ok=True)
    assert p.m_table[1][1] == 3 and p.m_refs == [1, 0, 0, 1]
    p.do(engine, "fork", [1], [0], ok=True)
    p.do(engine, "resize", [0, 2], [0, 32], ok=False)
    assert p.m_len == [0, 20, 0] and p.m_refs == [1, 0, 0, 1]


@pytest.mark.parametrize("page,fits", [(2**26, True), (2**26 + 1, False), (2**27, False)])
def test_pages_of_more_tokens_than_a_copy_counts_are_refused(engine, page, fits):
    """The description alone: no call gets as far as the pools."""
    p = Pool(page=16, layers=1, max_pages=7)
    p.pages._keep[-1][0].page_size = page
    none = ints([])
    for call in (lambda: engine.kv_resize_dev(p.pages, none, none), lambda: engine.kv_fork_dev(p.pages, none, none)):
        if fits:
            call()
        else:
            with pytest.raises(hb.CudaError, match="2\\^26"):
                call()
