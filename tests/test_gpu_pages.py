"""Packed rows into page pools (fused.paged_fill_cache) and the page table (pages.PagePools) against plain Python: all of it moves
values and counts pages, so every comparison is for equality."""
import random

import pytest
import torch

from palu_tt import fused
from palu_tt.cache import LatentCache
from palu_tt.pages import PagePools

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _cu(lens, dev):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).to(dev)


# ---- fill ---------------------------------------------------------------------------------------

def _fill_case(layout, w, page, new, start, dev, G=3, spread=0, seed=0):
    g = torch.Generator().manual_seed(seed)
    cap = max([max(s, 0) + n for s, n in zip(start, new)] + [1])
    slots = -(-cap // page)
    B = len(new)
    n_pages = B * slots + 2
    table = torch.randperm(n_pages, generator=g)[:B * slots].view(B, slots).to(torch.int32)
    T = sum(new)
    src = torch.randn(T, G, w + spread, generator=g).to(BF)[:, :, :w]
    pool = torch.randn(n_pages, G, page, w, generator=g).to(BF)
    exp = pool.clone()
    at = 0
    for b, (n, s) in enumerate(zip(new, start)):
        for i in range(n):
            if 0 <= s + i < slots * page:
                exp[table[b, (s + i) // page], :, (s + i) % page] = src[at + i]
        at += n
    d_src = torch.randn(T, G, w + spread).to(dev, BF)
    d_src[:, :, :w] = src.to(dev)
    d_src = d_src[:, :, :w]
    d_pool = pool.to(dev)
    cache = d_pool if layout == "rows" else LatentCache.from_rows(d_pool, layout)
    fused.paged_fill_cache(cache, d_src, _cu(new, dev), table.to(dev), start_pos=_ints(start, dev))
    got = cache if layout == "rows" else cache.to_rows()
    assert torch.equal(got.cpu(), exp)


@pytest.mark.parametrize("layout", ["rows", "k", "v"])
@pytest.mark.parametrize("new,start", [([1], [0]), ([5, 1, 40], [3, 31, 0]), ([33, 0, 64, 100], [32, 7, 1, 95]), ([7, 300], [1, 500])],
                         ids=str)
@pytest.mark.parametrize("w,page", [(64, 32), (128, 64), (32, 256)])
def test_fill(gpu, layout, new, start, w, page):
    _fill_case(layout, w, page, new, start, gpu)


@pytest.mark.parametrize("layout,w", [("rows", 8), ("rows", 40), ("rows", 512), ("k", 16), ("k", 48), ("k", 112), ("v", 16), ("v", 80),
                                      ("v", 512), ("k", 512)])
def test_fill_widths_and_strides(gpu, layout, w):
    _fill_case(layout, w, 64, [50, 13], [9, 64], gpu, spread=24, seed=w)


def test_fill_of_many_sequences(gpu):
    g = torch.Generator().manual_seed(1)
    new = torch.randint(0, 50, (150,), generator=g).tolist()
    start = torch.randint(0, 90, (150,), generator=g).tolist()
    _fill_case("rows", 32, 32, new, start, gpu)


def test_fill_skips_positions_and_pages_that_do_not_exist(gpu):
    rows = torch.ones(40, 1, 32, dtype=BF, device=gpu)
    for role in ("rows", "k", "v"):
        pool = torch.zeros(3, 1, 32, 32, dtype=BF, device=gpu)
        cache = pool if role == "rows" else LatentCache.from_rows(pool, role)
        # the first sequence starts before position 0 and its second page is not in the pool; the second runs past the table; rows
        # 38 and 39 belong to none
        fused.paged_fill_cache(cache, rows, _ints([0, 30, 38], gpu), _ints([[2, 7], [0, 1]], gpu), start_pos=_ints([-10, 60], gpu))
        got = cache if role == "rows" else cache.to_rows()
        exp = torch.zeros_like(pool)
        exp[2, :, :20] = 1
        exp[1, :, 28:] = 1
        assert torch.equal(got, exp)


def test_fill_refusals(gpu):
    pool = torch.zeros(3, 2, 32, 32, dtype=BF, device=gpu)
    rows, cu, table = torch.zeros(4, 2, 32, dtype=BF, device=gpu), _ints([0, 4], gpu), _ints([[0]], gpu)
    fused.paged_fill_cache(pool, rows[:0], _ints([0, 0], gpu), table)
    for args, what in [((pool, rows[:, :1], cu, table), "rows must be"), ((pool, rows.float(), cu, table), "bfloat16"),
                       ((pool, rows, cu, _ints([[0], [1]], gpu)), "rows for batch"), ((pool, rows, cu[:1], table), "at least one"),
                       ((pool[:, :, :16].contiguous(), rows, cu, table), "power of two")]:
        with pytest.raises(RuntimeError, match=what):
            fused.paged_fill_cache(*args)


# ---- update ---------------------------------------------------------------------------------------

def _update(table, lens, parents, new, n_pages, page):
    """(table, lengths, copies [(from, to)]) after an update, one row after the other."""
    B, slots = len(table), len(table[0])
    ok = lambda p: 0 <= p < n_pages
    parents = list(range(B)) if parents is None else [p if 0 <= p < B else -1 for p in parents]
    have = [min(max(lens[p], 0), slots * page) if p >= 0 else 0 for p in parents]
    want = have if new is None else [min(max(n, 0), slots * page) for n in new]
    keep = [min(a, b) for a, b in zip(have, want)]
    rows = [table[p][:k // page] if p >= 0 else [] for p, k in zip(parents, keep)]
    used = {p for r in rows for p in r if ok(p)}
    last, writers = [], set()
    for b in range(B):
        p = table[parents[b]][keep[b] // page] if keep[b] % page else -1
        if ok(p) and p not in used and p not in writers:
            writers.add(p)
            rows[b] = rows[b] + [p]
            p = -1
        last.append(p)
    used |= writers
    free = [p for p in range(n_pages) if p not in used]
    copies, out, lengths = [], [], []
    for b in range(B):
        r = list(rows[b])
        while len(r) * page < want[b] and free:
            p = free.pop(0)
            if len(r) == keep[b] // page and ok(last[b]):
                copies.append((last[b], p))
            r.append(p)
        lengths.append(min(want[b], len(r) * page))
        out.append(r + [-1] * (slots - len(r)))
    return out, lengths, copies


def _pools(n_pages, page, dev, seed):
    g = torch.Generator().manual_seed(seed)
    a = torch.randn(n_pages, 2, page, 48, generator=g).to(dev, BF)        # a page of 4.5 KB or more, one of several pieces
    b = torch.randn(n_pages, 3, page, 96, generator=g).to(dev, BF)
    return [a, LatentCache.from_rows(b, "k")]


def _stores(pools):
    return [p.data if isinstance(p, LatentCache) else p for p in pools]


def _draw_rows(r, B, slots, page, n_pages, share):
    """A table of random rows over distinct pages, some of them then forked from others (shared whole pages)."""
    ids = r.sample(range(n_pages), min(n_pages, B * slots))
    table, lens = [], []
    for b in range(B):
        room = min(slots, len(ids))
        n = r.randint(0, room * page)
        k = -(-n // page)
        table.append(ids[:k] + [-1] * (slots - k))
        lens.append(n)
        ids = ids[k:]
    for b in range(B):
        if share and r.random() < share:
            a = r.randrange(B)
            n = min(lens[a], r.choice([lens[a], lens[a] // page * page, r.randint(0, lens[a])]))
            k = -(-n // page)
            table[b], lens[b] = table[a][:k] + [-1] * (slots - k), n
    return table, lens


def _run_update(dev, table, lens, parents, new, n_pages, page, seed=0):
    pools = _pools(n_pages, page, dev, seed)
    exp_pools = [s.clone() for s in _stores(pools)]
    opt = lambda x: None if x is None else _ints(x, dev)
    t0, l0 = _ints(table, dev), _ints(lens, dev)
    got_t, got_l = PagePools(pools).update(t0, l0, parents=opt(parents), new_lengths=opt(new))
    exp_t, exp_l, copies = _update(table, lens, parents, new, n_pages, page)
    assert got_l.tolist() == exp_l
    assert got_t.tolist() == exp_t
    assert t0.tolist() == table and l0.tolist() == lens                   # the old ones are not touched
    for s in exp_pools:
        if copies:
            s[[b for _, b in copies]] = s[[a for a, _ in copies]]
    assert all(torch.equal(x, y) for x, y in zip(_stores(pools), exp_pools))
    return copies


@pytest.mark.parametrize("B,slots,page,spare", [(1, 1, 32, 0), (1, 7, 32, 3), (4, 3, 32, 2), (7, 9, 64, 5), (33, 5, 32, 0), (64, 16, 32, 40),
                                                (300, 4, 32, 30), (1100, 2, 32, 5)])
def test_update_of_random_rows(gpu, B, slots, page, spare):
    """Forks, ends, cuts, growth and fresh rows at once, with pages to spare and without."""
    copied = 0
    for seed in range(4):
        r = random.Random(100 * B + seed)
        n_pages = max(1, B * slots * (1 + seed) // 4 + spare)
        table, lens = _draw_rows(r, B, slots, page, n_pages, 0.4 if seed % 2 else 0)
        parents = [r.randint(-1, B) for _ in range(B)] if seed else None
        new = [r.choice([0, r.randint(0, slots * page), r.randint(-3, slots * page + 40)]) for _ in range(B)]
        copied += len(_run_update(gpu, table, lens, parents, new, n_pages, page, seed))
    assert copied or B < 4


def test_update_without_lengths_or_parents(gpu):
    table, lens = [[3, 1, -1], [0, -1, -1], [-1, -1, -1]], [40, 32, 0]
    assert _run_update(gpu, table, lens, None, None, 6, 32) == []
    assert _run_update(gpu, table, lens, [0, 0, 1], None, 6, 32) == [(1, 2)]     # page 0 is row 2's now


def test_update_beam_rules(gpu):
    """Who keeps a page that several rows would write: the first of them, unless a row holds it whole."""
    table, lens = [[4, 2, 7], [5, -1, -1], [6, 3, -1]], [80, 10, 64]
    # rows 1 and 2 fork from row 0 in page 7: row 0 keeps it
    assert _run_update(gpu, table, lens, [0, 0, 0], None, 9, 32) == [(7, 0), (7, 1)]
    # row 0 goes on from row 1; the first of rows 1 and 2 keeps page 7
    assert _run_update(gpu, table, lens, [1, 0, 0], [11, 81, 90], 9, 32) == [(7, 0)]
    # a row cut into page 2, which row 1 holds whole, copies it though it is the first
    assert _run_update(gpu, table, lens, [0, 0, 2], [40, 70, 64], 9, 32) == [(2, 0)]


def test_update_grants_what_the_pool_has(gpu):
    table, lens = [[0, -1, -1, -1], [1, -1, -1, -1], [2, -1, -1, -1]], [20, 32, 5]
    _run_update(gpu, table, lens, None, [100, 128, 6], 5, 32)              # 2 free pages, 6 wanted: the first row gets them
    _run_update(gpu, table, lens, [0, 0, 0], [128, 21, 21], 3, 32)         # forks without a page for the copy fall back to whole pages
    _run_update(gpu, table, lens, [0, 0, 0], [21, 21, 21], 2, 32)


def test_update_of_tables_with_ids_outside_the_pool(gpu):
    table, lens = [[-1, 9, 1, -1], [0, 77, -5, -1]], [96, 90]
    for new in ([97, 100], [33, 70], [96, 90], [10, 40]):
        _run_update(gpu, table, lens, None, new, 6, 32)
        _run_update(gpu, table, lens, [1, 0], new, 6, 32)


@pytest.mark.parametrize("n_pages,B", [(700_000, 3), (1_000_000, 2), (64, 4096), (200_001, 900)])
def test_update_of_large_pools_and_batches(gpu, n_pages, B):
    r = random.Random(n_pages)
    pool = torch.zeros(n_pages, 1, 32, 8, dtype=BF, device=gpu)
    slots = 3
    table = [[r.randrange(n_pages) for _ in range(slots)] for _ in range(B)]
    lens = [r.randint(0, 96) for _ in range(B)]
    new = [min(96, n + r.randint(0, 40)) for n in lens]
    got_t, got_l = PagePools([pool]).update(_ints(table, gpu), _ints(lens, gpu), new_lengths=_ints(new, gpu))
    exp_t, exp_l, _ = _update(table, lens, None, new, n_pages, 32)
    assert got_l.tolist() == exp_l and got_t.tolist() == exp_t


@pytest.mark.parametrize("B,slots,page,n_pages", [(1, 3, 32, 40), (5, 6, 32, 33), (12, 8, 64, 200), (40, 4, 32, 161), (2, 2, 32, 90_000)])
def test_compact(gpu, B, slots, page, n_pages):
    for seed in range(4):
        r = random.Random(seed + B)
        table, lens = _draw_rows(r, B, slots, page, n_pages, 0.3)
        if seed == 3:
            table[0][:2], lens[0] = [n_pages + 3, -1], 40                   # ids outside the pool stay as they are
        pools = _pools(n_pages, page, gpu, seed) if n_pages < 1000 else [torch.randn(n_pages, 1, page, 8, device=gpu).to(BF)]
        exp_pools = [s.clone() for s in _stores(pools)]
        got, n = PagePools(pools).compact(_ints(table, gpu), _ints(lens, gpu))
        live = sorted({p for row, k in zip(table, lens) for p in row[:-(-k // page)] if 0 <= p < n_pages})
        gaps = [p for p in range(len(live)) if p not in set(live)]
        to = dict(zip([p for p in live if p >= len(live)], gaps))
        exp = [[to.get(p, p) if j < -(-k // page) else -1 for j, p in enumerate(row)] for row, k in zip(table, lens)]
        assert n.tolist() == [len(live)] and got.tolist() == exp
        for s in exp_pools:
            if to:
                s[list(to.values())] = s[list(to.keys())]
        assert all(torch.equal(x, y) for x, y in zip(_stores(pools), exp_pools))


def test_pages_of_a_pool_past_32_bits(gpu):
    """A copy and a move at the end of a pool of more than 2^32 bytes."""
    n_pages = 40_000
    pool = torch.empty(n_pages, 8, 32, 128, dtype=BF, device=gpu)
    assert pool.numel() * 2 > 2 ** 31 and pool.numel() * 2 // n_pages * n_pages > 2 ** 31
    last = torch.randn(8, 32, 128).to(gpu, BF)
    pool[n_pages - 1] = last
    h = PagePools([pool])
    table, lens = h.update(_ints([[n_pages - 1], [-1]], gpu), _ints([5, 0], gpu), parents=_ints([0, 0], gpu), new_lengths=_ints([6, 6], gpu))
    assert table.tolist() == [[n_pages - 1], [0]] and lens.tolist() == [6, 6] and torch.equal(pool[0], last)
    pool[0] = 0
    table, n = h.compact(table[:1].contiguous(), lens[:1].contiguous())
    assert table.tolist() == [[0]] and n.tolist() == [1] and torch.equal(pool[0], last)


def test_more_pools_than_one_launch_takes(gpu):
    pools = [torch.randn(4, 1, 32, 8).to(gpu, BF) for _ in range(150)]
    exp = [p[1].clone() for p in pools]
    PagePools(pools).update(_ints([[1], [-1]], gpu), _ints([3, 0], gpu), parents=_ints([0, 0], gpu))
    assert all(torch.equal(p[0], e) for p, e in zip(pools, exp))


def test_update_and_compact_in_graphs_and_on_streams(gpu):
    """A captured step (every row one position more) replayed on tables that change between the replays, beside a captured
    compaction with a workspace of its own; then two updates over different pools on two streams at once."""
    page, n_pages, B, slots = 32, 60, 6, 8
    pools = _pools(n_pages, page, gpu, 0)
    h = PagePools(pools)
    r = random.Random(3)
    table, lens = _draw_rows(r, B, slots - 1, page, n_pages - 12, 0.5)
    table = [row + [-1] for row in table]
    t, ln, new = _ints(table, gpu), _ints(lens, gpu), _ints([n + 1 for n in lens], gpu)
    h.update(t, ln, new_lengths=new)                                      # sets kernel attributes outside capture
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        t1, l1 = h.update(t, ln, new_lengths=new)
    with torch.cuda.graph(g2):
        t2, n2 = h.compact(t, ln)
    for step in range(5):
        g1.replay()
        exp_t, exp_l, _ = _update(table, lens, None, [n + 1 for n in lens], n_pages, page)
        assert t1.tolist() == exp_t and l1.tolist() == exp_l
        table, lens = exp_t, exp_l
        t.copy_(t1)
        ln.copy_(l1)
        new.copy_(l1 + 1)
        if step == 2:
            g2.replay()
            live = sorted({p for row, k in zip(table, lens) for p in row[:-(-k // page)]})
            assert n2.tolist() == [len(live)]
            t.copy_(t2)
            table = t2.tolist()
            assert sorted({p for row, k in zip(table, lens) for p in row[:-(-k // page)]}) == list(range(len(live)))
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    others = PagePools(_pools(n_pages, page, gpu, 1))
    torch.cuda.synchronize()
    outs = []
    for _ in range(10):
        for s, x in ((s1, h), (s2, others)):
            with torch.cuda.stream(s):
                outs.append(x.update(t, ln, parents=_ints([0] * B, gpu), new_lengths=new))
    torch.cuda.synchronize()
    assert all(torch.equal(a[0], outs[0][0]) and torch.equal(a[1], outs[0][1]) for a in outs)


def test_page_refusals(gpu):
    pool = torch.zeros(4, 2, 32, 16, dtype=BF, device=gpu)
    t, ln = _ints([[0, 1]], gpu), _ints([40], gpu)
    with pytest.raises(RuntimeError, match="at least one pool"):
        PagePools([])
    with pytest.raises(RuntimeError, match="agree"):
        PagePools([pool, torch.zeros(5, 2, 32, 16, dtype=BF, device=gpu)])
    with pytest.raises(RuntimeError, match="overlap"):
        PagePools([pool, pool])
    with pytest.raises(RuntimeError, match="contiguous"):
        PagePools([pool[:, :, :, ::2]])
    with pytest.raises(RuntimeError, match="bf16"):
        PagePools([pool.float()])
    h = PagePools([pool])
    for kw, what in [(dict(parents=_ints([0, 0], gpu)), "parents"), (dict(new_lengths=torch.zeros(1, device=gpu)), "integer"),
                     (dict(out=(t, _ints([0], gpu))), "memory of its own"), (dict(out=(_ints([[0, 1]], gpu), ln)), "memory of its own"),
                     (dict(out=(_ints([[0]], gpu), _ints([0], gpu))), "out: page_table"),
                     (dict(workspace=torch.empty(8, dtype=torch.uint8, device=gpu)), "workspace")]:
        with pytest.raises(RuntimeError, match=what):
            h.update(t, ln, **kw)
    with pytest.raises(RuntimeError, match="lengths"):
        h.update(t, _ints([1, 2], gpu))
    with pytest.raises(RuntimeError, match="power of two"):
        PagePools([torch.zeros(4, 2, 48, 16, dtype=BF, device=gpu)]).update(t, ln)
    with pytest.raises(RuntimeError, match="at least one row"):
        h.compact(t[:0], ln[:0])
    assert h.update(t[:0], ln[:0])[0].shape == (0, 2)


@pytest.mark.parametrize("shape", [(0, 2, 32, 16), (4, 0, 32, 16), (4, 2, 32, 0)])
def test_empty_pools_are_refused(gpu, shape):
    with pytest.raises(RuntimeError, match="not empty"):
        PagePools([torch.zeros(*shape, dtype=BF, device=gpu)])


@pytest.mark.parametrize("role", ["rows", "k"])
def test_caches_whose_storage_was_replaced(gpu, role):
    """Between two calls a cache gets another storage: the copies go there, and the old one keeps what it holds."""
    g = torch.Generator().manual_seed(4)
    rand = lambda: torch.randn(6, 2, 32, 32, generator=g).to(gpu, BF)
    cache = rand() if role == "rows" else LatentCache.from_rows(rand(), role)
    other = rand()
    h = PagePools([cache, other])
    t, ln = _ints([[4], [-1]], gpu), _ints([5, 0], gpu)
    fork = lambda: h.update(t, ln, parents=_ints([0, 0], gpu), new_lengths=_ints([6, 6], gpu))
    fork()
    store = cache if role == "rows" else cache.data
    old = store.detach()
    was = old.clone()
    new = rand() if role == "rows" else LatentCache.from_rows(rand(), role).data
    if role == "rows":
        cache.data = new
    else:
        cache.data = new.clone()
    store = cache if role == "rows" else cache.data
    table, lengths = fork()
    assert table.tolist() == [[4], [0]] and lengths.tolist() == [6, 6]
    assert torch.equal(store[0], store[4]) and torch.equal(store[1:], new[1:]) and torch.equal(old, was)
    assert torch.equal(other[0], other[4])
    store[3] = 7
    table, n = h.compact(_ints([[3]], gpu), _ints([2], gpu))
    assert table.tolist() == [[0]] and (store[0] == 7).all() and torch.equal(old, was)
