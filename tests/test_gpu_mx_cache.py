"""Rows into quantised caches and any paged cache's rows back out (fused.paged_fill_cache, paged_update_cache, paged_read_cache)
against cache.mx_quantize, whose values the CPU tests hold to the definition: bytes and scales are equal, what is not written stays."""
import math

import pytest
import torch

from palu_tt import cache, fused
from palu_tt.cache import LatentCache, MXCache
from palu_tt.pages import PagePools

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _cu(lens, dev):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).to(dev)


def _noise(n, G, page, w, role, fmt, dev, seed=0):
    """A pool of arbitrary bytes."""
    g = torch.Generator().manual_seed(seed)
    data = torch.randint(0, 256, (n, G, page // 32, MXCache.block_bytes(fmt, w)), generator=g, dtype=torch.uint8)
    return MXCache(data.to(dev), role, fmt, w)


def _values(T, G, w, seed=0):
    """Rows of many magnitudes, with blocks of zeros, of tiny, huge and equal values and of values that are not finite."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, G, w, generator=g) * torch.exp(torch.randn(T, G, w // 32, generator=g) * 3).repeat_interleave(32, -1)
    blocks = x.view(-1, 32)
    for i, v in enumerate([0.0, -0.0, 2.0 ** -120, 3e38, 5e-41, 464.0, 1.0]):
        blocks[i + 1::23] = v
    blocks[9::41, 3] = math.nan
    blocks[11::53, 30] = -math.inf
    blocks[12::31] *= 2.0 ** -125
    return x.to(BF)


def _same(a, b):
    """Equal, NaN where NaN is; False alone in a failure's message."""
    return bool(((a == b) | ((a != a) & (b != b))).all())


def _where(lens, start, table, page):
    """(row, page id, position in the page) of every packed row that has a place in the table and pool."""
    out, at = [], 0
    for b, n in enumerate(lens):
        for i in range(n):
            p = start[b] + i
            if 0 <= p < table.shape[1] * page:
                out.append((at + i, int(table[b, p // page]), p % page))
        at += n
    return out


_CASES = [([1], [0]), ([1, 1, 1, 1], [0, 31, 32, 63]), ([57, 0, 3], [100, 5, 64]), ([33, 8, 9, 16], [0, 8, 23, 40]), ([130], [-3]),
          ([40], [170]), ([7, 200], [1, 9])]


def _pages(lens, start, page, slots, seed=1):
    n = len(lens) * slots + 3
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(n, generator=g)[:len(lens) * slots].view(len(lens), slots).to(torch.int32), n


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("role", ["k", "v"])
@pytest.mark.parametrize("lens,start", _CASES, ids=str)
@pytest.mark.parametrize("G,w,page", [(2, 128, 64), (3, 32, 32), (1, 96, 128), (5, 64, 64), (2, 512, 32)])
def test_fill_and_read(gpu, fmt, role, lens, start, G, w, page):
    T, slots = sum(lens), -(-200 // page)
    table, n = _pages(lens, start, page, slots)
    pool, rows = _noise(n, G, page, w, role, fmt, gpu), _values(T, G, w)
    codes, scales = pool.parts()
    exp_codes, exp_scales = codes.clone(), scales.clone()
    c, s = cache.mx_quantize(rows, fmt)
    where = _where(lens, start, table, page)
    for t, pid, p in where:
        exp_codes[pid, :, p], exp_scales[pid, :, p] = c[t].to(gpu), s[t].to(gpu)
    args = (_cu(lens, gpu), table.to(gpu), _ints(start, gpu))
    # the rows are columns of a wider tensor, whose rows behind the last sequence are not looked at
    wide = torch.full((T + 4, G * w + 24), math.nan, dtype=BF, device=gpu)
    wide[:T, 8:8 + G * w] = rows.view(T, -1).to(gpu)
    fused.paged_fill_cache(pool, wide[:, 8:8 + G * w].unflatten(1, (G, w)), *args)
    got_codes, got_scales = pool.parts()
    assert _same(got_scales, exp_scales) and _same(got_codes, exp_codes)
    back = fused.paged_read_cache(pool, T + 2, *args, out=torch.full((T + 2, G, w), 7.0, dtype=BF, device=gpu))
    exp = torch.zeros(T, G, w, dtype=BF)
    for t, _, _ in where:
        exp[t] = cache.mx_dequantize(c[t], s[t], fmt)
    assert _same(back[:T], exp.to(gpu)) and (back[T:] == 7).all()


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("role", ["k", "v"])
def test_every_bf16_value(gpu, fmt, role):
    """All 65536, each in a block of its own kind: alone, and beside a larger one."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(BF)
    blocks = torch.zeros(2, 65536, 32, dtype=BF)
    blocks[0, :, 5] = x
    blocks[1, :, 5], blocks[1, :, 20] = x, (x.float() * 37).to(BF)
    rows = blocks.view(1024, 1, 4096)[:, :, :].view(1024 * 8, 1, 512)
    pool = MXCache.zeros(8192 // 64, 1, 64, 512, gpu, role, fmt)
    table = torch.arange(8192 // 64, dtype=torch.int32, device=gpu)[None]
    fused.paged_fill_cache(pool, rows.to(gpu), _cu([8192], gpu), table)
    exp = MXCache.from_rows(rows.view(128, 64, 1, 512).transpose(1, 2), role, fmt)
    assert _same(pool.data.cpu(), exp.data)
    assert _same(pool.to_rows().cpu(), exp.to_rows())


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("role", ["k", "v"])
@pytest.mark.parametrize("paged", [True, False], ids=["paged", "contiguous"])
@pytest.mark.parametrize("G,w", [(8, 128), (1, 32), (3, 96), (2, 64)])
def test_append(gpu, fmt, role, paged, G, w):
    B, page, slots = 9, 64, 3
    idx = [0, 31, 32, 63, 64, 100, -1, 191, 192]
    table, n = _pages([1] * B, idx, page, slots)
    table[5, 1] = n + 2                                                  # a page that is not there
    pool = _noise(n if paged else B, G, page if paged else 192, w, role, fmt, gpu, seed=3)
    rows = _values(B, G, w, seed=w)
    codes, scales = (x.clone() for x in pool.parts())
    c, s = cache.mx_quantize(rows, fmt)
    for b, p in enumerate(idx):
        if 0 <= p < 192 and not (paged and b == 5):
            at = (int(table[b, p // page]), p % page) if paged else (b, p)
            codes[at[0], :, at[1]], scales[at[0], :, at[1]] = c[b].to(gpu), s[b].to(gpu)
    fused.paged_update_cache(pool, rows.to(gpu), _ints(idx, gpu), page_table=table.to(gpu) if paged else None)
    got = pool.parts()
    assert _same(got[0], codes) and _same(got[1], scales)


@pytest.mark.parametrize("layout", ["rows", "tiled k", "tiled v"])
@pytest.mark.parametrize("w", [8, 16, 40, 48, 64, 112, 128, 512])
def test_read_of_bf16_pools(gpu, layout, w):
    if layout != "rows" and w % 16:
        w += 8
    lens, start, page = [57, 1, 0, 90], [100, 64, 3, -2], 32
    table, n = _pages(lens, start, page, 6)
    table[0, 4], table[3, 1] = -1, n                                     # pages that are not there
    g = torch.Generator().manual_seed(w)
    pool = torch.randn(n, 3, page, w, generator=g).to(gpu, BF)
    store = pool if layout == "rows" else LatentCache.from_rows(pool, layout[-1])
    got = fused.paged_read_cache(store, sum(lens), _cu(lens, gpu), table.to(gpu), _ints(start, gpu))
    exp = torch.zeros(sum(lens), 3, w, dtype=BF, device=gpu)
    for t, pid, p in _where(lens, start, table, page):
        if 0 <= pid < n:
            exp[t] = pool[pid, :, p]
    assert _same(got, exp)


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
def test_pages_that_are_not_there(gpu, fmt):
    pool = _noise(4, 2, 32, 64, "v", fmt, gpu)
    before = pool.data.clone()
    table, cu = _ints([[-1, 4], [2 ** 30, -2 ** 31]], gpu), _cu([64, 50], gpu)
    fused.paged_fill_cache(pool, _values(114, 2, 64).to(gpu), cu, table)
    assert _same(pool.data, before) and (fused.paged_read_cache(pool, 114, cu, table) == 0).all()


def test_offsets_past_32_bits(gpu):
    """Pages at the end of a pool of more than 2^32 bytes."""
    n, G, w = 140_000, 8, 128
    pool = MXCache(torch.empty(n, G, 1, MXCache.block_bytes("fp8", w), dtype=torch.uint8, device=gpu), "v", "fp8", w)
    assert pool.data.numel() > 2 ** 32
    rows, cu, table = _values(96, G, w, seed=5).to(gpu), _cu([96], gpu), _ints([[n - 1, 3, n - 2]], gpu)
    small = MXCache.zeros(3, G, 32, w, gpu, "v", "fp8")
    fused.paged_fill_cache(pool, rows, cu, table)
    fused.paged_fill_cache(small, rows, cu, _ints([[0, 1, 2]], gpu))
    assert _same(pool.data[[n - 1, 3, n - 2]], small.data)
    assert torch.equal(fused.paged_read_cache(pool, 96, cu, table).view(torch.int16),
                       fused.paged_read_cache(small, 96, cu, _ints([[0, 1, 2]], gpu)).view(torch.int16))


def test_streams_and_graph_replays(gpu):
    """A captured fill, append and read, replayed with other rows and positions between eager work; and on a second stream."""
    pool, table, cu = MXCache.zeros(12, 2, 32, 64, gpu, "k", "fp4"), _ints([[3, 5, 7], [1, 0, 2]], gpu), _cu([40, 9], gpu)
    rows, one, start, idx = (x.to(gpu) for x in (_values(49, 2, 64), _values(2, 2, 64, 1), torch.tensor([0, 20], dtype=torch.int32),
                                                 torch.tensor([40, 29], dtype=torch.int32)))

    def run(pool, rows, one, start, idx):
        fused.paged_fill_cache(pool, rows, cu, table, start_pos=start)
        fused.paged_update_cache(pool, one, idx, page_table=table)
        return fused.paged_read_cache(pool, 60, _cu([50, 10], gpu) if pool is not static else cu2, table, start_pos=start)

    cu2, static = _cu([50, 10], gpu), pool
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run(pool, rows, one, start, idx)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = run(pool, rows, one, start, idx)
    for i in range(4):
        rows.copy_(_values(49, 2, 64, 10 + i))
        one.copy_(_values(2, 2, 64, 20 + i))
        start.add_(i)
        idx.add_(i)
        other = MXCache(pool.data.clone(), "k", "fp4", 64)
        graph.replay()
        exp = run(other, rows, one, start, idx)
        torch.cuda.synchronize()
        assert _same(pool.data, other.data) and _same(y, exp)


def test_page_pools_copy_quantised_pages(gpu):
    """Forks copy the page that is written next, a compaction moves whole pages, scales and all."""
    pools = [_noise(8, 2, 64, 128, "k", "fp8", gpu), _noise(8, 2, 64, 32, "v", "fp4", gpu, 1), torch.randn(8, 2, 64, 32, device=gpu).to(BF)]
    before = [(p.data if isinstance(p, MXCache) else p).clone() for p in pools]
    table, lengths = PagePools(pools).update(_ints([[6, 4], [-1, -1]], gpu), _ints([100, 0], gpu), parents=_ints([0, 0], gpu),
                                             new_lengths=_ints([101, 101], gpu))
    assert lengths.tolist() == [101, 101] and table[0, 0] == table[1, 0] == 6 and {int(table[0, 1]), int(table[1, 1])} == {4, 0}
    for p, b in zip(pools, before):
        data = p.data if isinstance(p, MXCache) else p
        assert _same(data[0], b[4]) and _same(data[1:], b[1:])
    table, n = PagePools(pools).compact(table, lengths)
    assert n.item() == 3
    for p, b in zip(pools, before):
        data = p.data if isinstance(p, MXCache) else p
        assert _same(data[table[0].long()], b[[6, 4]]) and _same(data[table[1].long()], b[[6, 4]])
