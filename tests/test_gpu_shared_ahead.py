"""fused.flash_decode_shared where prefixes are read ahead (a launch of their own, taken where the page tables can name more than 64
MiB): every test looks at the workspace to see that the prefixes' pieces were written. Batches and bound are test_gpu_step's."""
import math

import pytest
import torch

from palu_tt import _native, fused
from palu_tt.cache import LatentCache, MXCache
from palu_tt.pages import PagePools
from test_gpu_step import _GROUPS, BF, HD, LAYOUTS, Batch, _check, _constants, _exact, _ints, _store

pytestmark = pytest.mark.gpu

LIMIT, UNUSED = 64 << 20, 0xAA
BLOCK = {"rows": 64, "tiled": 64, "fp8": 33, "fp4": 17}                  # bytes of a 32-position block for a channel


def _named(layout, B, nkv, w, positions):
    """Bytes that the tables of a batch can name."""
    return B * nkv * (positions // 32) * BLOCK[layout] * (HD + w)


def _written(ws, need, B, nq, nkv, w):
    """(the prefixes' pieces, the rows' records: 32 bytes each, at the end) were written."""
    lo = -(-_native.load().palu_mx_decode_workspace_bytes(B, nq, nkv, w) // 16) * 16
    return bool((ws[lo:need - 32 * B] != UNUSED).any()), bool((ws[need - 32 * B:need] != UNUSED).any())


def _run(x, positions=65536, ahead=True, pieces=True, cu=True, **kw):
    """The call over tables for that many positions: both launches (ahead), with pieces of prefixes written, or one."""
    B, nq = len(x.lens), x.q.shape[2]
    own = torch.nn.functional.pad(x.own, (0, positions // x.page - x.own.shape[1]), value=-1).to(x.dev)
    assert (_named(x.layout, B, x.nkv, x.w, own.shape[1] * x.page) > LIMIT) == ahead
    n = x.cu.numel() - 1 if cu else 1
    need = _native.load().palu_flash_decode_shared_workspace_bytes(B, n, nq, x.nkv, x.w)
    ws = torch.full((need,), UNUSED, dtype=torch.uint8, device=x.dev)
    got = fused.flash_decode_shared(x.q, x.k, x.v, x.pos, own, x.shared, x.cu if cu else None, workspace=ws, **kw)
    assert _written(ws, need, B, nq, x.nkv, x.w) == (ahead and pieces, ahead)
    return got


def _padded(layout, lens, nkv, w):
    """With as many short rows of no group as it takes to read ahead over tables for 65536 positions."""
    rows = LIMIT // _named(layout, 1, nkv, w, 65536) + 1
    return lens + [33 + b for b in range(rows - len(lens))]


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("groups,shared,lens", _GROUPS, ids=str)
@pytest.mark.parametrize("nq,nkv", [(8, 2), (6, 2), (7, 1), (16, 1), (4, 4)])
@pytest.mark.parametrize("empty", [0, 20])                               # empty groups behind the others: fewer columns a wave
def test_groups(gpu, layout, groups, shared, lens, nq, nkv, empty):
    x = Batch(gpu, layout, _padded(layout, lens, nkv, 64), nq, nkv, groups=groups + [0] * empty, shared=shared + [64] * empty,
              seed=sum(lens), page=64 if sum(lens) % 2 else 32)
    x.check(_run(x, pieces=any(n > 1 and s >= 32 for n, s in zip(groups, shared))))


@pytest.mark.parametrize("layout", LAYOUTS)
def test_both_sides_of_the_bound(gpu, layout):
    x = Batch(gpu, layout, [330, 300, 299, 70, 66], 16, 8, 128, groups=[3, 2], shared=[290, 64])
    slots = LIMIT // _named(layout, 5, 8, 128, 32)
    x.check(_run(x, 32 * slots, ahead=False))
    x.check(_run(x, 32 * (slots + 1)))


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("rows", [[4, 1, 1], [1, 3, 1, 1, 1], [2, 1], [1, 2, 1, 1], [1, 1, 1], [1]], ids=str)
def test_lone_rows_beside_groups(gpu, layout, rows):
    shared = [900 if n == 1 else 700 for n in rows]
    lens = [s + 13 * i for i, (n, s) in enumerate(zip(rows, shared)) for _ in range(n)]
    x = Batch(gpu, layout, _padded(layout, lens, 4, 64), 16, 4, 64, 64, rows, shared, seed=len(lens))
    x.check(_run(x, pieces=any(n > 1 for n in rows)))


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("std", [0.5, 20.0])
def test_scales_and_output_types(gpu, layout, scale, dtype, std):
    x = Batch(gpu, layout, [200, 170, 161], 16, 4, groups=[3], shared=[160], std=std)
    got = _run(x, scale=scale, out_dtype=dtype)
    assert got.dtype == dtype
    x.check(got, scale)


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("std", [0.5, 3.0, 20.0])
def test_equal_values_come_back_exactly(gpu, layout, std):
    x = Batch(gpu, layout, [1000, 1400, 64, 2000, 1], 16, 4, groups=[3, 2], shared=[990, 640], std=std, seed=3)
    rows = _constants(x)
    assert torch.equal(_run(x)[0], rows.repeat_interleave(4, 0).expand(5, -1, -1))


@pytest.mark.parametrize("layout", LAYOUTS)
def test_nan_reaches_the_rows_that_see_it(gpu, layout):
    """One inside the prefix, which a row of the group that ends before it does not see; one behind it."""
    x = Batch(gpu, layout, [200, 90, 180, 100], 16, 4, groups=[3, 1], shared=[160, 0], garbage=0.0)
    clean = _run(x)
    for page, row, rows in ((3, 0, (0, 2)), (5, 2, (2,))):
        bad = x.krows.clone()
        bad[int(x.table[row, page]), 1, 5, 9] = math.nan
        k, x.k = x.k, _store(bad, "k", layout)[0]
        got, x.k = _run(x), k
        hit = torch.zeros_like(clean, dtype=torch.bool)
        hit[0, list(rows), 4:8] = True
        assert got[hit].isnan().all() and torch.equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("layout", LAYOUTS)
def test_without_groups_and_rows_of_no_group(gpu, layout):
    x = Batch(gpu, layout, [100, 70, 65, 90], 16, 4, groups=[4], shared=[64])
    assert torch.equal(_run(x), _run(x, cu=False))                       # no cu_groups: one group
    y = Batch(gpu, layout, [100, 70, 65, 90], 16, 4, groups=[1, 2], shared=[64, 64])     # rows 1 and 2; row 0 alone, row 3 of none
    y.cu, y.shared = _ints([1, 3], gpu), _ints([64], gpu)
    y.lead, y.blocks, y.own = [0, 1, 1, 3], [0, 2, 2, 0], y.table.clone()
    y.check(_run(y))


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("nq,nkv,prefix", [(2, 1, 60000), (10, 5, 33000)])
def test_a_long_prefix_beside_many_short_rows(gpu, layout, nq, nkv, prefix):
    """More items than workgroups, a few of which have hundreds of pieces of a prefix to join."""
    B = 600 if nkv == 1 else 110
    g = torch.Generator().manual_seed(nkv)
    lens = torch.randint(0, 200, (B - 3,), generator=g).tolist()
    lens = lens[:50] + [prefix + 33, prefix, prefix + 200] + lens[50:]
    x = Batch(gpu, layout, lens, nq, nkv, 64, 64, [50, 3], [0, prefix], seed=nkv, garbage=0.0)
    got = _run(x)
    x.check(got, rows=[0, 49, 50, 51, 52, 53, B - 1])
    assert torch.equal(got, _run(x))


@pytest.mark.parametrize("layout", LAYOUTS)
def test_a_few_pieces_beside_many_short_rows(gpu, layout):
    """More items than workgroups, each with seven pieces of the prefix, or up to three, to join."""
    lens = [2000 + 3 * b for b in range(66)] + [100 + b for b in range(4)] + [30] * 4
    x = Batch(gpu, layout, lens, 32, 8, 64, 64, [66, 4], [2000, 96], garbage=0.0)
    x.check(_run(x))


@pytest.mark.parametrize("layout", LAYOUTS)
def test_offsets_past_32_bits(gpu, layout):
    """The same batch over pools whose pages lie past 4 GiB and over ones of three pages."""
    n = 140_000 if layout in ("fp8", "fp4") else 70_000
    n *= 2 if layout == "fp4" else 1
    g = torch.Generator().manual_seed(8)
    rows = [torch.randn(3, 8, 32, HD, generator=g).to(gpu, BF) for _ in "kv"]
    small = [_store(r, role, layout)[0] for r, role in zip(rows, "kv")]
    ids, large = [n - 1, 3, n - 2], []
    for c, role in zip(small, "kv"):
        data = c if layout == "rows" else c.data
        pool = torch.empty(n, *data.shape[1:], dtype=data.dtype, device=gpu)
        assert pool.numel() * pool.element_size() > 2 ** 32
        pool[ids] = data
        large.append(pool if layout == "rows" else LatentCache(pool, role) if layout == "tiled" else MXCache(pool, role, layout, HD))
    q, pos, shared = torch.randn(1, 2, 8, HD, generator=g).to(gpu, BF), _ints([70, 95], gpu), _ints([64], gpu)
    need = _native.load().palu_flash_decode_shared_workspace_bytes(2, 1, 8, 8, HD)
    outs = []
    for pools, t in ((small, [0, 1, 2]), (large, ids)):
        ws = torch.full((need,), UNUSED, dtype=torch.uint8, device=gpu)
        table = torch.nn.functional.pad(_ints([t] * 2, gpu), (0, 2045), value=-1)
        outs.append(fused.flash_decode_shared(q, *pools, pos, table, shared, workspace=ws))
        assert _written(ws, need, 2, 8, 8, HD) == (True, True)
    assert torch.equal(*outs)
    for b, m in enumerate((71, 96)):
        k, v = ((r if layout in ("rows", "tiled") else _store(r, role, layout)[1]).transpose(1, 2).flatten(0, 1)[:m]
                for r, role in zip(rows, "kv"))
        _check(outs[0][0, b], *_exact(q[0, b], k, v))


@pytest.mark.parametrize("layout", LAYOUTS)
def test_a_server_s_run(gpu, layout):
    """Prompts, samples of them, steps, a sample that ends, a compaction, a captured step: tables for 65536 positions."""
    g = torch.Generator().manual_seed(6)
    rand = lambda *s: torch.randn(*s, generator=g).to(BF)
    n_pages, B, nq, nkv, w, page = 48, 7, 32, 8, 128, 32
    zeros = [torch.zeros(n_pages, nkv, page, x, dtype=BF, device=gpu) for x in (HD, w)]
    kp, vp = (_store(z, role, layout)[0] for z, role in zip(zeros, "kv"))
    pools = PagePools([kp, vp])
    table, lengths = torch.full((B, 65536 // page), -1, dtype=torch.int32, device=gpu), _ints([0] * B, gpu)
    groups, shared = _ints([0, 4, 5, 7], gpu), _ints([200, 0, 70], gpu)
    need = _native.load().palu_flash_decode_shared_workspace_bytes(B, 3, nq, nkv, w)

    def put(n, start=None):
        cu = torch.tensor([0] + n).cumsum(0).to(torch.int32).to(gpu)
        for pool, x in ((kp, HD), (vp, w)):
            fused.paged_fill_cache(pool, rand(sum(n), nkv, x).to(gpu), cu, table, start_pos=start)

    def step(q, ws):
        return fused.flash_decode_shared(q, kp, vp, lengths - 1, table, shared, groups, workspace=ws)

    def check(q, out):
        n = lengths.tolist()
        cu = torch.tensor([0] + n).cumsum(0).to(torch.int32).to(gpu)
        k, v = (fused.paged_read_cache(pool, sum(n), cu, table) for pool in (kp, vp))
        for b, (a, e) in enumerate(zip(cu.tolist(), cu.tolist()[1:])):
            if e > a:
                _check(out[0, b], *_exact(q[0, b], k[a:e], v[a:e]), f"row {b}:")
            else:
                assert (out[0, b] == 0).all()

    table, lengths = pools.update(table, lengths, new_lengths=_ints([200, 0, 0, 0, 90, 70, 0], gpu))
    put([200, 0, 0, 0, 90, 70, 0])
    table, lengths = pools.update(table, lengths, parents=_ints([0, 0, 0, 0, 4, 5, 5], gpu))
    for i in range(5):
        if i == 2:                                                       # the first sample ends
            table, lengths = pools.update(table, lengths, new_lengths=lengths * _ints([0, 1, 1, 1, 1, 1, 1], gpu))
        if i == 3:
            table, _ = pools.compact(table, lengths)
        live = [int(x > 0) for x in lengths.tolist()]
        start = lengths.clone()
        table, lengths = pools.update(table, lengths, new_lengths=lengths + _ints(live, gpu))
        put(live, start)
        q, ws = rand(1, B, nq, HD).to(gpu), torch.full((need,), UNUSED, dtype=torch.uint8, device=gpu)
        out = step(q, ws)
        assert _written(ws, need, B, nq, nkv, w) == (True, True)
        check(q, out)
    lengths = lengths.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step(q, ws)
    for _ in range(3):                                                   # a step further back each time
        graph.replay()
        exp = step(q, torch.empty_like(ws))
        torch.cuda.synchronize()
        assert torch.equal(y, exp)
        check(q, y)
        lengths.sub_(1).clamp_(min=0)
