"""fused.flash_decode_shared of groups whose first rows have ended: PagePools leaves such a row's table empty (-1), and the samples
that go on read their prefix through the first row that still has pages. Against 64-bit torch, with test_gpu_step's bound."""
import pytest
import torch

from palu_tt import fused
from palu_tt.cache import LatentCache, MXCache
from palu_tt.pages import PagePools
from test_gpu_step import BF, HD, LAYOUTS, Batch, _check, _exact, _ints

pytestmark = pytest.mark.gpu


def _batch(dev, layout, lens, groups, shared, **kw):
    """A batch in which rows of no positions have ended: their tables are empty, their group's prefix lies in the pages of its first
    row that has some; the other rows' entries before its end name a page of NaN."""
    x = Batch(dev, layout, lens, groups=groups, shared=shared, **kw)
    bad = int(x.own[x.own != x.table][0])
    x.own, at = x.table.clone(), 0
    for n in groups:
        lead = next((b for b in range(at, at + n) if lens[b]), at)
        for b in range(at, at + n):
            x.lead[b] = lead
            if b != lead:
                whole = x.blocks[b] * 32 // x.page
                x.own[b, :whole] = torch.where(x.own[b, :whole] >= 0, bad, -1)
        at += n
    return x


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("groups,shared,lens", [
    ([3], [100], [0, 130, 97]),
    ([4, 1, 3], [200, 64, 96], [0, 230, 201, 150, 70, 0, 0, 130]),       # a row that ends inside the prefix, two that have ended
    ([2, 3], [64, 500], [0, 0, 0, 510, 600]),                            # a whole group that has ended
    ([9, 3], [1000, 320], [0, 0, 1001, 0, 1200, 40, 1031, 0, 990, 330, 0, 321])], ids=str)
@pytest.mark.parametrize("nq,nkv", [(8, 2), (7, 1), (32, 8)])
@pytest.mark.parametrize("wide", [True, False])
def test_first_rows_that_have_ended(gpu, layout, groups, shared, lens, nq, nkv, wide):
    x = _batch(gpu, layout, lens, groups, shared, nq=nq, nkv=nkv, page=64 if nkv == 1 else 32, seed=sum(lens))
    x.check(x.decode_shared(wide))


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("B,ended,nkv", [(70, 64, 2), (150, 129, 2), (200, 131, 4)])
@pytest.mark.parametrize("wide", [True, False])
def test_many_rows_that_have_ended(gpu, layout, B, ended, nkv, wide):
    """More of them at a group's start than a wave looks at at once; more items than workgroups."""
    g = torch.Generator().manual_seed(B)
    lens = [0] * ended + [400] + [400 + int(torch.randint(0, 90, (), generator=g)) for _ in range(B - ended - 1)]
    lens[-1] = 0
    x = _batch(gpu, layout, lens, [B], [400], nq=4 * nkv, nkv=nkv, seed=B)
    x.check(x.decode_shared(wide), rows=[0, ended - 1, *range(ended, B)])


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("wide", [True, False])
def test_a_captured_call_follows_rows_that_end(gpu, layout, wide):
    x = _batch(gpu, layout, [700, 690, 800, 650], [4], [640], nq=16, nkv=2 if not wide else 4)
    x.own[1:, :640 // x.page] = x.own[0, :640 // x.page]                 # the samples of one prompt
    x.lead = [0] * 4
    if wide:
        x.own = torch.nn.functional.pad(x.own, (0, 65536 // x.page - x.own.shape[1]), value=-1)
    x.own = x.own.to(gpu)
    x.decode_shared(False)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = x.decode_shared(False)
    for ends in (None, 0, 2, 1):                                         # rows 0, 2 and 1 end, one after the other
        if ends is not None:
            x.own[ends], x.pos[ends], x.lens[ends] = -1, -1, 0
        for _ in range(2):
            graph.replay()
            exp = x.decode_shared(False)
            torch.cuda.synchronize()
            assert torch.equal(y, exp)
        x.check(y)


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("slots", [8, 65536 // 32])
def test_samples_of_a_pool_go_on_without_their_first(gpu, layout, slots):
    """As a server does it: a prompt, samples forked from it, the first of them ended, its place in the group kept; the pages are
    those of another request by then."""
    g = torch.Generator().manual_seed(4)
    rand = lambda *s: torch.randn(*s, generator=g).to(BF)
    n_pages, B, nq, nkv, w, page = 40, 6, 16, 4, 64, 32
    rows = [torch.zeros(n_pages, nkv, page, x, dtype=BF, device=gpu) for x in (HD, w)]
    if layout == "rows":
        kp, vp = rows
    elif layout == "tiled":
        kp, vp = (LatentCache.from_rows(r, role) for r, role in zip(rows, "kv"))
    else:
        kp, vp = (MXCache.from_rows(r, role, layout) for r, role in zip(rows, "kv"))
    pools = PagePools([kp, vp])
    table, lengths = torch.full((B, slots), -1, dtype=torch.int32, device=gpu), _ints([0] * B, gpu)

    def put(n, start):
        cu = torch.tensor([0] + n).cumsum(0).to(torch.int32).to(gpu)
        fused.paged_fill_cache(kp, rand(sum(n), nkv, HD).to(gpu), cu, table, start_pos=start)
        fused.paged_fill_cache(vp, rand(sum(n), nkv, w).to(gpu), cu, table, start_pos=start)

    table, lengths = pools.update(table, lengths, new_lengths=_ints([150, 0, 0, 0, 0, 0], gpu))
    put([150] + [0] * 5, None)
    table, lengths = pools.update(table, lengths, parents=_ints([0, 0, 0, 0, -1, -1], gpu))
    groups, shared = _ints([0, 4], gpu), _ints([150], gpu)
    for ended in ([], [0], [0], [0, 1]):
        n = [0 if b in ended else x for b, x in enumerate(lengths.tolist())]
        table, lengths = pools.update(table, lengths, new_lengths=_ints(n, gpu))     # those rows' pages are free again
        new = [int(x > 0) for x in n]
        new[4 if 1 in ended else 5] += 64                                            # another request takes pages
        start = lengths.clone()
        table, lengths = pools.update(table, lengths, new_lengths=lengths + _ints(new, gpu))
        put(new, start)
        q, pos = rand(1, B, nq, HD).to(gpu), lengths - 1
        out = fused.flash_decode_shared(q, kp, vp, pos, table, shared, groups)
        N, at = sum(lengths.tolist()), 0
        cu = torch.tensor([0] + lengths.tolist()).cumsum(0).to(torch.int32).to(gpu)
        k, v = fused.paged_read_cache(kp, N, cu, table), fused.paged_read_cache(vp, N, cu, table)
        for b, x in enumerate(lengths.tolist()):
            if x:
                exp, err = _exact(q[0, b], k[at:at + x], v[at:at + x])
                _check(out[0, b], exp, err, f"{ended} row {b}:")
            else:
                assert (out[0, b] == 0).all()
            at += x
