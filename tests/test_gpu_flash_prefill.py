"""Attention of packed sequences (fused.flash_prefill) against 64-bit torch, over packed rows and over page pools.

Bound per output element, relative to A = sum_t p_t |v_t| (p the exact probabilities): the probabilities are rounded to bf16
(2^-8 of each at most), a score is off by at most d = (8 MFMA steps + 4) 2^-24 of scale * sum |q_i k_i| plus 2^-22 of its own size
(the fp32 exponent's argument), which moves numerator and denominator by a factor e^(+-d) each, and the fp32 sums over n keys
add n / 16 + 64 steps of 2^-24; then half a bf16 step of the result.
"""
import math

import pytest
import torch

from palu_tt import fused
from palu_tt.cache import LatentCache

pytestmark = pytest.mark.gpu

HD = 128
BF = torch.bfloat16


def _ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _cu(lens, dev):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).to(dev)


def _pages(lens, page, g, spare=3, slots=None):
    """A page table for rows of these lengths over shuffled pages (-1 past them), and the pool's page count."""
    need = [-(-n // page) for n in lens]
    total = sum(need) + spare
    perm = torch.randperm(total, generator=g)[:sum(need)].tolist()
    slots = slots or max(1, max(need))
    table = []
    for n in need:
        table.append(perm[:n] + [-1] * (slots - n))
        perm = perm[n:]
    return torch.tensor(table, dtype=torch.int32), total


def _keys_of(pool, table, b, n):
    """Positions 0 .. n - 1 of row b, [n, heads, width], from a row-major pool."""
    page = pool.shape[2]
    ids = table[b, :-(-n // page)].long().clamp(0, pool.shape[0] - 1)
    return pool[ids].transpose(1, 2).reshape(-1, pool.shape[1], pool.shape[3])[:n]


def _exact(q, k, v, pos, scale):
    """One sequence in 64 bits: q [L, n_q, 128], k [n, n_kv, 128], v [n, n_kv, w], row i at position pos[i] (negative: zeros).
    Returns (out, bound) [L, n_q, w]."""
    L, nq, _ = q.shape
    n, nkv, w = v.shape
    rep = nq // nkv
    out = torch.zeros(L, nq, w, dtype=torch.float64, device=q.device)
    err = torch.zeros_like(out)
    seen = torch.arange(n, device=q.device) <= pos[:, None]                         # [L, n]
    for h in range(nq):
        qq, kk, vv = q[:, h].double(), k[:, h // rep].double(), v[:, h // rep].double()
        s = (qq @ kk.T.contiguous()) * scale
        s = torch.where(seen, s, -math.inf)
        p = torch.softmax(s, -1).nan_to_num(0.0)
        mag = (qq.abs() @ kk.abs().T.contiguous()) * abs(scale)
        d = (torch.where(seen, mag, 0).amax(-1) * 12 * 2.0 ** -24 + torch.where(seen, s, 0).abs().amax(-1) * 2.0 ** -22)[:, None]
        out[:, h] = p @ vv
        a = p @ vv.abs()
        err[:, h] = a * (2.0 ** -8 + 2 * d + (n / 16 + 64) * 2.0 ** -24) + 2.0 ** -8 * out[:, h].abs() + 1e-30
    return out, err


def _check(got, exp, err):
    assert torch.isfinite(got).all()
    r = ((got.double() - exp).abs() / (err * 1.001)).max().item() if got.numel() else 0.0
    assert r <= 1.0, f"error {r:.3f} of the bound"


def _packed(lens, nq, nkv, w, dev, seed=0, std=1.5):
    g = torch.Generator().manual_seed(seed)
    T = sum(lens)
    q = (torch.randn(T, nq, HD, generator=g) * std).to(dev, BF)
    k = torch.randn(T, nkv, HD, generator=g).to(dev, BF)
    v = torch.randn(T, nkv, w, generator=g).to(dev, BF)
    return q, k, v


def _packed_check(q, k, v, lens, scale=HD ** -0.5, **kw):
    dev = q.device
    got = fused.flash_prefill(q, k, v, _cu(lens, dev), **kw)
    at = 0
    for n in lens:
        if n:
            sl = slice(at, at + n)
            _check(got[sl], *_exact(q[sl], k[sl], v[sl], torch.arange(n, device=dev), scale))
        at += n
    return got


# lengths around the 32-row waves, 64-key tiles and 128-row tiles; head groups that divide the 128 rows and that don't
_LENS = [[1], [2, 1, 31], [32, 33, 1, 63], [64, 65, 127], [128, 129, 7], [300, 0, 17, 255, 0], [1025]]


@pytest.mark.parametrize("lens", _LENS, ids=str)
@pytest.mark.parametrize("nq,nkv", [(4, 4), (8, 2), (6, 2), (7, 1), (32, 1)])
def test_packed_lengths_and_groups(gpu, lens, nq, nkv):
    _packed_check(*_packed(lens, nq, nkv, 128, gpu, seed=sum(lens)), lens)


@pytest.mark.parametrize("w", [16, 32, 48, 64, 80, 96, 112, 128])
def test_packed_value_widths(gpu, w):
    lens = [70, 3, 200]
    _packed_check(*_packed(lens, 8, 2, w, gpu, seed=w), lens)


def test_more_query_heads_than_rows_of_a_tile(gpu):
    lens = [3, 9]
    _packed_check(*_packed(lens, 150, 1, 64, gpu), lens)


@pytest.mark.parametrize("n", [64, 65, 200, 256, 257, 1000])
def test_more_sequences_than_lanes(gpu, n):
    g = torch.Generator().manual_seed(n)
    lens = torch.randint(0, 20, (n,), generator=g).tolist()
    lens[n // 2], lens[-1] = 500, 150
    _packed_check(*_packed(lens, 4, 2, 64, gpu), lens)


def test_many_sequences_over_pages(gpu):
    g = torch.Generator().manual_seed(9)
    new, ctx = (torch.randint(lo, 30, (300,), generator=g).tolist() for lo in (0, 1))
    ctx[250] = 700
    _paged_check(new, ctx, 4, 2, 64, 32, "rows", gpu)


def test_sequence_tables_that_make_no_sense_stay_inside_the_rows(gpu):
    """Offsets that fall, or lie past the rows: what is computed is not defined, but nothing outside `out` is written."""
    q, k, v = _packed([100], 4, 2, 64, gpu)
    for cu in ([0, 50, 30, 200], [-5, 40, 100], [90, 10, 100], [200, 300, 400], [0] * 400 + [100, 0, 100, 7]):
        guard = torch.full((300, 4, 64), 7.0, dtype=BF, device=gpu)
        fused.flash_prefill(q, k, v, _ints(cu, gpu), out=guard[100:200])
        assert (guard[:100] == 7).all() and (guard[200:] == 7).all() and torch.isfinite(guard).all()


def test_strided_views_of_a_projection(gpu):
    """q, k and v as column views of one projection's rows, an unrelated column block between them."""
    g = torch.Generator().manual_seed(2)
    lens, nq, nkv, w = [90, 41], 8, 2, 64
    cols = nq * HD + 40 + nkv * (HD + w)
    rows = torch.randn(sum(lens), cols, generator=g).to(gpu, BF)
    q = rows[:, :nq * HD].view(-1, nq, HD)
    k = rows[:, nq * HD + 40:nq * HD + 40 + nkv * HD].view(-1, nkv, HD)
    v = rows[:, nq * HD + 40 + nkv * HD:].view(-1, nkv, w)
    assert not k.is_contiguous()
    got = _packed_check(q, k, v, lens)
    assert torch.equal(got, fused.flash_prefill(q.contiguous(), k.contiguous(), v.contiguous(), _cu(lens, gpu)))
    # heads before rows in memory
    t = lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(got, fused.flash_prefill(t(q), t(k), t(v), _cu(lens, gpu)))


@pytest.mark.parametrize("scale", [-0.05, 0.0, 0.4])
def test_scales(gpu, scale):
    lens = [100, 30]
    q, k, v = _packed(lens, 4, 2, 64, gpu)
    got = fused.flash_prefill(q, k, v, _cu(lens, gpu), scale=scale)
    for sl in (slice(0, 100), slice(100, 130)):
        _check(got[sl], *_exact(q[sl], k[sl], v[sl], torch.arange(sl.stop - sl.start, device=gpu), scale))


def test_rows_of_no_sequence_keep_what_they_held(gpu):
    lens = [40, 25]
    q, k, v = _packed(lens + [30], 4, 2, 64, gpu)                       # a padded batch: 30 rows behind the last sequence
    out = torch.full((95, 4, 64), 7.0, dtype=BF, device=gpu)
    got = fused.flash_prefill(q, k, v, _cu(lens, gpu), out=out)
    assert got is out and (out[65:] == 7).all()
    assert torch.equal(out[:65], fused.flash_prefill(q[:65], k[:65], v[:65], _cu(lens, gpu)))


def test_large_scores_underflow_to_exact_zeros(gpu):
    """Scores spread over hundreds: one key takes all the weight, and late large scores rescale what came before."""
    lens = [200]
    q, k, v = _packed(lens, 4, 2, 64, gpu, std=60.0)
    _packed_check(q, k, v, lens)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("layout", ["packed", "rows", "tiled"])
def test_non_finite_values_reach_only_the_rows_that_see_them(gpu, bad, layout):
    lens, at = [150, 70], 101                                            # position 101 of the first sequence
    q, k, v = _packed(lens, 4, 2, 64, gpu)
    if layout == "packed":
        run = lambda kk, vv: fused.flash_prefill(q, kk, vv, _cu(lens, gpu))
    else:
        run = lambda kk, vv: _paged_run(q, kk, vv, lens, [0, 0], 32, layout)[0]
    clean = run(k, v)
    v2 = v.clone()
    v2[at, 1, 5] = bad
    got = run(k, v2)
    hit = torch.zeros_like(clean, dtype=torch.bool)
    hit[at:150, 2:, 5] = True
    assert torch.equal(got[~hit], clean[~hit])
    if math.isnan(bad):
        assert got[hit].isnan().all()
    else:
        assert ((got[hit] == bad) | got[hit].isnan()).all() and (got[at, 2:, 5] == bad).all()   # its own row weighs it
    k2 = k.clone()
    k2[at, 0, 0] = math.nan
    got = run(k2, v)
    hit = torch.zeros_like(clean, dtype=torch.bool)
    hit[at:150, :2] = True
    assert torch.equal(got[~hit], clean[~hit]) and got[hit].isnan().all()


def _paged_run(q, k, v, new, ctx, page, layout, garbage=math.nan, **kw):
    """flash_prefill over pages that hold k / v of every sequence (ctx + new positions each, [positions, heads, width] one after
    another); unused positions and pages hold `garbage`."""
    dev = q.device
    g = torch.Generator().manual_seed(11)
    lens = [a + b for a, b in zip(new, ctx)]
    table, n_pages = _pages(lens, page, g)
    pools = []
    for t in (k, v):
        pool = torch.full((n_pages, t.shape[1], page, t.shape[2]), garbage, dtype=BF, device=dev)
        at = 0
        for b, n in enumerate(lens):
            for p in range(0, n, page):
                m = min(page, n - p)
                pool[table[b, p // page], :, :m] = t[at + p:at + p + m].transpose(0, 1)
            at += n
        pools.append(pool)
    kp, vp = pools
    if layout == "tiled":
        kp, vp = LatentCache.from_rows(kp, "k"), LatentCache.from_rows(vp, "v")
    out = fused.flash_prefill(q, kp, vp, _cu(new, dev), page_table_tensor=table.to(dev), start_pos=_ints(ctx, dev), **kw)
    return out, pools, table


def _paged_check(new, ctx, nq, nkv, w, page, layout, dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    total = sum(new) + sum(ctx)
    q = (torch.randn(sum(new), nq, HD, generator=g) * 1.5).to(dev, BF)
    k = torch.randn(total, nkv, HD, generator=g).to(dev, BF)
    v = torch.randn(total, nkv, w, generator=g).to(dev, BF)
    got, _, _ = _paged_run(q, k, v, new, ctx, page, layout)
    a = c = 0
    for n, x in zip(new, ctx):
        if n:
            _check(got[a:a + n], *_exact(q[a:a + n], k[c:c + n + x], v[c:c + n + x], x + torch.arange(n, device=dev), HD ** -0.5))
        a, c = a + n, c + n + x
    return got


@pytest.mark.parametrize("layout", ["rows", "tiled"])
@pytest.mark.parametrize("page", [32, 64, 256])
@pytest.mark.parametrize("new,ctx", [([1], [0]), ([5, 1, 40], [3, 200, 0]), ([130, 64, 1], [77, 64, 511]), ([0, 33], [40, 95])], ids=str)
def test_paged(gpu, layout, page, new, ctx):
    _paged_check(new, ctx, 8, 2, 128, page, layout, gpu, seed=page)


@pytest.mark.parametrize("layout,w", [("rows", 32), ("rows", 64), ("rows", 96), ("tiled", 48), ("tiled", 80), ("tiled", 96)])
def test_paged_value_widths(gpu, layout, w):
    _paged_check([50, 7], [100, 300], 4, 2, w, 64, layout, gpu, seed=w)


@pytest.mark.parametrize("layout", ["rows", "tiled"])
@pytest.mark.parametrize("new,ctx", [([1], [5000]), ([1, 3], [20000, 9]), ([17, 1, 2], [6000, 700, 130]), ([260], [3000])], ids=str)
def test_few_rows_over_long_contexts_are_split_and_joined(gpu, layout, new, ctx):
    _paged_check(new, ctx, 8, 2, 64, 64, layout, gpu, seed=ctx[0])


@pytest.mark.parametrize("layout", ["rows", "tiled"])
@pytest.mark.parametrize("rows", [1, 3, 6])
def test_more_pieces_than_the_chip_holds_at_once(gpu, layout, rows):
    """Some hundred tiles per KV head, some of them cut: all of the work order, and joins of 1, 8 and more rows."""
    g = torch.Generator().manual_seed(rows)
    ctx = torch.randint(1, 900, (100,), generator=g).tolist()
    ctx[3], ctx[40], ctx[99] = 9000, 12_000, 7000
    _paged_check([rows] * 100, ctx, 32, 8, 48, 32, layout, gpu, seed=rows)


def test_cut_contexts_of_more_query_heads_than_rows_of_a_tile(gpu):
    _paged_check([2, 1], [5000, 30], 256, 1, 16, 64, "rows", gpu, seed=3)


def test_non_finite_values_of_cut_contexts(gpu):
    """A NaN or infinity in one piece reaches the rows of its sequence and KV head, through the join."""
    new, ctx = [3, 1], [6000, 700]
    g = torch.Generator().manual_seed(6)
    q = torch.randn(4, 4, HD, generator=g).to(gpu, BF)
    k, v = (torch.randn(6704, 2, w, generator=g).to(gpu, BF) for w in (HD, 64))
    run = lambda k, v: _paged_run(q, k, v, new, ctx, 64, "rows")[0]
    clean = run(k, v)
    for bad in (math.nan, math.inf):
        v2 = v.clone()
        v2[4321, 1, 5] = bad
        got = run(k, v2)
        hit = torch.zeros_like(clean, dtype=torch.bool)
        hit[:3, 2:, 5] = True
        assert torch.equal(got[~hit], clean[~hit]) and (got[hit].isnan() | (got[hit] == bad)).all()
    k2 = k.clone()
    k2[70, 0, 9] = math.nan
    got = run(k2, v)
    hit = torch.zeros_like(clean, dtype=torch.bool)
    hit[:3, :2] = True
    assert torch.equal(got[~hit], clean[~hit]) and got[hit].isnan().all()


def test_single_tokens_agree_with_the_flash_decode(gpu):
    """One new row per sequence is a decode step: the stock flash-decode over the same pages, both against 64 bits elsewhere;
    here to each other within the roundings of both (the bound above, twice, for values of spread 1)."""
    new, ctx = [1, 1, 1], [0, 500, 1999]
    g = torch.Generator().manual_seed(4)
    q = torch.randn(3, 8, HD, generator=g).to(gpu, BF)
    k, v = (torch.randn(sum(new) + sum(ctx), 2, HD, generator=g).to(gpu, BF) for _ in range(2))
    got, (kp, vp), table = _paged_run(q, k, v, new, ctx, 64, "rows", garbage=0.0)
    dec = fused.flash_decode(q[None], kp, vp, _ints(ctx, gpu), page_table_tensor=table.to(gpu))[0]
    at = 0
    for b, x in enumerate(ctx):
        exp, err = _exact(q[b:b + 1], k[at:at + x + 1], v[at:at + x + 1], torch.tensor([x], device=gpu), HD ** -0.5)
        assert ((got[b] - dec[b]).double().abs() <= 2 * err[0] + 2.0 ** -8 * exp[0].abs()).all()
        at += x + 1


def test_rows_before_position_zero_and_past_the_table(gpu):
    """Rows at negative positions see nothing and give zeros; rows past the table's end see all that it holds."""
    g = torch.Generator().manual_seed(6)
    q = torch.randn(40, 4, HD, generator=g).to(gpu, BF)
    kp, vp = (torch.randn(4, 2, 32, HD, generator=g).to(gpu, BF) for _ in range(2))
    table = _ints([[2, 0], [1, 3]], gpu)
    got = fused.flash_prefill(q, kp, vp, _ints([0, 20, 40], gpu), page_table_tensor=table, start_pos=_ints([-7, 55], gpu))
    assert (got[:7] == 0).all()
    for b, (lo, hi, start) in enumerate([(7, 20, 0), (20, 40, 55)]):
        k, v = _keys_of(kp, table, b, 64), _keys_of(vp, table, b, 64)
        pos = (start + torch.arange(hi - lo, device=gpu)).clamp(max=63)
        _check(got[lo:hi], *_exact(q[lo:hi], k, v, pos, HD ** -0.5))
    assert (fused.flash_prefill(q, kp, vp, _ints([0, 20, 40], gpu), page_table_tensor=table, start_pos=_ints([-100, -20], gpu)) == 0).all()


def test_page_ids_outside_the_pool_stay_inside_it(gpu):
    g = torch.Generator().manual_seed(7)
    q = torch.randn(4, 4, HD, generator=g).to(gpu, BF)
    kp, vp = (torch.randn(3, 2, 32, HD, generator=g).to(gpu, BF) for _ in range(2))
    run = lambda t: fused.flash_prefill(q, kp, vp, _ints([0, 4], gpu), page_table_tensor=_ints(t, gpu), start_pos=_ints([60], gpu))
    assert torch.equal(run([[-5, 999]]), run([[0, 2]]))


def test_pool_offsets_past_32_bits(gpu):
    """Pages at the end of a pool of more than 2^32 bytes and 2^31 elements."""
    n_pages, page = 70000, 32
    kp = torch.empty(n_pages, 8, page, HD, dtype=BF, device=gpu)
    assert kp.numel() > 2 ** 31
    g = torch.Generator().manual_seed(8)
    ids = [n_pages - 1, 3, n_pages - 2]
    small = torch.randn(3, 8, page, HD, generator=g).to(gpu, BF)
    kp[ids] = small
    q = torch.randn(20, 8, HD, generator=g).to(gpu, BF)
    kw = dict(start_pos=_ints([70], gpu))
    got = fused.flash_prefill(q, kp, kp, _ints([0, 20], gpu), page_table_tensor=_ints([ids], gpu), **kw)
    assert torch.equal(got, fused.flash_prefill(q, small, small, _ints([0, 20], gpu), page_table_tensor=_ints([[0, 1, 2]], gpu), **kw))


def test_streams_and_graph_replays(gpu):
    """Two packed calls on two streams at once, and a captured call replayed between eager ones with new inputs (a split one:
    its partial results go through the workspace)."""
    new, ctx = [3, 20], [4000, 900]
    g = torch.Generator().manual_seed(9)
    q = torch.randn(23, 8, HD, generator=g).to(gpu, BF)
    k, v = (torch.randn(sum(new) + sum(ctx), 2, HD, generator=g).to(gpu, BF) for _ in range(2))
    alone, (kp, vp), table = _paged_run(q, k, v, new, ctx, 64, "rows")
    args = (_cu(new, gpu),)
    kw = dict(page_table_tensor=table.to(gpu), start_pos=_ints(ctx, gpu))
    run = lambda x: fused.flash_prefill(x, kp, vp, *args, **kw)
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [[], []]
    torch.cuda.synchronize()
    for _ in range(10):
        for s, o in zip(streams, outs):
            with torch.cuda.stream(s):
                o.append(run(q))
    torch.cuda.synchronize()
    assert all(torch.equal(o, alone) for os in outs for o in os)
    static = q.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = run(static)
    for i in range(4):
        x = torch.randn(23, 8, HD, generator=g).to(gpu, BF)
        static.copy_(x)
        graph.replay()
        exp = run(x)
        torch.cuda.synchronize()
        assert torch.equal(y, exp)


def test_workspace_and_out_are_the_callers(gpu):
    from palu_tt import _native
    new, ctx = [2], [5000]
    g = torch.Generator().manual_seed(10)
    q = torch.randn(2, 8, HD, generator=g).to(gpu, BF)
    k, v = (torch.randn(5002, 2, HD, generator=g).to(gpu, BF) for _ in range(2))
    exp, (kp, vp), table = _paged_run(q, k, v, new, ctx, 64, "rows")
    need = _native.load().palu_flash_prefill_workspace_bytes(2, 1, 8, 2, table.shape[1] * 64, HD)
    assert need > 0
    kw = dict(page_table_tensor=table.to(gpu), start_pos=_ints(ctx, gpu))
    for fill in (0, 255):                                                # any contents will do
        ws = torch.full((need,), fill, dtype=torch.uint8, device=gpu)
        out = torch.empty(2, 8, HD, dtype=BF, device=gpu)
        assert torch.equal(fused.flash_prefill(q, kp, vp, _cu(new, gpu), workspace=ws, out=out, **kw), exp)
    with pytest.raises(RuntimeError, match="workspace"):
        fused.flash_prefill(q, kp, vp, _cu(new, gpu), workspace=torch.empty(need - 1, dtype=torch.uint8, device=gpu), **kw)


def test_empty_batches_and_refusals(gpu):
    q, k, v = _packed([8], 4, 2, 64, gpu)
    cu = _cu([8], gpu)
    assert fused.flash_prefill(q[:0], k[:0], v[:0], _ints([0, 0], gpu)).shape == (0, 4, 64)
    for args, what in [((q.float(), k, v, cu), "bfloat16"), ((q[:, :, :64], k, v, cu), "q must be"), ((q, k[:7], v, cu), "rows of q"),
                       ((q, k, v[:, :, ::2], cu), "contiguous heads"), ((q[:, :3], k, v, cu), "multiple of the KV head"),
                       ((q, k, v[:, :, :40], cu), "head_dim_v"), ((q, k, v, cu[:1]), "at least one"), ((q, k, v, cu.float()), "integer"),
                       ((q.cpu(), k, v, cu), "GPU")]:
        with pytest.raises(RuntimeError, match=what):
            fused.flash_prefill(*args)
    with pytest.raises(RuntimeError, match="start_pos needs"):
        fused.flash_prefill(q, k, v, cu, start_pos=_ints([0], gpu))
    with pytest.raises(RuntimeError, match="backward"):
        fused.flash_prefill(q.requires_grad_(), k, v, cu)
    with torch.no_grad():
        fused.flash_prefill(q, k, v, cu)
    q = q.detach()
    pool = torch.zeros(2, 2, 48, HD, dtype=BF, device=gpu)
    with pytest.raises(RuntimeError, match="power of two"):
        fused.flash_prefill(q, pool, pool, cu, page_table_tensor=_ints([[0, 1]], gpu))
    pool = torch.zeros(2, 2, 32, HD, dtype=BF, device=gpu)
    with pytest.raises(RuntimeError, match="rows for batch"):
        fused.flash_prefill(q, pool, pool, cu, page_table_tensor=_ints([[0], [1]], gpu))
    with pytest.raises(RuntimeError, match="tile order"):
        fused.flash_prefill(q, LatentCache.from_rows(pool, "v"), LatentCache.from_rows(pool, "v"), cu, page_table_tensor=_ints([[0]], gpu))


# A mean of equal values is that value: the sum of the weights that divides has to be that of the rounded weights that multiplied. A
# dominating key's probability is rounded by up to 2^-8 where it is not the running maximum's own (which lags behind by up to 2^8);
# divided by the sum of unrounded ones that is up to 2^-8 of the result, half a bf16 step near the lower end of a binade and a
# whole one near the upper. The fp32 sums of n keys are off by (n + 64) 2^-23 together, 2^-12 for n = 2000: less than half the
# 2^-9 between a bf16 value and the nearest rounding border (just below a power of two), so the result is the value itself.
_CONSTANTS = [1.9921875, 1.0, 1.9921875 * 2.0 ** 20, -1.5, -1.9921875, 2.0 ** -30]


def _constant_values(rows, nkv, w, dev):
    c = torch.tensor(_CONSTANTS, dtype=BF, device=dev).repeat(-(-w // len(_CONSTANTS)))[:w]
    v = torch.stack([c.roll(j) for j in range(nkv)])
    return v.expand(rows, nkv, w).contiguous(), v


@pytest.mark.parametrize("std", [0.5, 3.0, 20.0])
def test_equal_values_come_back_exactly(gpu, std):
    lens = [1, 70, 300, 1000, 129]
    q, k, _ = _packed(lens, 8, 2, 64, gpu, seed=int(std * 2), std=std)
    vals, c = _constant_values(sum(lens), 2, 64, gpu)
    got = fused.flash_prefill(q, k, vals, _cu(lens, gpu))
    assert torch.equal(got, c.repeat_interleave(4, 0).expand_as(got))


@pytest.mark.parametrize("layout", ["rows", "tiled"])
@pytest.mark.parametrize("new,ctx", [([40, 7], [100, 500]), ([1, 3], [2000, 9])], ids=str)
def test_equal_values_in_pages_come_back_exactly(gpu, layout, new, ctx):
    g = torch.Generator().manual_seed(12)
    q = (torch.randn(sum(new), 8, HD, generator=g) * 4).to(gpu, BF)
    k = torch.randn(sum(new) + sum(ctx), 2, HD, generator=g).to(gpu, BF)
    vals, c = _constant_values(sum(new) + sum(ctx), 2, 64, gpu)
    got = _paged_run(q, k, vals, new, ctx, 64, layout)[0]
    assert torch.equal(got, c.repeat_interleave(4, 0).expand_as(got))


def test_values_that_cancel(gpu):
    """Neighbouring keys of almost equal scores and opposite values: the result is small beside sum p |v|, of which the rounding
    of the probabilities is up to 2^-8. (The bound of every test here; where the result is small it is the larger part.)"""
    lens = [400, 33]
    q, k, v = _packed(lens, 8, 2, 64, gpu, seed=13)
    k[1::2], v[1::2] = k[:-1:2][:k[1::2].shape[0]], -v[:-1:2][:v[1::2].shape[0]]
    got = _packed_check(q, k, v, lens)
    k[1::2, :, 0] += 2.0 ** -5                                          # no longer equal: what is left is a difference of weights
    assert got[1::2][:200].abs().max() < 0.05 and _packed_check(q, k, v, lens).isfinite().all()


@pytest.mark.parametrize("nq,nkv", [(6, 2), (7, 1), (18, 3), (40, 8)])
@pytest.mark.parametrize("new,ctx", [([1, 5], [5000, 30]), ([40, 3, 1], [3000, 7000, 300]), ([1], [290])], ids=str)
def test_cut_contexts_of_head_groups_that_do_not_divide_a_tile(gpu, nq, nkv, new, ctx):
    _paged_check(new, ctx, nq, nkv, 48, 32, "rows", gpu, seed=nq)


@pytest.mark.parametrize("rows,B,nq,nkv", [(1, 200, 4, 1), (3, 60, 8, 2), (1, 256, 3, 1), (2, 31, 32, 8)])
def test_overlapping_sequences_stay_inside_the_workspace(gpu, rows, B, nq, nkv):
    """Offsets that fall back to the first row again and again, all over long contexts: more pieces than the workspace holds. What
    comes out is not defined, what lies around the output and the workspace keeps what it holds."""
    from palu_tt import _native
    g = torch.Generator().manual_seed(rows)
    q = torch.randn(rows, nq, HD, generator=g).to(gpu, BF)
    kp, vp = (torch.randn(5, nkv, 64, w, generator=g).to(gpu, BF) for w in (HD, 64))
    table = torch.randint(0, 5, (2 * B, 500), generator=g).to(gpu, torch.int32)[:min(256, 2 * B)]
    B = table.shape[0]
    cu = _ints([0, rows] * (B // 2) + [0], gpu)[:B + 1]
    need = _native.load().palu_flash_prefill_workspace_bytes(rows, B, nq, nkv, 500 * 64, 64)
    ws, out = torch.full((need + 8192,), 77, dtype=torch.uint8, device=gpu), torch.full((rows + 2, nq, 64), 7.0, dtype=BF, device=gpu)
    fused.flash_prefill(q, kp, vp, cu, page_table_tensor=table, start_pos=torch.full((B,), 31_000, dtype=torch.int32, device=gpu),
                        out=out[1:-1], workspace=ws[4096:4096 + need])
    assert need and (ws[:4096] == 77).all() and (ws[4096 + need:] == 77).all() and (out[0] == 7).all() and (out[-1] == 7).all()
