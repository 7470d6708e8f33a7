"""Decode attention over quantised caches (fused.flash_decode of MXCache) and of batches that share prefixes
(fused.flash_decode_shared, every layout) against 64-bit torch on what the caches hold.

Bound per output element, relative to A = sum_t p_t |v_t| (p the exact probabilities): the probabilities are rounded to bf16
(2^-8 of each at most), a score is off by at most d = (4 MFMA steps of 32 products + 4) 2^-24 of scale * sum |q_i k_i| plus 2^-22 of
its own size (the fp32 exponent's argument), which moves numerator and denominator by a factor e^(+-d) each, and the fp32 sums
over n keys and their parts add n / 16 + 128 steps of 2^-24; then half a step of a bf16 result. (An MFMA step adds its products and the
accumulator, each rounded or cut at most once per product: 32 steps of 2^-24 of the sum of magnitudes.)
"""
import math

import pytest
import torch

from palu_tt import _native, fused
from palu_tt.cache import LatentCache, MXCache

pytestmark = pytest.mark.gpu

HD = 128
BF = torch.bfloat16
LAYOUTS = ["rows", "tiled", "fp8", "fp4"]


def _ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _store(rows, role, layout):
    """(cache object, the rows that it holds)."""
    if layout == "rows":
        return rows, rows
    if layout == "tiled":
        return LatentCache.from_rows(rows, role), rows
    c = MXCache.from_rows(rows, role, layout)
    return c, c.to_rows()


def _exact(q, k, v, scale=HD ** -0.5, f32=False):
    """q [n_q, 128] over k [n, n_kv, 128], v [n, n_kv, w] in 64 bits: (out, bound) [n_q, w]."""
    nq, (n, nkv, w) = q.shape[0], v.shape
    rep = nq // nkv
    qq = q.double().view(nkv, rep, HD)
    kk, vv = k.double().transpose(0, 1), v.double().transpose(0, 1)
    s = (qq @ kk.transpose(1, 2).contiguous()) * scale
    p = torch.softmax(s, -1)
    mag = (qq.abs() @ kk.abs().transpose(1, 2).contiguous()) * abs(scale)
    d = mag.amax(-1, keepdim=True) * (128 + 4) * 2.0 ** -24 + s.abs().amax(-1, keepdim=True) * 2.0 ** -22
    out, a = p @ vv, p @ vv.abs()
    err = a * (2.0 ** -8 + 2 * d + (n / 16 + 128) * 2.0 ** -24) + (2.0 ** -24 if f32 else 2.0 ** -8) * out.abs() + 1e-30
    return out.reshape(nq, w), err.reshape(nq, w)


def _check(got, exp, err, what=""):
    assert torch.isfinite(got).all(), what
    r = ((got.double() - exp).abs() / (err * 1.001)).max().item()
    assert r <= 1.0, f"{what} error {r:.3f} of the bound"


class Batch:
    """Rows over page pools: lens[b] positions each (0: none); groups of rows whose first shared positions lie in the first
    row's pages, the other rows' entries before that pointing at pages of NaN."""

    def __init__(self, dev, layout, lens, nq=8, nkv=2, w=64, page=32, groups=None, shared=None, seed=0, std=1.5, garbage=math.nan, slots=None):
        g = torch.Generator().manual_seed(seed)
        B = len(lens)
        self.lens, self.layout, self.page, self.nkv, self.w = lens, layout, page, nkv, w
        slots = slots or max(1, max(-(-n // page) for n in lens))
        need = [-(-n // page) for n in lens]
        total = sum(need) + 3
        perm = torch.randperm(total, generator=g).tolist()
        bad = perm.pop()                                                 # the page of garbage
        self.table = torch.full((B, slots), -1, dtype=torch.int32)
        for b, n in enumerate(need):
            self.table[b, :n] = torch.tensor([perm.pop() for _ in range(n)], dtype=torch.int32)
        k, v = (torch.randn(total, nkv, page, x, generator=g).to(dev, BF) for x in (HD, w))
        k[bad] = garbage
        v[bad] = garbage
        for b, n in enumerate(lens):                                     # garbage behind every row's last position, too
            if n % page:
                last = int(self.table[b, n // page])
                k[last, :, n % page:] = garbage
                v[last, :, n % page:] = garbage
        self.lead, self.blocks = list(range(B)), [0] * B
        if groups:
            at = 0
            for rows, s in zip(groups, shared):
                for b in range(at, at + rows):
                    self.lead[b], self.blocks[b] = at, max(s, 0) // 32
                at += rows
        self.k, self.krows = _store(k, "k", layout)
        self.v, self.vrows = _store(v, "v", layout)
        self.own = self.table.clone()
        for b in range(B):                                               # whole pages that must not be read through the own table
            whole = self.blocks[b] * 32 // page
            if self.lead[b] != b:
                self.own[b, :whole] = torch.where(self.own[b, :whole] >= 0, bad, -1)
        self.q = (torch.randn(1, B, nq, HD, generator=g) * std).to(dev, BF)
        self.pos = _ints([n - 1 for n in lens], dev)
        self.dev = dev
        if groups:
            self.cu = torch.tensor([0] + groups).cumsum(0).to(torch.int32).to(dev)
            self.shared = _ints(shared, dev)

    def seen(self, pool, b):
        out = []
        for j in range(-(-self.lens[b] // 32)):
            row = self.lead[b] if j < self.blocks[b] else b
            pid = int(self.table[row, j * 32 // self.page])
            out.append(pool[pid, :, j * 32 % self.page:j * 32 % self.page + 32].transpose(0, 1))
        return torch.cat(out)[:self.lens[b]]

    def check(self, got, scale=HD ** -0.5, rows=None):
        assert got.shape == (1, len(self.lens), self.q.shape[2], self.w)
        for b in rows or range(len(self.lens)):
            if self.lens[b] == 0:
                assert (got[0, b] == 0).all()
                continue
            exp, err = _exact(self.q[0, b], self.seen(self.krows, b), self.seen(self.vrows, b), scale, got.dtype == torch.float32)
            _check(got[0, b], exp, err, f"row {b}:")

    def decode(self, **kw):
        return fused.flash_decode(self.q, self.k, self.v, self.pos, page_table_tensor=self.table.to(self.dev), **kw)

    def decode_shared(self, wide=True, **kw):
        """wide: over a table with room for 65536 positions, where prefixes are read ahead (but for a few rows in 4 bits)."""
        own = self.own
        if wide:
            own = torch.nn.functional.pad(own, (0, 65536 // self.page - own.shape[1]), value=-1)
        return fused.flash_decode_shared(self.q, self.k, self.v, self.pos, own.to(self.dev), self.shared, self.cu, **kw)


# ---- quantised caches ----------------------------------------------------------------------------

@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("lens", [[1], [32, 33, 31], [0, 64, 0, 7], [300, 1, 129], [513, 512, 511], [2100, 40]], ids=str)
@pytest.mark.parametrize("nq,nkv", [(4, 4), (8, 2), (6, 2), (7, 1), (16, 1), (32, 8)])
def test_lengths_and_head_groups(gpu, fmt, lens, nq, nkv):
    x = Batch(gpu, fmt, lens, nq, nkv, seed=sum(lens))
    x.check(x.decode())


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("w", [32, 64, 96, 128])
@pytest.mark.parametrize("page", [32, 64, 256, 4096])
def test_widths_and_page_sizes(gpu, fmt, w, page):
    x = Batch(gpu, fmt, [700, 5, 4097], w=w, page=page, seed=w + page)
    x.check(x.decode())


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("B,longest,nkv", [(1, 20000, 1), (3, 40000, 2), (64, 600, 8), (300, 90, 2), (17, 3000, 8), (700, 40, 1), (33, 5000, 1)])
def test_splits(gpu, fmt, B, longest, nkv):
    """Batches whose items are cut into pieces, and ones of which every workgroup takes an even share."""
    g = torch.Generator().manual_seed(B)
    lens = [longest] + torch.randint(0, longest + 1, (B - 1,), generator=g).tolist()
    x = Batch(gpu, fmt, lens, 4 * nkv, nkv, 32, 64, seed=B)
    x.check(x.decode(), rows=list(range(0, B, max(1, B // 40))))


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("B,nkv,nq,short,long", [
    (150, 4, 16, 60, []), (110, 5, 5, 256, []), (180, 3, 12, 200, [3000]), (400, 3, 3, 40, []), (300, 6, 18, 300, [20000, 700]),
    (70, 8, 32, 257, [288, 289, 5000]), (1100, 1, 16, 33, [900])])
def test_many_items(gpu, fmt, B, nkv, nq, short, long):
    """More items than workgroups: a KV head of a short row to a wave (numbers of them that are no multiple of 4, too), pieces of long
    rows between them, empty rows."""
    g = torch.Generator().manual_seed(B)
    lens = long + torch.randint(0, short + 1, (B - len(long),), generator=g).tolist()
    lens = [lens[i] for i in torch.randperm(B, generator=g).tolist()]
    x = Batch(gpu, fmt, lens, nq, nkv, 96 if nkv % 2 else 64, 64, seed=B)
    got = x.decode()
    x.check(got, rows=sorted({*range(0, B, max(1, B // 40)), *(b for b, n in enumerate(lens) if n > short), B - 1}))
    assert torch.equal(got, x.decode())


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("S,lens", [(32, [1, 32, 0]), (160, [160, 33, 1, 97]), (8192, [8192, 5000, 31])], ids=str)
def test_contiguous(gpu, fmt, S, lens):
    g = torch.Generator().manual_seed(S)
    B = len(lens)
    k, v = (torch.randn(B, 2, S, x, generator=g).to(gpu, BF) for x in (HD, 96))
    for b, n in enumerate(lens):
        k[b, :, n:], v[b, :, n:] = math.inf, math.nan
    (kc, kr), (vc, vr) = _store(k, "k", fmt), _store(v, "v", fmt)
    q = torch.randn(1, B, 8, HD, generator=g).to(gpu, BF)
    got = fused.flash_decode(q, kc, vc, _ints([n - 1 for n in lens], gpu))
    for b, n in enumerate(lens):
        if n:
            _check(got[0, b], *_exact(q[0, b], kr[b, :, :n].transpose(0, 1), vr[b, :, :n].transpose(0, 1)))
        else:
            assert (got[0, b] == 0).all()
    assert torch.equal(fused.scaled_dot_product_attention_decode(q, kc, vc, _ints([n - 1 for n in lens], gpu)), got)
    past = fused.flash_decode(q, kc, vc, _ints([S + 1000] * B, gpu))       # past the end: all positions
    assert torch.equal(past[0, 0], got[0, 0]) == (lens[0] == S)


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0, 1e-3])
@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_scales_and_output_types(gpu, fmt, scale, dtype):
    x = Batch(gpu, fmt, [400, 33, 0, 90])
    got = x.decode(scale=scale, out_dtype=dtype)
    assert got.dtype == dtype
    x.check(got, scale)


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("std", [0.2, 8.0, 60.0])
def test_peaked_and_flat_rows(gpu, fmt, std):
    x = Batch(gpu, fmt, [900, 64, 3000], std=std, seed=int(std))
    x.check(x.decode())


def _constants(x):
    """Every position's values one vector (which the format holds exactly): a mean of equal values is that value."""
    c = torch.tensor([1.5, 1.0, 4.0, -1.5, -3.0, 2.0, 6.0, -0.5], dtype=BF, device=x.dev).repeat(x.w // 8)
    rows = (c * torch.tensor([2.0 ** 9, 2.0 ** -30], device=x.dev).repeat(x.nkv)[:x.nkv, None].to(BF))
    x.v, x.vrows = _store(rows[None, :, None].expand(x.vrows.shape).contiguous(), "v", x.layout)
    assert torch.equal(x.vrows[0, :, 0], rows)
    return rows


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("std", [0.5, 3.0, 20.0])
def test_equal_values_come_back_exactly(gpu, fmt, std):
    """What divides is the sum of the rounded probabilities that multiplied: n keys' fp32 sums, off by (n + 64) 2^-23 together, stay
    within the 2^-9 to the nearest rounding border (n = 2000: 2^-12)."""
    x = Batch(gpu, fmt, [1, 70, 300, 1000, 2000], std=std, seed=3)
    rows = _constants(x)
    assert torch.equal(x.decode()[0], rows.repeat_interleave(4, 0).expand(5, -1, -1))


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
def test_nan_reaches_the_rows_that_see_it(gpu, fmt):
    x = Batch(gpu, fmt, [200, 90, 64], 8, 2, garbage=0.0)
    clean = x.decode()
    bad = x.krows.clone()
    bad[int(x.table[0, 3]), 1, 5, 9] = math.nan
    x.k = _store(bad, "k", fmt)[0]
    got = x.decode()
    hit = torch.zeros_like(clean, dtype=torch.bool)
    hit[0, 0, 4:] = True
    assert got[hit].isnan().all() and torch.equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
def test_page_ids_outside_the_pool_stay_inside_it(gpu, fmt):
    x = Batch(gpu, fmt, [64], garbage=0.0)
    n = x.krows.shape[0]
    run = lambda t: fused.flash_decode(x.q, x.k, x.v, x.pos, page_table_tensor=_ints([t], gpu))
    assert torch.equal(run([-7, n + 1000]), run([0, n - 1]))


def test_offsets_past_32_bits(gpu):
    n = 140_000
    k, v = (MXCache(torch.empty(n, 8, 1, MXCache.block_bytes("fp8", HD), dtype=torch.uint8, device=gpu), r, "fp8", HD) for r in "kv")
    assert k.data.numel() > 2 ** 32
    g = torch.Generator().manual_seed(8)
    ks, vs = (MXCache.from_rows(torch.randn(3, 8, 32, HD, generator=g).to(gpu, BF), r, "fp8") for r in "kv")
    ids = [n - 1, 3, n - 2]
    k.data[ids], v.data[ids] = ks.data, vs.data
    q = torch.randn(1, 2, 8, HD, generator=g).to(gpu, BF)
    pos = _ints([70, 95], gpu)
    exp = fused.flash_decode(q, ks, vs, pos, page_table_tensor=_ints([[0, 1, 2]] * 2, gpu))
    assert torch.equal(fused.flash_decode(q, k, v, pos, page_table_tensor=_ints([ids] * 2, gpu)), exp)
    kw = dict(shared_len=_ints([64], gpu))
    assert torch.equal(fused.flash_decode_shared(q, k, v, pos, _ints([ids] * 2, gpu), **kw),
                       fused.flash_decode_shared(q, ks, vs, pos, _ints([[0, 1, 2]] * 2, gpu), **kw))


# ---- shared prefixes -----------------------------------------------------------------------------

_GROUPS = [
    ([1], [0], [5]),                                            # one row
    ([3], [100], [101, 130, 97]),                               # one that sees all of the shared blocks, ones behind them
    ([3], [100], [96, 95, 1]),                                  # nothing behind them; rows that end inside them
    ([4, 1, 2], [64, 500, 40], [70, 64, 200, 65, 510, 41, 33]),
    ([2, 3], [2000, 31], [2001, 2400, 32, 1, 60]),
    ([5], [-4], [1, 2, 3, 0, 33]),                              # nothing shared, an empty row
    ([2, 2], [5000, 320], [5100, 0, 320, 330]),
    ([6], [10000], [300] * 6),                                  # longer than the table
    ([3, 0, 2], [64, 64, 64], [70, 71, 72, 73, 74])]            # an empty group


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("groups,shared,lens", _GROUPS, ids=str)
@pytest.mark.parametrize("nq,nkv", [(8, 2), (6, 2), (7, 1), (16, 1), (4, 4)])
def test_groups(gpu, layout, groups, shared, lens, nq, nkv):
    x = Batch(gpu, layout, lens, nq, nkv, groups=groups, shared=shared, seed=sum(lens), page=64 if sum(lens) % 2 else 32)
    x.check(x.decode_shared())
    x.check(x.decode_shared(wide=False))                                 # little enough for a launch without the prefixes'


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("B,groups,prefix,tail,nq,nkv", [
    (64, 1, 3000, 60, 32, 8), (40, 1, 1000, 300, 7, 1), (33, 3, 700, 40, 12, 4), (96, 16, 400, 50, 16, 4), (200, 100, 96, 40, 4, 2),
    (9, 1, 9000, 10, 16, 1), (300, 2, 200, 33, 3, 1)])
def test_batches(gpu, layout, B, groups, prefix, tail, nq, nkv):
    """Column tiles of 16, 32 and 64 queries, rows that straddle two of them, prefixes cut into many pieces and not at all."""
    g = torch.Generator().manual_seed(B)
    cuts = sorted(torch.randperm(B - 1, generator=g)[:groups - 1].add(1).tolist())
    rows = [b - a for a, b in zip([0] + cuts, cuts + [B])]
    shared = [prefix] + torch.randint(1, prefix + 1, (groups - 1,), generator=g).tolist()
    lens = [s + int(torch.randint(0, tail, (), generator=g)) for n, s in zip(rows, shared) for _ in range(n)]
    x = Batch(gpu, layout, lens, nq, nkv, 64 if B % 2 else 128, 64, rows, shared, seed=B, garbage=0.0)
    x.check(x.decode_shared(), rows=list(range(0, B, max(1, B // 24))) + [B - 1])


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("rows", [[4, 1, 1], [1, 3, 1, 1, 1], [2, 1], [1, 2, 1, 1], [1, 1, 1], [1]], ids=str)
def test_lone_rows_beside_groups(gpu, layout, rows):
    """Rows that are a group of their own: few enough that they are read with the larger groups, too many for that, only such."""
    shared = [900 if n == 1 else 700 for n in rows]
    lens = [s + 13 * i for i, (n, s) in enumerate(zip(rows, shared)) for _ in range(n)]
    x = Batch(gpu, layout, lens, 8, 2, 64, 64, rows, shared, seed=len(lens))
    x.check(x.decode_shared())
    x.check(x.decode_shared(wide=False))


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("B,groups,prefix,tail,nq,nkv", [(150, 1, 700, 60, 16, 4), (180, 60, 300, 300, 9, 3), (270, 9, 96, 500, 20, 5)])
def test_many_items_behind_prefixes(gpu, layout, B, groups, prefix, tail, nq, nkv):
    g = torch.Generator().manual_seed(B)
    cuts = sorted(torch.randperm(B - 1, generator=g)[:groups - 1].add(1).tolist())
    rows = [b - a for a, b in zip([0] + cuts, cuts + [B])]
    shared = [prefix] + torch.randint(1, prefix + 1, (groups - 1,), generator=g).tolist()
    lens = [s + int(torch.randint(0, tail, (), generator=g)) for n, s in zip(rows, shared) for _ in range(n)]
    x = Batch(gpu, layout, lens, nq, nkv, 48 if layout in ("rows", "tiled") else 64, 64, rows, shared, seed=B, garbage=0.0)
    x.check(x.decode_shared(), rows=list(range(0, B, 7)) + [B - 1])
    x.check(x.decode_shared(wide=False), rows=list(range(0, B, 7)) + [B - 1])


@pytest.mark.parametrize("layout", ["rows", "tiled"])
@pytest.mark.parametrize("w", [16, 32, 48, 80, 96, 112, 128])
def test_shared_widths_bf16(gpu, layout, w):
    x = Batch(gpu, layout, [330, 300, 299, 70, 66], 8, 2, w, groups=[3, 2], shared=[290, 64], seed=w)
    x.check(x.decode_shared())


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("w", [32, 96, 128])
def test_shared_widths_quantised(gpu, fmt, w):
    x = Batch(gpu, fmt, [330, 300, 299, 70, 66], 8, 2, w, page=128, groups=[3, 2], shared=[290, 64], seed=w)
    x.check(x.decode_shared())


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_shared_scales_and_output_types(gpu, layout, scale, dtype):
    x = Batch(gpu, layout, [200, 170, 161], groups=[3], shared=[160])
    got = x.decode_shared(scale=scale, out_dtype=dtype)
    assert got.dtype == dtype
    x.check(got, scale)


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("std", [0.5, 3.0, 20.0])
def test_shared_equal_values_come_back_exactly(gpu, layout, std):
    x = Batch(gpu, layout, [1000, 1400, 64, 2000, 1], groups=[3, 2], shared=[990, 640], std=std, seed=3)
    rows = _constants(x)
    assert torch.equal(x.decode_shared()[0], rows.repeat_interleave(4, 0).expand(5, -1, -1))


@pytest.mark.parametrize("layout", LAYOUTS)
def test_shared_without_groups_and_rows_of_no_group(gpu, layout):
    x = Batch(gpu, layout, [100, 70, 65, 90], groups=[4], shared=[64])
    got = x.decode_shared(wide=False)
    assert torch.equal(got, fused.flash_decode_shared(x.q, x.k, x.v, x.pos, x.own.to(gpu), x.shared))   # no cu_groups: one group
    cu, x.cu = x.cu, None
    ahead, x.cu = x.decode_shared(), cu
    assert torch.equal(x.decode_shared(), ahead)
    y = Batch(gpu, layout, [100, 70, 65, 90], groups=[1, 2], shared=[64, 64])     # groups of rows 1 and 2; row 0 alone, row 3 of none
    y.cu, y.shared = _ints([1, 3], gpu), _ints([64], gpu)
    y.lead, y.blocks, y.own = [0, 1, 1, 3], [0, 2, 2, 0], y.table.clone()
    y.check(y.decode_shared())
    y.check(y.decode_shared(wide=False))


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("wide", [True, False])
def test_shared_nan_reaches_the_rows_that_see_it(gpu, layout, wide):
    """One inside the prefix, which a row of the group that ends before it does not see; one behind it."""
    x = Batch(gpu, layout, [200, 90, 180, 100], 8, 2, groups=[3, 1], shared=[160, 0], garbage=0.0)
    clean = x.decode_shared(wide)
    for page, row, rows in ((3, 0, (0, 2)), (5, 2, (2,))):
        bad = x.krows.clone()
        bad[int(x.table[row, page]), 1, 5, 9] = math.nan
        k, x.k = x.k, _store(bad, "k", layout)[0]
        got, x.k = x.decode_shared(wide), k
        hit = torch.zeros_like(clean, dtype=torch.bool)
        hit[0, list(rows), 4:] = True
        assert got[hit].isnan().all() and torch.equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("layout", LAYOUTS)
def test_offsets_that_make_no_sense_stay_inside(gpu, layout):
    """Groups that overlap, fall back, or lie outside the batch: what comes out is not defined, what lies around the output and
    the workspace keeps what it holds."""
    B, n = 24, 40
    x = Batch(gpu, layout, [300] * B, 16, 1, garbage=0.0)
    g = torch.Generator().manual_seed(1)
    wide = torch.nn.functional.pad(x.table, (0, 65536 // x.page - x.table.shape[1]), value=-1)
    for cu, table in [(cu, table) for table in (wide, x.table) for cu in
                      ([0, B] * (n // 2) + [0], torch.randint(-100, 200, (n + 1,), generator=g).tolist(), [2 ** 31 - 1] * n + [-2 ** 31],
                       [B] * n + [0])]:
        need = _native.load().palu_flash_decode_shared_workspace_bytes(B, n, 16, 1, 64)
        ws, out = torch.full((need + 8192,), 77, dtype=torch.uint8, device=gpu), torch.full((1, B + 2, 16, 64), 7.0, dtype=BF, device=gpu)
        fused.flash_decode_shared(x.q, x.k, x.v, x.pos, table.to(gpu), _ints([2 ** 31 - 1, 300, -2 ** 31, 64] * (n // 4), gpu), _ints(cu, gpu),
                                  out=out[:, 1:-1], workspace=ws[4096:4096 + need])
        assert (ws[:4096] == 77).all() and (ws[4096 + need:] == 77).all() and (out[0, 0] == 7).all() and (out[0, -1] == 7).all()
    x.check(x.decode())                                                  # and nothing is left behind


# ---- both: repeated, on streams, captured --------------------------------------------------------

def _both(gpu, layout):
    x = Batch(gpu, layout, [3000, 3100, 40, 700, 690, 2999], 16, 2, 64, 64, [2, 1, 2, 1], [2900, 32, 640, 0], garbage=0.0)
    calls = [x.decode_shared] + ([x.decode] if layout in ("fp8", "fp4") else [])
    return x, calls


@pytest.mark.parametrize("layout", LAYOUTS)
def test_streams_and_graph_replays(gpu, layout):
    """Repeated calls are bit-identical, on two streams at once and captured: replays with new queries, positions and prefixes
    between eager calls of the same shapes."""
    x, calls = _both(gpu, layout)
    for call in calls:
        alone = call()
        streams, outs = [torch.cuda.Stream() for _ in range(2)], [[], []]
        torch.cuda.synchronize()
        for _ in range(10):
            for s, o in zip(streams, outs):
                with torch.cuda.stream(s):
                    o.append(call())
        torch.cuda.synchronize()
        assert all(torch.equal(o, alone) for os in outs for o in os)
        own, table = x.own, x.table
        x.own, x.table = own.to(gpu), table.to(gpu)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = call()
        g = torch.Generator().manual_seed(5)
        pos, shared = x.pos.clone(), x.shared.clone()
        for i in range(4):
            x.q.copy_(torch.randn(x.q.shape, generator=g))
            x.pos.sub_(i * 7).clamp_(min=0)
            x.shared.sub_(32 * i)
            graph.replay()
            exp = call()
            torch.cuda.synchronize()
            assert torch.equal(y, exp)
        x.pos.copy_(pos)
        x.shared.copy_(shared)
        x.own, x.table = own, table


@pytest.mark.parametrize("layout", LAYOUTS)
def test_two_graphs_share_a_workspace(gpu, layout):
    """Two captured calls over one workspace, replayed in turn and with an eager call between them, whatever it holds."""
    x, calls = _both(gpu, layout)
    f = _native.load()
    need = max(f.palu_flash_decode_shared_workspace_bytes(6, 4, 16, 2, 64), f.palu_mx_decode_workspace_bytes(6, 16, 2, 64))
    ws = torch.full((need,), 255, dtype=torch.uint8, device=gpu)
    x.own, x.table = x.own.to(gpu), x.table.to(gpu)
    exp = [c() for c in calls + calls[:1]]
    graphs = []
    for c in calls + calls[:1]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = c(workspace=ws)
        graphs.append((graph, y))
    for fill in (255, 0, 37):
        for i in range(3):
            for (graph, y), e, c in zip(graphs, exp, calls + calls[:1]):
                graph.replay()
                z = c(workspace=ws)
                torch.cuda.synchronize()
                assert torch.equal(y, e) and torch.equal(z, e)
        ws.fill_(fill)


def test_empty_batches(gpu):
    x = Batch(gpu, "fp8", [40, 3])
    for call in (lambda q, pos, t: fused.flash_decode_shared(q, x.k, x.v, pos, t, _ints([32], gpu)),):
        assert call(x.q[:, :0].contiguous(), x.pos[:0], x.table[:0].to(gpu)).shape == (1, 0, 8, 64)
