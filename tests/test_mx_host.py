"""The 8- and 4-bit cache formats on the CPU (values, rounding, scales, byte order) and the refusals of the ops over them: the
C-ABI checks its arguments before any launch, the Python layer before any call."""
import ctypes
import math

import pytest
import torch

from palu_tt import _build, _native, cache, decoder_ops, fused
from palu_tt.cache import LatentCache, MXCache
from palu_tt.pages import PagePools

BF = torch.bfloat16
P = 4096                                                     # a 16-byte aligned address that no refused call reads


@pytest.fixture(scope="module")
def lib():
    if not _build.library_path().exists():
        _build.build_native()
    return _native.load()


def _refused(lib, rc, code, what):
    assert rc == code and what in lib.palu_last_error().decode(), (rc, lib.palu_last_error().decode())


# ---- the formats --------------------------------------------------------------------------------

def test_values_of_the_codes():
    assert cache.mx_values("fp4").tolist() == [0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6]
    v = cache.mx_values("fp8")
    ref = torch.arange(256, dtype=torch.int32).to(torch.uint8).view(torch.float8_e4m3fn).float()
    assert torch.equal(v.nan_to_num(1e9), ref.nan_to_num(1e9)) and v[126] == 448 and v[127].isnan() and v[255].isnan()


def _grid(fmt):
    return [0.0, .5, 1, 1.5, 2, 3, 4, 6] if fmt == "fp4" else cache.mx_values("fp8")[:127].tolist()


def _nearest(x, fmt):
    """One block of 32 finite values by the definition, in 64 bits: (values, scale exponent)."""
    grid, held = _grid(fmt), 7.0 if fmt == "fp4" else 464.0
    x = [max(-1.75 * 2.0 ** 127, min(1.75 * 2.0 ** 127, v)) for v in x]
    e = -117
    while max(abs(v) for v in x) > held * 2.0 ** e:
        e += 1
    out = []
    for v in x:
        y = abs(v) / 2.0 ** e
        best = min(range(len(grid)), key=lambda i: (abs(grid[i] - y), i % 2))
        out.append(math.copysign(grid[best] * 2.0 ** e, v))
    return out, e


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("what", ["normal", "wide", "tiny", "huge", "ties", "zeros"])
def test_quantise_is_the_nearest_over_the_smallest_scale(fmt, what):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(12, 32, generator=g)
    if what == "wide":
        x = x * 2.0 ** (torch.randn(12, 32, generator=g) * 6)
    elif what == "tiny":
        x = x * 2.0 ** torch.randint(-133, -105, (12, 1), generator=g).float()
    elif what == "huge":
        x = (x * 2.0 ** 126).clamp(-3.38e38, 3.38e38)
    elif what == "ties":                                     # halfway between two elements, at and past the borders of the scale
        v = torch.tensor(_grid(fmt))
        mid = (v[1:] + v[:-1]) / 2
        x = torch.cat([mid, mid[-1:] + 1, v[-1:] * 1.04, torch.tensor([464.0, 466, 7, 7.03])])
        x = x[torch.randint(0, x.numel(), (12, 32), generator=g)] * 2.0 ** torch.randint(-3, 4, (12, 1), generator=g).float()
    elif what == "zeros":
        x = torch.zeros(12, 32)
        x[1::2, 7] = torch.tensor([1.0, -1e-30, 2.0 ** -126, -3e38, 5e-41, 448.0])
    x = x.to(BF)
    codes, scales = cache.mx_quantize(x, fmt)
    got = cache.mx_dequantize(codes, scales, fmt)
    for row, c, s in zip(x.tolist(), got.tolist(), scales[:, 0].tolist()):
        exp, e = _nearest(row, fmt)
        assert c == exp and s == e + 127 and all(map(math.isfinite, c))
    # the documented error: half a step of the element, relative to the value in its normal range
    xf, s = x.double().clamp(-1.75 * 2.0 ** 127, 1.75 * 2.0 ** 127), 2.0 ** (scales.double() - 127)
    rel, least = (2.0 ** -4, 2.0 ** -10) if fmt == "fp8" else (0.25, 0.25)
    assert ((got.double() - xf).abs() <= torch.maximum(rel * xf.abs(), least * s)).all()


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
def test_blocks_that_are_not_finite(fmt):
    x = torch.ones(4, 96, dtype=BF)
    x[0, 40], x[1, 64], x[2, 95] = math.inf, math.nan, -math.inf
    codes, scales = cache.mx_quantize(x, fmt)
    got = cache.mx_dequantize(codes, scales, fmt)
    bad = torch.zeros(4, 96, dtype=torch.bool)
    bad[0, 32:64] = bad[1, 64:] = bad[2, 64:] = True
    assert torch.equal(got.isnan(), bad) and (got[~bad] == 1).all() and (codes[bad] == 0).all()


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("role", ["k", "v"])
@pytest.mark.parametrize("w", [32, 96, 128, 512])
def test_byte_order(fmt, role, w):
    """Every element and scale where the C header says it lies."""
    g = torch.Generator().manual_seed(w)
    rows = (torch.randn(2, 3, 64, w, generator=g) * 4).to(BF)
    c = MXCache.from_rows(rows, role, fmt)
    codes, scales = cache.mx_quantize(rows, fmt)
    assert c.shape == (2, 3, 64, w) and c.nbytes() == 2 * 3 * 2 * (33 if fmt == "fp8" else 17) * w
    assert torch.equal(c.to_rows(), cache.mx_dequantize(codes, scales, fmt))
    nb, size = w // 32, (32 if fmt == "fp8" else 16) * w
    for _ in range(200):
        b, gr, p, x = (int(torch.randint(0, n, (), generator=g)) for n in (2, 3, 64, w))
        blk, q = c.data[b, gr, p // 32], p % 32
        if role == "k":
            n, half, gg = 4 * (q // 8) + q % 4, q // 4 % 2, x // 32
            at = ((half * 2 + x // 16 % 2) * nb + gg) * 256 + n * 16 + x % 16 if fmt == "fp8" else \
                (half * nb + gg) * 256 + n * 16 + x % 32 // 2
            s = size + (gg * 16 + n) * 2 + half
        else:
            o, j, bb, m = q // 8, q % 8, x // 32, x % 32 // 2
            at = ((bb * 4 + o) * 16 + m) * 8 + j
            at = at * 2 + x % 2 if fmt == "fp8" else at
            s = size + bb * 32 + q
        got = int(blk[at])
        if fmt == "fp4":
            got = got >> 4 if x % 2 else got & 15
        assert got == int(codes[b, gr, p, x]) and int(blk[s]) == int(scales[b, gr, p, x // 32])


def test_cache_objects():
    z = MXCache.zeros(2, 3, 64, 96, "cpu", "v", "fp4")
    assert z.shape == (2, 3, 64, 96) and (z.to_rows() == 0).all()
    data = torch.zeros(2, 3, 2, 33 * 64, dtype=torch.uint8)
    MXCache(data, "k", "fp8", 64)
    for args in [(data, "q", "fp8", 64), (data, "k", "int4", 64), (data, "k", "fp8", 48), (data, "k", "fp4", 64), (data, "k", "fp8", 32),
                 (data.to(torch.int8), "k", "fp8", 64), (data[0], "k", "fp8", 64)]:
        with pytest.raises(AssertionError):
            MXCache(*args)
    with pytest.raises(AssertionError):
        MXCache.zeros(1, 1, 40, 64, "cpu")


# ---- the C-ABI -----------------------------------------------------------------------------------

E, U = _native.PALU_EINVAL, _native.PALU_EUNSUPPORTED


@pytest.mark.parametrize("layout", [4, 5, 6, 7])
@pytest.mark.parametrize("kw,code,what", [
    (dict(width=48), E, "multiple of 32"), (dict(width=544), E, "up to 512"), (dict(rows=None), E, "null"), (dict(cu=None), E, "null"),
    (dict(pt=None), E, "page_table"), (dict(page=16), E, "power of two"), (dict(st=4), E, "strides"), (dict(cache=P + 8), E, "16-byte"),
    (dict(n=0), E, "positive")])
def test_fill_refusals(lib, layout, kw, code, what):
    a = dict(cache=P, rows=P, st=128, sg=64, cu=P, start=None, pt=P, n=5, batch=1, groups=2, pages=9, page=64, slots=4, width=64,
             layout=layout, stream=None)
    a.update(kw)
    _refused(lib, lib.palu_latent_fill_paged(*a.values()), code, what)


@pytest.mark.parametrize("kw,code,what", [
    (dict(width=40), E, "multiple of 32"), (dict(width=40, layout=1), E, "multiple of 16"), (dict(width=20, layout=0), E, "multiple of 8"),
    (dict(layout=8), E, "cache layout"), (dict(layout=3), E, "cache layout"), (dict(out=None), E, "null"), (dict(cache=None), E, "null"),
    (dict(out=P + 8), E, "16-byte"), (dict(n=0), E, "positive"), (dict(batch=0), E, "positive"), (dict(batch=70000), U, "grid"),
    (dict(slots=2048), U, "65536"), (dict(pages=0), E, "num_pages")])
def test_read_refusals(lib, kw, code, what):
    a = dict(cache=P, out=P, cu=P, start=None, pt=P, n=5, batch=1, groups=2, pages=9, page=64, slots=4, width=64, layout=4, stream=None)
    a.update(kw)
    _refused(lib, lib.palu_latent_read_paged(*a.values()), code, what)


@pytest.mark.parametrize("layout", [4, 7])
@pytest.mark.parametrize("kw,code,what", [
    (dict(width=48), E, "multiple of 32"), (dict(S=40), E, "32-position"), (dict(rows=None), E, "null"), (dict(batch=0), E, "positive"),
    (dict(cache=P + 4), E, "16-byte")])
def test_append_refusals(lib, layout, kw, code, what):
    a = dict(cache=P, rows=P, idx=P, batch=2, groups=2, S=64, width=64, layout=layout, stream=None)
    a.update(kw)
    _refused(lib, lib.palu_latent_append(*a.values()), code, what)


def test_bf16_only_ops_refuse_the_layouts(lib):
    """Entry points that read or write bf16 caches alone."""
    _refused(lib, lib.palu_latent_append_strided(P, P, 64, 64, P, 1, 1, 64, 64, 4, None), E, "cache layout")
    _refused(lib, lib.palu_flash_prefill_paged(P, 1024, 128, P, P, P, None, P, P, 0.1, 5, 1, 8, 2, 9, 64, 4, 64, 4, None, 0, None), E,
             "cache layout")
    _refused(lib, lib.palu_latent_fill(P, 0, 0, P, 64, 64, 1, 1, 1, 32, 64, 4, None, None, 0, None), E, "layout")
    _refused(lib, lib.palu_naive_decode(P, P, P, P, P, 64, P, P, P, 0.1, 1, 4, 1, 64, 64, 32, 32, 1, 4, 0, P, 1 << 30, None), E, "layout")


@pytest.mark.parametrize("kw,code,what", [
    (dict(q=None), E, "null"), (dict(cur=None), E, "null"), (dict(batch=0), E, "positive"), (dict(n_q=7), E, "KV head count"),
    (dict(n_q=34), E, "KV head count"), (dict(dv=48), U, "head_dim_v"), (dict(dv=160), U, "head_dim_v"), (dict(dtype=3), E, "dtype"),
    (dict(S=48), E, "32-position"), (dict(S=1 << 17), U, "65536"), (dict(layout=5), E, "cache layout"), (dict(v=P + 8), E, "16-byte"),
    (dict(batch=40000), U, "grid"), (dict(ws=None), E, "workspace"), (dict(ws=P + 8), E, "workspace"), (dict(bytes=100), E, "workspace")])
def test_decode_refusals(lib, kw, code, what):
    a = dict(q=P, k=P, v=P, cur=P, out=P, scale=0.1, batch=3, n_q=8, n_kv=2, S=64, dv=64, dtype=1, layout=4, det=0, ws=P, bytes=1 << 30,
             stream=None)
    a.update(kw)
    _refused(lib, lib.palu_flash_decode(*a.values()), code, what)


@pytest.mark.parametrize("kw,code,what", [
    (dict(pt=None), E, "page_table"), (dict(page=48), E, "power of two"), (dict(slots=2048), U, "65536"), (dict(shared=None), E, "null"),
    (dict(cu=None, groups=2), E, "one without"), (dict(groups=0), E, "groups"), (dict(batch=5000, n_kv=1, n_q=1), U, "4096"),
    (dict(n_q=34), E, "KV head count"), (dict(dv=40), U, "head_dim_v"), (dict(dv=48, layout=4), U, "head_dim_v"),
    (dict(layout=2), E, "cache layout"), (dict(layout=3), E, "cache layout"), (dict(k=P + 2), E, "16-byte"), (dict(out=None), E, "null"),
    (dict(dtype=2), E, "dtype"), (dict(ws=None), E, "workspace"), (dict(bytes=4096), E, "workspace"), (dict(ws=P + 4), E, "workspace")])
def test_shared_refusals(lib, kw, code, what):
    a = dict(q=P, k=P, v=P, cur=P, pt=P, cu=P, shared=P, out=P, scale=0.1, batch=3, groups=2, n_q=8, n_kv=2, pages=9, page=64, slots=4,
             dv=64, dtype=1, layout=0, ws=P, bytes=1 << 30, stream=None)
    a.update(kw)
    _refused(lib, lib.palu_flash_decode_shared(*a.values()), code, what)


def test_workspaces(lib):
    """Per part of a split item its query heads' results and statistics and a flag; the prefixes' pieces behind them."""
    f, s = lib.palu_mx_decode_workspace_bytes, lib.palu_flash_decode_shared_workspace_bytes
    assert f(0, 8, 2, 64) == f(1, 7, 2, 64) == f(1, 34, 2, 64) == f(1, 8, 2, 40) == f(40000, 8, 2, 64) == 0
    assert f(1, 8, 2, 64) == 514 * (4 * 66 * 4 + 8) and f(1000, 8, 2, 128) == 2512 * (4 * 130 * 4 + 8)
    assert s(4, 0, 8, 2, 64) == 0 and s(4, 1, 8, 2, 64) > f(4, 8, 2, 64)
    assert all(s(b, g, 32, 8, 128) > 0 for b in (1, 64, 4096) for g in (1, 7, 4096))


# ---- the Python layer, with the launch taken down: tensors that say they are on the GPU ------------------------------

class _OnGpu(torch.Tensor):
    is_cuda = property(lambda self: True)


def _t(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_OnGpu)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32)


def _mx(n=4, G=2, page=32, w=64, role="k", fmt="fp8"):
    return MXCache(_t(n, G, page // 32, MXCache.block_bytes(fmt, w), dtype=torch.uint8), role, fmt, w)


@pytest.fixture
def launches(lib, monkeypatch):
    calls = []
    monkeypatch.setattr(_native, "launch", lambda name, device, *args: calls.append((name, args)))
    return calls


def test_layouts_that_reach_the_library(launches):
    cu, table, pos = _ints([0, 3]), _ints([[0, 1]]), _ints([5])
    for fmt, base in (("fp8", 4), ("fp4", 6)):
        for role, layout in (("k", base), ("v", base + 1)):
            c = _mx(role=role, fmt=fmt)
            fused.paged_fill_cache(c, _t(3, 2, 64), cu, table)
            fused.paged_read_cache(c, 3, cu, table)
            fused.paged_update_cache(c, _t(1, 2, 64), pos, page_table=table)
            fused.paged_update_cache(_mx(n=1, role=role, fmt=fmt), _t(1, 2, 64), pos)
            assert [a[-1] for _, a in launches[-4:]] == [layout] * 4
        k, v = _mx(w=128, fmt=fmt), _mx(role="v", fmt=fmt)
        fused.flash_decode(_t(1, 1, 4, 128), k, v, pos, page_table_tensor=table)
        fused.flash_decode(_t(1, 4, 4, 128), k, v, _ints([1, 2, 3, 4]))
        fused.flash_decode_shared(_t(1, 1, 4, 128), k, v, pos, table, _ints([32]))
        assert [(n, a[i]) for (n, a), i in zip(launches[-3:], (15, 12, 18))] == [
            ("flash_decode_paged", base), ("flash_decode", base), ("flash_decode_shared", base)]


def test_wrong_orders_and_mixtures(launches):
    q, pos, table = _t(1, 1, 4, 128), _ints([5]), _ints([[0, 1]])
    k8, v8, v4 = _mx(w=128), _mx(role="v"), _mx(role="v", fmt="fp4")
    for fn in (lambda k, v: fused.flash_decode(q, k, v, pos, page_table_tensor=table),
               lambda k, v: fused.flash_decode_shared(q, k, v, pos, table, _ints([3]))):
        for k, v, what in [(k8, v4, "same cache layout"), (k8, _t(4, 2, 32, 64), "same cache layout"), (_mx(w=128, role="v"), v8, "order"),
                           (k8, _mx(), "order"), (_mx(w=64), v8, "k must be"), (k8, _mx(n=3, role="v"), "does not match")]:
            with pytest.raises(RuntimeError, match=what):
                fn(k, v)
    assert not launches


def test_ops_of_bf16_caches_refuse_quantised_ones(launches):
    k, v = _mx(w=128), _mx(role="v")
    q, pos, cu, table = _t(1, 4, 4, 128), _ints([0] * 4), _ints([0, 4]), _ints([[0, 1]])
    for call in [lambda: fused.flash_prefill(_t(4, 4, 128), k, v, cu, page_table_tensor=table),
                 lambda: fused.palu_sdpa_decode(q, k, _t(1, 2, 128, 256), _t(1, 1, 64, 256), v, 64, pos),
                 lambda: fused.naive_decode(q, k, _t(2, 128, 128), _t(64, 128), _t(64, 128), v, pos, 32),
                 lambda: decoder_ops.append_from(k, _t(4, 512), 128, 128, pos),
                 lambda: decoder_ops.fill_from(k, 0, _t(4, 512), 1, 4, 0, 128),
                 lambda: decoder_ops.qkv_post(_t(1, 4, 1024, dtype=torch.float32), pos, _t(64, 128, dtype=torch.float32),
                                              _t(64, 128, dtype=torch.float32), 4, k, 512, 128, 128, v, 768, 64, 64)]:
        with pytest.raises(RuntimeError, match="MXCache"):
            call()
    assert not launches


def test_storage_that_was_replaced_is_looked_at(launches):
    """A cache's data may be another tensor than at its start; blocks of another size would be read past their end."""
    cu, table, pos, q = _ints([0, 3]), _ints([[0, 1]]), _ints([5]), _t(1, 1, 4, 128)
    for other in (_mx(w=32), _mx(fmt="fp4")):
        c, v = _mx(), _mx(role="v")
        c.data = v.data = other.data
        for call in [lambda: fused.paged_fill_cache(c, _t(3, 2, 64), cu, table), lambda: fused.paged_read_cache(c, 3, cu, table),
                     lambda: fused.paged_update_cache(c, _t(1, 2, 64), pos, page_table=table),
                     lambda: fused.flash_decode(q, _mx(w=128), v, pos, page_table_tensor=table)]:
            with pytest.raises(RuntimeError, match="blocks of"):
                call()
    assert not launches


def test_page_pools_take_quantised_pools(launches):
    k, v, rows = _mx(n=5, w=128), _mx(n=5, role="v", fmt="fp4"), _t(5, 2, 32, 32)
    PagePools([k, v, rows]).compact(_ints([[0, 1]]), _ints([3]))
    ptrs, sizes, n = launches[0][1][4:7]
    assert list(zip(list(ptrs), list(sizes)))[:n] == [(k.data.data_ptr(), 2 * 33 * 128), (v.data.data_ptr(), 2 * 17 * 64),
                                                      (rows.data_ptr(), 2 * 32 * 32 * 2)]
    with pytest.raises(RuntimeError, match="agree"):
        PagePools([k, _mx(n=4, role="v")])
    with pytest.raises(RuntimeError, match="bf16"):
        PagePools([k, k.data.unflatten(-1, (-1, 1))[..., 0]])              # bytes without the object that says what they are


def test_read_arguments(launches):
    cu, table = _ints([0, 3]), _ints([[0, 1]])
    assert fused.paged_read_cache(_t(4, 2, 32, 40), 0, cu, table).shape == (0, 2, 40) and not launches
    fused.paged_read_cache(LatentCache(_t(4, 2, 1, 4, 64, 8), "v"), 3, cu, table, start_pos=_ints([7]))
    assert launches.pop()[1][-1] == _native.LAYOUT_TILED_V
    out = _t(3, 2, 64)
    assert fused.paged_read_cache(_mx(), 3, cu, table, out=out) is out
    c = _mx()
    over = c.data.view(-1)[:3 * 2 * 64 * 2].view(BF).view(3, 2, 64)
    for kw, what in [(dict(out=_t(3, 2, 32)), "out must be"), (dict(out=_t(3, 2, 64, dtype=torch.float32)), "bfloat16"),
                     (dict(out=over), "memory of its own"), (dict(n_rows=-1), "negative"), (dict(cu_seqlens=_ints([0])), "at least one"),
                     (dict(page_table=_ints([[0], [1]])), "rows for batch"), (dict(start_pos=_ints([0, 1])), "start_pos"),
                     (dict(cache=torch.zeros(4, 2, 32, 64, dtype=BF)), "GPU"), (dict(cache=[1]), "must be"),
                     (dict(cache=_t(4, 2, 32, 64, dtype=torch.float16)), "bfloat16")]:
        a = dict(cache=c, n_rows=3, cu_seqlens=cu, page_table=table)
        a.update(kw)
        with pytest.raises(RuntimeError, match=what):
            fused.paged_read_cache(**a)
    assert len(launches) == 1


def test_decode_arguments(launches, lib):
    q, pos, table = _t(1, 2, 4, 128), _ints([5, 6]), _ints([[0, 1], [2, 3]])
    k, v = _mx(w=128), _mx(role="v")
    run = {"decode": lambda **kw: fused.flash_decode(q, k, v, pos, page_table_tensor=table, **kw),
           "shared": lambda **kw: fused.flash_decode_shared(q, k, v, pos, table, _ints([32]), **kw)}
    need = {"decode": lib.palu_mx_decode_workspace_bytes(2, 4, 2, 64), "shared": lib.palu_flash_decode_shared_workspace_bytes(2, 1, 4, 2, 64)}
    for name, call in run.items():
        ws = torch.zeros(need[name], dtype=torch.uint8)
        out = _t(1, 2, 4, 64)
        assert call(out=out, workspace=ws) is out
        assert call(out_dtype=torch.float32).dtype == torch.float32
        over = lambda t: t.view(-1).view(torch.uint8)[:2 * 2 * 4 * 64].view(BF).view(1, 2, 4, 64).as_subclass(_OnGpu)
        for kw, what in [(dict(out=_t(1, 2, 4, 32)), "out must be"), (dict(out=out.float()), "bfloat16"), (dict(out_dtype=torch.float16), "out_dtype"),
                         (dict(out=over(q)), "memory of its own"), (dict(out=over(v.data)), "memory of its own"),
                         (dict(out=over(ws), workspace=ws), "memory of its own"), (dict(workspace=ws[1:]), "workspace"),
                         (dict(workspace=ws.expand(2, -1)[:, ::2]), "workspace"), (dict(head_dim_v=32), "head_dim_v")]:
            with pytest.raises(RuntimeError, match=what):
                call(**kw)
    for kw, what in [(dict(cu_groups=_ints([0])), "at least one"), (dict(shared_len=_ints([1, 2])), "shared_len"),
                     (dict(shared_len=torch.zeros(1)), "shared_len"), (dict(page_table_tensor=None), "page_table"),
                     (dict(page_table_tensor=table[:1]), "rows for batch"), (dict(cur_pos_tensor=_ints([1])), "cur_pos")]:
        a = dict(cur_pos_tensor=pos, page_table_tensor=table, shared_len=_ints([32]))
        a.update(kw)
        with pytest.raises(RuntimeError, match=what):
            fused.flash_decode_shared(q, k, v, **a)
    assert len(launches) == 4


def test_derivatives_are_refused(launches):
    import torch.autograd.forward_ad as fw
    cu, table, pos = _ints([0, 3]), _ints([[0, 1]]), _ints([5])
    k, v, rk, rv = _mx(w=128), _mx(role="v"), _t(4, 2, 32, 128), _t(4, 2, 32, 64)
    calls = [lambda x: fused.paged_fill_cache(v, x(_t(3, 2, 64)), cu, table),
             lambda x: fused.paged_update_cache(v, x(_t(1, 2, 64)), pos, page_table=table),
             lambda x: fused.paged_read_cache(x(_t(4, 2, 32, 64)), 3, cu, table),
             lambda x: fused.flash_decode(x(_t(1, 1, 4, 128)), k, v, pos, page_table_tensor=table),
             lambda x: fused.flash_decode_shared(x(_t(1, 1, 4, 128)), rk, rv, pos, table, _ints([3])),
             lambda x: fused.flash_decode_shared(_t(1, 1, 4, 128), x(rk.clone()), rv, pos, table, _ints([3])),
             lambda x: fused.flash_decode_shared(_t(1, 1, 4, 128), rk, x(rv.clone()), pos, table, _ints([3]))]
    for call in calls:
        with pytest.raises(RuntimeError, match="backward"):
            call(lambda t: t.requires_grad_())
        with fw.dual_level():
            with pytest.raises(RuntimeError, match="tangent"):
                call(lambda t: fw.make_dual(t, torch.ones_like(t)))
        assert not launches
        with torch.no_grad():
            call(lambda t: t.requires_grad_())
        assert launches.pop() and not launches
