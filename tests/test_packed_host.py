"""Refusals of the packed-batch entry points (prompts' attention, page fills, page tables, token log probabilities) without a GPU:
the C-ABI checks its arguments before any launch, the Python layer before any call."""
import ctypes

import pytest
import torch

from palu_tt import _build, _native, decoder_ops, fused
from palu_tt.pages import PagePools

P = 4096                                                     # a 16-byte aligned address that no refused call reads


@pytest.fixture(scope="module")
def lib():
    if not _build.library_path().exists():
        _build.build_native()
    return _native.load()


def _refused(lib, rc, code, what):
    assert rc == code and what in lib.palu_last_error().decode(), (rc, lib.palu_last_error().decode())


@pytest.mark.parametrize("kw,code,what", [
    (dict(q=None), _native.PALU_EINVAL, "null"), (dict(cu=None), _native.PALU_EINVAL, "null"),
    (dict(rows=0), _native.PALU_EINVAL, "must be positive"), (dict(batch=-1), _native.PALU_EINVAL, "must be positive"),
    (dict(n_q=6, n_kv=4), _native.PALU_EINVAL, "multiple of the KV head"), (dict(dv=24), _native.PALU_EUNSUPPORTED, "head_dim_v"),
    (dict(dv=144), _native.PALU_EUNSUPPORTED, "head_dim_v"), (dict(rows=1 << 28, n_q=8), _native.PALU_EUNSUPPORTED, "grid"),
    (dict(q_st=1028), _native.PALU_EINVAL, "strides"), (dict(v_sh=-8), _native.PALU_EINVAL, "strides"),
    (dict(k=P + 8), _native.PALU_EINVAL, "16-byte"), (dict(out=P + 2), _native.PALU_EINVAL, "16-byte")])
def test_flash_prefill_refusals(lib, kw, code, what):
    a = dict(q=P, q_st=1024, q_sh=128, k=P, k_st=256, k_sh=128, v=P, v_st=128, v_sh=64, cu=P, out=P, scale=0.1, rows=5, batch=1, n_q=8,
             n_kv=2, dv=64, stream=None)
    a.update(kw)
    _refused(lib, lib.palu_flash_prefill(*a.values()), code, what)


@pytest.mark.parametrize("kw,code,what", [
    (dict(pt=None), _native.PALU_EINVAL, "page_table is null"), (dict(page=48), _native.PALU_EINVAL, "power of two"),
    (dict(pages=0), _native.PALU_EINVAL, "num_pages"), (dict(slots=2048), _native.PALU_EUNSUPPORTED, "65536"),
    (dict(layout=2), _native.PALU_EINVAL, "cache layout"), (dict(layout=3), _native.PALU_EINVAL, "cache layout"),
    (dict(v=None), _native.PALU_EINVAL, "null"), (dict(dv=40), _native.PALU_EUNSUPPORTED, "head_dim_v"),
    (dict(q_sh=4), _native.PALU_EINVAL, "strides"), (dict(slots=512), _native.PALU_EINVAL, "workspace"),
    (dict(slots=512, ws=P + 8, bytes=1 << 40), _native.PALU_EINVAL, "workspace"),
    (dict(slots=512, ws=P, bytes=64), _native.PALU_EINVAL, "workspace")])
def test_flash_prefill_paged_refusals(lib, kw, code, what):
    a = dict(q=P, q_st=1024, q_sh=128, k=P, v=P, cu=P, start=P, pt=P, out=P, scale=0.1, rows=5, batch=1, n_q=8, n_kv=2, pages=9, page=64,
             slots=4, dv=64, layout=0, ws=None, bytes=0, stream=None)
    a.update(kw)
    _refused(lib, lib.palu_flash_prefill_paged(*a.values()), code, what)


def test_flash_prefill_workspace(lib):
    """None for contexts that are not cut, slots of 128 rows for every KV head else."""
    f = lib.palu_flash_prefill_workspace_bytes
    assert f(1, 1, 32, 8, 256, 128) == 0 and f(1 << 24, 1, 32, 8, 65536, 128) == 0
    need = f(1, 1, 32, 8, 32768, 128)
    assert need > 0 and need % (8 * (128 * 130 * 4 + 32)) == 0
    assert f(0, 1, 32, 8, 100, 128) == 0 and f(5, 1, 7, 2, 100, 128) == 0 and f(5, 1, 8, 2, -1, 128) == 0


@pytest.mark.parametrize("kw,code,what", [
    (dict(cache=None), _native.PALU_EINVAL, "null"), (dict(pt=None), _native.PALU_EINVAL, "page_table"),
    (dict(n=0), _native.PALU_EINVAL, "must be positive"), (dict(groups=0), _native.PALU_EINVAL, "must be positive"),
    (dict(layout=3), _native.PALU_EINVAL, "cache layout"), (dict(width=20), _native.PALU_EINVAL, "multiple of 8"),
    (dict(width=24, layout=1), _native.PALU_EINVAL, "multiple of 16"), (dict(width=520), _native.PALU_EINVAL, "up to 512"),
    (dict(st=100), _native.PALU_EINVAL, "strides"), (dict(rows=P + 4), _native.PALU_EINVAL, "16-byte"),
    (dict(page=16), _native.PALU_EINVAL, "power of two"), (dict(groups=70000), _native.PALU_EUNSUPPORTED, "grid")])
def test_fill_refusals(lib, kw, code, what):
    a = dict(cache=P, rows=P, st=128, sg=64, cu=P, start=None, pt=P, n=5, batch=1, groups=2, pages=9, page=64, slots=4, width=64, layout=0,
             stream=None)
    a.update(kw)
    _refused(lib, lib.palu_latent_fill_paged(*a.values()), code, what)


def _pools(n, ptr=P, size=4096):
    return (ctypes.c_void_p * n)(*[ptr] * n), (ctypes.c_longlong * n)(*[size] * n)


@pytest.mark.parametrize("kw,code,what", [
    (dict(table=None), _native.PALU_EINVAL, "null"), (dict(out=P), _native.PALU_EINVAL, "old one's memory"),
    (dict(len_out=2 * P), _native.PALU_EINVAL, "memory of its own"), (dict(batch=0), _native.PALU_EINVAL, "batch"),
    (dict(pages=0), _native.PALU_EINVAL, "num_pages"), (dict(page=33), _native.PALU_EINVAL, "power of two"),
    (dict(slots=4096), _native.PALU_EUNSUPPORTED, "65536"), (dict(ws=None), _native.PALU_EINVAL, "workspace"),
    (dict(bytes=91), _native.PALU_EINVAL, "workspace"), (dict(batch=5000), _native.PALU_EUNSUPPORTED, "4096"),
    (dict(pages=1_400_000), _native.PALU_EUNSUPPORTED, "LDS"), (dict(pools=_pools(2, P + 4)), _native.PALU_EINVAL, "pool 0"),
    (dict(pools=_pools(1, P, 40)), _native.PALU_EINVAL, "pool 0"), (dict(pools=(None, None)), _native.PALU_EINVAL, "pools")])
def test_update_refusals(lib, kw, code, what):
    a = dict(table=P, len=2 * P, parents=None, new=None, out=3 * P, len_out=4 * P, pools=_pools(2), batch=3, pages=9, page=64, slots=4,
             ws=P, bytes=1 << 30)
    a.update(kw)
    pools, sizes = a.pop("pools")
    rc = lib.palu_pages_update(a["table"], a["len"], None, None, a["out"], a["len_out"], pools, sizes, 2 if pools is None else len(pools),
                               a["batch"], a["pages"], a["page"], a["slots"], a["ws"], a["bytes"], None)
    _refused(lib, rc, code, what)


def test_compact_refusals(lib):
    pools, sizes = _pools(1)
    call = lambda table=P, n=5 * P, pages=9, ws=P: lib.palu_pages_compact(table, 2 * P, 3 * P, n, pools, sizes, 1, 3, pages, 64, 4, ws,
                                                                          1 << 30, None)
    _refused(lib, call(table=None), _native.PALU_EINVAL, "null")
    _refused(lib, call(n=None), _native.PALU_EINVAL, "null")
    _refused(lib, call(ws=None), _native.PALU_EINVAL, "workspace")
    _refused(lib, call(pages=1_400_000), _native.PALU_EUNSUPPORTED, "LDS")
    assert lib.palu_pages_workspace_bytes(0, 5) == 0 and lib.palu_pages_workspace_bytes(3, 100) >= 16 + 4 * (2 * 51 + 100)


@pytest.mark.parametrize("kw,code,what", [
    (dict(x=None), _native.PALU_EINVAL, "null"), (dict(top_id=None), _native.PALU_EINVAL, "null"), (dict(rows=0), _native.PALU_EINVAL, "positive"),
    (dict(n=0), _native.PALU_EINVAL, "positive"), (dict(dtype=2), _native.PALU_EINVAL, "dtype"), (dict(top=65), _native.PALU_EINVAL, "top"),
    (dict(n=3, top=4), _native.PALU_EINVAL, "top"), (dict(top=-1), _native.PALU_EINVAL, "top"),
    (dict(n=(1 << 30) + 1), _native.PALU_EUNSUPPORTED, "logits"), (dict(n=128256, ws=None), _native.PALU_EINVAL, "workspace"),
    (dict(n=128256, bytes=100), _native.PALU_EINVAL, "workspace"), (dict(n=128256, ws=P + 8), _native.PALU_EINVAL, "workspace")])
def test_token_logprobs_refusals(lib, kw, code, what):
    a = dict(x=P, ld=100, dtype=1, tokens=P, rows=2, n=100, top=5, lp=P, ent=P, top_lp=P, top_id=P, ws=P, bytes=1 << 30, stream=None)
    a.update(kw)
    _refused(lib, lib.palu_token_logprobs(*a.values()), code, what)


def test_cpu_tensors_are_refused():
    t = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    ints = lambda x: torch.tensor(x, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU"):
        fused.flash_prefill(t(4, 4, 128), t(4, 2, 128), t(4, 2, 64), ints([0, 4]))
    with pytest.raises(RuntimeError, match="GPU"):
        fused.paged_fill_cache(t(3, 2, 32, 64), t(4, 2, 64), ints([0, 4]), ints([[0]]))
    with pytest.raises(RuntimeError, match="GPU"):
        PagePools([t(3, 2, 32, 64)])
    with pytest.raises(RuntimeError, match="GPU"):
        decoder_ops.token_logprobs(t(4, 10), ints([0, 1, 2, 3]))


# ---- calls of the Python layer with the launch taken down: tensors that say they are on the GPU ---------------------

class _OnGpu(torch.Tensor):
    is_cuda = property(lambda self: True)


def _gpu_like(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_OnGpu)


@pytest.fixture
def launches(lib, monkeypatch):
    """The launches' arguments in place of the launches."""
    calls = []
    monkeypatch.setattr(_native, "launch", lambda name, device, *args: calls.append((name, args)))
    return calls


def _ints(x):
    return torch.tensor(x, dtype=torch.int32)


def _pool_addresses(args, at):
    """The pools' addresses and page bytes that a page-table call was given."""
    ptrs, sizes, n = args[at:at + 3]
    return list(zip(list(ptrs), list(sizes)))[:n]


def test_page_pools_follow_their_caches(launches):
    """A cache whose storage was replaced, and a tensor that was, are read where they are now."""
    from palu_tt.cache import LatentCache
    cache, rows = LatentCache(_gpu_like(5, 2, 1, 2, 64, 8), "k"), _gpu_like(5, 2, 32, 32)
    h = PagePools([cache, rows])
    call = lambda: h.update(_ints([[0, 1]]), _ints([3]))
    call()
    cache.data = _gpu_like(5, 2, 1, 4, 64, 8)                          # wider, elsewhere
    rows.set_(_gpu_like(5, 3, 32, 32))
    call()
    h.compact(_ints([[0, 1]]), _ints([3]))
    now = [(cache.data.data_ptr(), 2 * 32 * 64 * 2), (rows.data_ptr(), 3 * 32 * 32 * 2)]
    assert _pool_addresses(launches[0][1], 6) != now
    assert _pool_addresses(launches[1][1], 6) == now and _pool_addresses(launches[2][1], 4) == now
    cache.data, rows.data = _gpu_like(7, 2, 1, 2, 64, 8), _gpu_like(7, 2, 32, 32)   # larger pools: their page count counts
    call()
    assert launches[3][1][10] == h.n_pages == 7
    for bad in (_gpu_like(6, 2, 1, 2, 64, 8), _gpu_like(7, 2, 2, 2, 64, 8), _gpu_like(7, 2, 1, 2, 64, 16)[..., ::2], rows,
                _gpu_like(7, 2, 1, 2, 64, 8, dtype=torch.float16)):
        cache.data = bad
        with pytest.raises(RuntimeError):
            call()
        with pytest.raises(RuntimeError):
            h.compact(_ints([[0, 1]]), _ints([3]))
    assert len(launches) == 4


def test_workspaces_in_one_piece(lib, launches):
    """A workspace of as many elements as asked for that do not lie next to each other, or lie elsewhere, is refused: by every
    call that takes one, before anything is launched."""
    t = lambda *s: _gpu_like(*s)
    pool = t(4, 2, 32, 128)
    table, ints = _ints([[0] * 16]), _ints([0, 1])
    need = lib.palu_flash_prefill_workspace_bytes(1, 1, 4, 2, 512, 128)
    assert need > 0
    h = PagePools([t(4, 1, 32, 8)])
    cur = _ints([5])
    run = {
        "flash_prefill": lambda ws: fused.flash_prefill(t(1, 4, 128), pool, pool, ints, page_table_tensor=table, workspace=ws),
        "update": lambda ws: h.update(_ints([[0]]), cur, workspace=ws),
        "compact": lambda ws: h.compact(_ints([[0]]), cur, workspace=ws),
        "flash_decode": lambda ws: fused.flash_decode(t(1, 1, 4, 128), t(1, 2, 16384, 128), t(1, 2, 16384, 128), cur, workspace=ws),
        "linear_argmax": lambda ws: decoder_ops.linear_argmax(t(8, 64), t(32, 64), 1, workspace=ws),
        "linear_tiled": lambda ws: decoder_ops.linear_tiled(t(4, 512), t(32, 512), 2, 4, out=t(4, 32), workspace=ws)}
    size = 1 << 27
    bad = {"expanded": torch.zeros(1, dtype=torch.uint8).expand(size), "strided": torch.zeros(2 * size, dtype=torch.uint8)[::2],
           "elsewhere": torch.zeros(size, dtype=torch.uint8, device="meta")}
    for call in run.values():
        for ws in bad.values():
            with pytest.raises(RuntimeError, match="workspace must be a contiguous tensor"):
                call(ws)
    assert not launches
    for name in ("flash_prefill", "update", "compact"):
        run[name](torch.zeros(size, dtype=torch.uint8))
    assert [name for name, _ in launches] == ["flash_prefill_paged", "pages_update", "pages_compact"]


def test_out_of_the_packed_attention_is_memory_of_its_own(launches):
    """An `out` over an input is refused; one that lies in the same allocation, behind or between the rows read, is not."""
    ints = _ints([0, 6])
    buf = _gpu_like(6 * 3 * 4 * 128)
    q = buf[:6 * 4 * 128].view(6, 4, 128)
    k, v = _gpu_like(6, 2, 128), _gpu_like(6, 2, 64)
    pool, vpool, table = _gpu_like(4, 2, 32, 128), _gpu_like(4, 2, 32, 64), _ints([[0, 1]])
    own, shared = _gpu_like(6, 4, 64), lambda t: t.view(-1)[:6 * 4 * 64].view(6, 4, 64)
    packed = lambda out, **kw: fused.flash_prefill(kw.get("q", q), kw.get("k", k), kw.get("v", v), ints, out=out)
    paged = lambda out, **kw: fused.flash_prefill(q, pool, vpool, ints, page_table_tensor=kw.get("table", table), out=out,
                                                  start_pos=kw.get("start"), workspace=kw.get("workspace"))
    wide = _gpu_like(6, 6, 128)                                             # k and v as columns of wider rows
    calls = [lambda: packed(shared(q)), lambda: packed(buf[6 * 4 * 128 - 8:][:6 * 4 * 64].view(6, 4, 64)),
             lambda: packed(shared(wide), k=wide[:, 2:4]), lambda: packed(shared(wide), v=wide[:, 4:, :64]),
             lambda: packed(shared(wide), k=wide.view(6, 768)[:, 512:].unflatten(1, (2, 128))),
             lambda: paged(shared(pool)), lambda: paged(shared(vpool)),
             lambda: paged(own, workspace=own.view(-1).view(torch.uint8)),
             lambda: paged(own, table=own.view(-1).view(torch.int32)[8:10].view(1, 2)),
             lambda: paged(own, start=own.view(-1).view(torch.int32)[:1])]
    for call in calls:
        with pytest.raises(RuntimeError, match="memory of its own"):
            call()
    assert not launches
    packed(own)
    paged(own)
    packed(buf[6 * 4 * 128:][:6 * 4 * 64].view(6, 4, 64))                 # right behind q
    apart = _gpu_like(6, 6 * 4 * 64 + 512)                                # rows so far apart that `out` fits between two
    packed(apart[2, 512:].view(6, 4, 64), q=apart[:, :512].unflatten(1, (4, 128)))
    one = _gpu_like(7, 4, 128)
    packed(one[3:].view(-1)[512:512 + 1536].view(6, 4, 64), q=torch.as_strided(one, (6, 4, 128), (0, 128, 1)).as_subclass(_OnGpu))
    assert len(launches) == 5
    with pytest.raises(RuntimeError, match="memory of its own"):
        packed(apart[2, 504:504 + 1536].view(6, 4, 64), q=apart[:, :512].unflatten(1, (4, 128)))
    with pytest.raises(RuntimeError, match="workspace must be"):          # (one in pieces over the output, too)
        paged(own, workspace=own.view(-1)[::2], table=_ints([list(range(4)) * 4]))


def _packed_inputs():
    from palu_tt.cache import LatentCache
    t = _gpu_like
    return dict(q=t(6, 4, 128), k=t(6, 2, 128), v=t(6, 2, 64), kp=t(4, 2, 32, 128), vp=t(4, 2, 32, 64),
                kc=LatentCache(t(4, 2, 1, 8, 64, 8), "k"), vc=LatentCache(t(4, 2, 1, 4, 64, 8), "v"), logits=t(3, 50))


def _forward_only_calls(a):
    """The forward-only calls, each with the names of the inputs that a derivative could come by."""
    cu, table = _ints([0, 6]), _ints([[0, 1]])
    return [(("q", "k", "v"), lambda: fused.flash_prefill(a["q"], a["k"], a["v"], cu)),
            (("q", "kp", "vp"), lambda: fused.flash_prefill(a["q"], a["kp"], a["vp"], cu, page_table_tensor=table)),
            (("q", "kc", "vc"), lambda: fused.flash_prefill(a["q"], a["kc"], a["vc"], cu, page_table_tensor=table)),
            (("logits",), lambda: decoder_ops.token_logprobs(a["logits"], _ints([1, 2, 3])))]


def _with(t, change):
    from palu_tt.cache import LatentCache
    return LatentCache(change(t.data), t.role) if isinstance(t, LatentCache) else change(t)


@pytest.mark.parametrize("grad", [True, False], ids=["grad", "no_grad"])
def test_tangents_are_refused(launches, grad):
    """A forward-mode tangent would be dropped without a word, with gradients enabled or not."""
    import torch.autograd.forward_ad as fw
    with torch.set_grad_enabled(grad):
        for i, (names, _) in enumerate(_forward_only_calls(_packed_inputs())):
            for name in names:
                a = _packed_inputs()
                with fw.dual_level():
                    a[name] = _with(a[name], lambda t: fw.make_dual(t, torch.ones_like(t)))
                    with pytest.raises(RuntimeError, match="tangent"):
                        _forward_only_calls(a)[i][1]()
            with fw.dual_level():
                _forward_only_calls(_packed_inputs())[i][1]()               # without tangents all is well
    assert len(launches) == 4


def test_gradients_are_refused(launches):
    """So would a backward pass, through a cache object's storage, too."""
    for i, (names, _) in enumerate(_forward_only_calls(_packed_inputs())):
        for name in names:
            a = _packed_inputs()
            a[name] = _with(a[name], lambda t: t.requires_grad_())
            with pytest.raises(RuntimeError, match="backward"):
                _forward_only_calls(a)[i][1]()
            with torch.no_grad():
                _forward_only_calls(a)[i][1]()
    assert len(launches) == 10


@pytest.mark.parametrize("which", ["rows", "cache", "tiled cache"])
def test_fill_refuses_derivatives(launches, which):
    """Rows or a cache with a gradient or a tangent: the attention over the pages would see neither."""
    import torch.autograd.forward_ad as fw
    from palu_tt.cache import LatentCache
    cu, table = _ints([0, 6]), _ints([[0, 1]])

    def call(change):
        rows, pool = _gpu_like(6, 2, 64), _gpu_like(4, 2, 1, 4, 64, 8) if which == "tiled cache" else _gpu_like(4, 2, 32, 64)
        rows, pool = (change(rows), pool) if which == "rows" else (rows, change(pool))
        fused.paged_fill_cache(LatentCache(pool, "v") if which == "tiled cache" else pool, rows, cu, table)

    with pytest.raises(RuntimeError, match="backward"):
        call(lambda t: t.requires_grad_())
    with fw.dual_level():
        with pytest.raises(RuntimeError, match="tangent"):
            call(lambda t: fw.make_dual(t, torch.ones_like(t)))
    assert not launches
    call(lambda t: t)
    with torch.no_grad():
        call(lambda t: t.requires_grad_())
    assert len(launches) == 2


def test_token_logprobs_workspace(lib):
    """Whole 16 bytes for every part of a row, whatever the number of entries: each starts with 16-byte aligned statistics."""
    f = lib.palu_token_logprobs_workspace_bytes
    parts = f(1, 128256, 0) // 16
    assert parts > 1 and f(3000, 128256, 5) == 0
    for top in range(1, 65):
        assert f(1, 128256, top) == parts * (16 + 8 * (top + top % 2)) and f(7, 128256, top) % 16 == 0


def test_flash_prefill_workspace_goes_by_the_batch(lib):
    """No more pieces than the batch's tiles can be cut into: a tile of 128 rows stands at most max_keys / 32 levels from the start
    (4 heads to a KV head) and is cut into pieces of 8 levels or more."""
    f = lib.palu_flash_prefill_workspace_bytes
    piece = 8 * (128 * 130 * 4 + 32)                                    # of every KV head
    assert f(1, 1, 32, 8, 256, 128) == 0
    assert f(1, 1, 32, 8, 288, 128) <= 2 * piece and f(1, 1, 32, 8, 512, 128) <= 3 * piece and f(4, 4, 32, 8, 512, 128) <= 12 * piece
    assert f(1, 1, 32, 8, 2048, 128) <= 9 * piece
    # long contexts: a piece to each of the 512 places' parts, and one more for every tile
    assert f(1, 1, 32, 8, 65536, 128) <= (512 // 8 + 1) * piece
    sizes = [f(rows, rows, 32, 8, 65536, 128) for rows in (1, 8, 64, 256)]
    assert sizes == sorted(sizes) and sizes[-1] <= 2 * (512 // 8 + 1) * piece
    assert f(257, 257, 32, 8, 65536, 128) == 0                          # more than 256 sequences are not cut


def test_out_of_an_update_is_memory_of_its_own(launches):
    """Neither a pool nor the workspace may be what the new table or the new lengths are written to."""
    pool = _gpu_like(4, 1, 32, 8)
    h = PagePools([pool])
    t, ln, ws = _ints([[0, 1]]), _ints([3]), torch.zeros(1024, dtype=torch.int32)
    over = lambda x: x.view(-1).as_subclass(torch.Tensor).view(torch.int32)
    for out in ((over(pool)[:2].view(1, 2), ln.clone()), (t.clone(), over(pool)[5:6]), (ws[8:10].view(1, 2), ln.clone()), (t.clone(), ws[1023:])):
        with pytest.raises(RuntimeError, match="memory of its own"):
            h.update(t, ln, out=out, workspace=ws)
    assert not launches
    h.update(t, ln, out=(t.clone(), ln.clone()), workspace=ws)
    assert len(launches) == 1
