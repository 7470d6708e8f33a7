"""Quantised page pools as a server uses them: packed prompts quantised into pages, samples forked from them, decode steps over the
forks with the prompts read once for all samples, a rejected draft, a compaction, a captured step, and the pages read back.
Every step is checked against plain attention in 64 bits over per-row lists of the keys and values that the caches should hold:
the rows that were written, quantised on the host."""
import pytest
import torch

from palu_tt import fused
from palu_tt.cache import MXCache, mx_dequantize, mx_quantize
from palu_tt.pages import PagePools

pytestmark = pytest.mark.gpu

HD, BF = 128, torch.bfloat16


def _attend(q, k, v):
    """q [n_q, 128] over k [n, n_kv, 128], v [n, n_kv, w] in 64 bits: (out, sum of p |v|)."""
    rep = q.shape[0] // k.shape[1]
    k, v = (t.double().repeat_interleave(rep, dim=1) for t in (k, v))
    p = torch.softmax((q.double()[None] * k).sum(-1) * HD ** -0.5, 0)[..., None]
    return (p * v).sum(0), (p * v.abs()).sum(0)


def _close(got, exp, mag):
    # the probabilities' rounding to bf16 (2^-8 of each), the result's, and 2^-10 for the fp32 scores and sums of a few hundred keys
    assert ((got.double() - exp).abs() <= mag * (2.0 ** -8 + 2.0 ** -10) + 2.0 ** -8 * exp.abs() + 1e-6).all()


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("page,w", [(32, 64), (64, 128)])
def test_prompts_samples_and_steps(gpu, fmt, page, w):
    g = torch.Generator().manual_seed(page)
    rand = lambda *s: torch.randn(*s, generator=g).to(BF)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)
    held = lambda rows: mx_dequantize(*mx_quantize(rows, fmt), fmt)
    n_pages, B, slots, nq, nkv = 64, 6, 10, 8, 2
    kp, vp = MXCache.zeros(n_pages, nkv, page, HD, gpu, "k", fmt), MXCache.zeros(n_pages, nkv, page, w, gpu, "v", fmt)
    kp.data.fill_(255)                                               # NaN wherever nothing has been written
    vp.data.fill_(255)
    pools = PagePools([kp, vp])
    table, lengths = torch.full((B, slots), -1, dtype=torch.int32, device=gpu), ints([0] * B)
    keys, vals = [[] for _ in range(B)], [[] for _ in range(B)]

    # prompts in rows 0 and 3, keys and values columns of one projection
    prompts = [150, 0, 0, 70, 0, 0]
    table, lengths = pools.update(table, lengths, new_lengths=ints(prompts))
    T, cu = sum(prompts), ints([sum(prompts[:b]) for b in range(B + 1)])
    qkv = rand(T, nkv * (HD + w)).to(gpu)
    k, v = qkv[:, :nkv * HD].unflatten(1, (nkv, HD)), qkv[:, nkv * HD:].unflatten(1, (nkv, w))
    fused.paged_fill_cache(kp, k, cu, table)
    fused.paged_fill_cache(vp, v, cu, table)
    at = 0
    for b, n in enumerate(prompts):
        keys[b] = list(held(k[at:at + n].cpu()).to(gpu))
        vals[b] = list(held(v[at:at + n].cpu()).to(gpu))
        at += n

    # samples: rows 1 and 2 of row 0's prompt, row 5 of row 3's, row 4 stays empty
    parents = [0, 0, 0, 3, -1, 3]
    table, lengths = pools.update(table, lengths, parents=ints(parents))
    keys, vals = ([list(x[p]) if p >= 0 else [] for p in parents] for x in (keys, vals))
    assert lengths.tolist() == [150, 150, 150, 70, 0, 70]
    # rows 0 to 2 are a group that shares its prompt, row 3 is one of its own, 4 and 5 one that shares nothing (4 is empty)
    groups, shared, alone = ints([0, 3, 4, 6]), ints([150, 0, 0]), ints([150, 70, 0])

    def step():
        """One decode step of all live rows: the single-position append, decode attention without groups and with them."""
        nonlocal table, lengths
        live = [bool(x) for x in keys]
        pos = torch.where(ints([int(x) for x in live]) > 0, lengths, -1).to(torch.int32)
        table, lengths = pools.update(table, lengths, new_lengths=lengths + ints([int(x) for x in live]))
        q, k, v = rand(B, nq, HD), rand(B, nkv, HD), rand(B, nkv, w)
        fused.paged_update_cache(kp, k.to(gpu), pos, page_table=table)
        fused.paged_update_cache(vp, v.to(gpu), pos, page_table=table)
        q = q.to(gpu)
        one = fused.flash_decode(q[None], kp, vp, pos, page_table_tensor=table)[0]
        both = fused.flash_decode_shared(q[None], kp, vp, pos, table, shared, groups)[0]
        lone = fused.flash_decode_shared(q[None], kp, vp, pos, table, alone, groups)[0]
        for b in range(B):
            if not live[b]:
                assert (one[b] == 0).all() and (both[b] == 0).all() and (lone[b] == 0).all()
                continue
            keys[b].append(held(k[b]).to(gpu))
            vals[b].append(held(v[b]).to(gpu))
            exp = _attend(q[b], torch.stack(keys[b]), torch.stack(vals[b]))
            for out in (one, both, lone):
                _close(out[b], *exp)
        return q, pos, both

    for _ in range(3):
        step()
    # a draft of 4 rows in row 1, of which 2 are kept
    start, cu4 = lengths.clone(), ints([0, 0, 4, 4, 4, 4, 4])
    table, lengths = pools.update(table, lengths, new_lengths=lengths + ints([0, 4, 0, 0, 0, 0]))
    k, v = rand(4, nkv, HD), rand(4, nkv, w)
    fused.paged_fill_cache(kp, k.to(gpu), cu4, table, start_pos=start)
    fused.paged_fill_cache(vp, v.to(gpu), cu4, table, start_pos=start)
    table, lengths = pools.update(table, lengths, new_lengths=lengths - ints([0, 2, 0, 0, 0, 0]))
    keys[1] += list(held(k[:2]).to(gpu))
    vals[1] += list(held(v[:2]).to(gpu))
    # row 2 ends, the pools are compacted, two more steps
    table, lengths = pools.update(table, lengths, new_lengths=ints([n if b != 2 else 0 for b, n in enumerate(lengths.tolist())]))
    keys[2], vals[2] = [], []
    groups, shared, alone = ints([0, 2, 3, 4, 6]), ints([150, 0, 0, 0]), ints([150, 0, 70, 0])
    before = table.clone()
    table, used = pools.compact(table, lengths)
    assert int(used) == len(set(before[before >= 0].tolist())) and int(table.max()) == int(used) - 1
    for _ in range(2):
        q, pos, both = step()

    # the last step again, captured: every replay gives what the eager call gave
    ws = torch.empty(1 << 23, dtype=torch.uint8, device=gpu)
    args = (q[None], kp, vp, pos, table, shared, groups)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            again = fused.flash_decode_shared(*args, workspace=ws)[0]
    for _ in range(3):
        again.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(again, both)
        assert torch.equal(fused.flash_decode_shared(*args, workspace=ws)[0], both)

    # every row's cache read back: exactly what was written, quantised
    n = lengths.tolist()
    cu = ints([sum(n[:b]) for b in range(B + 1)])
    for pool, rows in ((kp, keys), (vp, vals)):
        got = fused.paged_read_cache(pool, sum(n), cu, table)
        assert torch.equal(got, torch.stack([x for row in rows for x in row]))
