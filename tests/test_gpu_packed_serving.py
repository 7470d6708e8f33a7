"""The packed-batch ops together, as a server over paged caches uses them: packed prompts into pages, their attention, beams forked
from them, decode steps over the forked rows, a compaction between two steps, and the scores of what was picked. Every step is
checked against plain attention in 64 bits over per-sequence lists of keys and values."""
import pytest
import torch

from palu_tt import decoder_ops, fused
from palu_tt.cache import LatentCache
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


@pytest.mark.parametrize("layout", ["rows", "tiled"])
def test_prompts_beams_and_scores(gpu, layout):
    g = torch.Generator().manual_seed(3)
    rand = lambda *s: torch.randn(*s, generator=g).to(gpu, BF)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)
    page, n_pages, B, slots, nq, nkv, w = 32, 40, 6, 8, 8, 2, 64
    kp, vp = (torch.full((n_pages, nkv, page, x), float("nan"), dtype=BF, device=gpu) for x in (HD, w))
    if layout == "tiled":
        kp, vp = LatentCache.from_rows(kp, "k"), LatentCache.from_rows(vp, "v")
    pools = PagePools([kp, vp])
    table, lengths = torch.full((B, slots), -1, dtype=torch.int32, device=gpu), ints([0] * B)
    keys, vals = [[] for _ in range(B)], [[] for _ in range(B)]      # what every row's cache should hold

    def feed(new):
        """new[b] rows of every sequence: pages for them, their keys and values into the pages, their attention."""
        nonlocal table, lengths
        start = lengths
        table, lengths = pools.update(table, lengths, new_lengths=lengths + ints(new))
        T, cu = sum(new), ints([sum(new[:b]) for b in range(B + 1)])
        q, k, v = rand(T, nq, HD), rand(T, nkv, HD), rand(T, nkv, w)
        fused.paged_fill_cache(kp, k, cu, table, start_pos=start)
        fused.paged_fill_cache(vp, v, cu, table, start_pos=start)
        out = fused.flash_prefill(q, kp, vp, cu, page_table_tensor=table, start_pos=start)
        if start.eq(0).all():                                        # prompts: the same over the packed rows themselves
            assert torch.equal(out, fused.flash_prefill(q, k, v, cu))
        at = 0
        for b, n in enumerate(new):
            for _ in range(n):
                keys[b].append(k[at])
                vals[b].append(v[at])
                _close(out[at], *_attend(q[at], torch.stack(keys[b]), torch.stack(vals[b])))
                at += 1

    feed([33, 7, 64, 1, 0, 20])
    # beams: rows 1, 3 and 4 go on from row 0 (in the middle of its second page), row 5 from row 2 (at a page's end), row 2 itself ends
    parents = [0, 0, 2, 0, 0, 2]
    table, lengths = pools.update(table, lengths, parents=ints(parents), new_lengths=ints([33, 33, 0, 33, 33, 64]))
    keys, vals = ([list(x[p]) if b != 2 else [] for b, p in enumerate(parents)] for x in (keys, vals))
    assert lengths.tolist() == [33, 33, 0, 33, 33, 64]
    used = table[table >= 0]
    assert table[0, 0] == table[1, 0] == table[4, 0] and len({int(table[b, 1]) for b in (0, 1, 3, 4)}) == 4 and used.max() < n_pages

    def step():
        """One decode step of all live rows, through the single-position append and the stock decode."""
        nonlocal table, lengths
        grow = ints([0 if not keys[b] else 1 for b in range(B)])
        pos = torch.where(grow > 0, lengths, -1).to(torch.int32)
        table, lengths = pools.update(table, lengths, new_lengths=lengths + grow)
        q, k, v = rand(B, nq, HD), rand(B, nkv, HD), rand(B, nkv, w)
        fused.paged_update_cache(kp, k[:, :, :], pos, page_table=table)
        fused.paged_update_cache(vp, v[:, :, :], pos, page_table=table)
        out = fused.flash_decode(q[None], kp, vp, pos, page_table_tensor=table)[0]
        again = fused.flash_prefill(q, kp, vp, ints(list(range(B + 1))), page_table_tensor=table, start_pos=pos)
        for b in range(B):
            if keys[b]:
                keys[b].append(k[b])
                vals[b].append(v[b])
                exp, mag = _attend(q[b], torch.stack(keys[b]), torch.stack(vals[b]))
                _close(out[b], exp, mag)
                _close(again[b], exp, mag)
            else:
                assert (again[b] == 0).all()
        return out

    step()
    live = table[table >= 0].unique().numel()
    table, n = pools.compact(table, lengths)
    assert n.item() == live and table.max() == live - 1
    feed([2, 0, 5, 40, 0, 1])                                        # a new request in the freed row, longer turns, after the move
    out = step()
    logits = out.reshape(B, -1).float() @ torch.randn(nq * w, 1000, generator=g).to(gpu)
    ids = torch.randint(0, 1000, (B,), generator=g).to(gpu)
    live_rows = [b for b in range(B) if keys[b]]
    lp, ent, top_lp, top_id = decoder_ops.token_logprobs(logits[live_rows], ids[live_rows], 5)
    ref = torch.log_softmax(logits[live_rows].double(), -1)
    assert (lp - ref.gather(1, ids[live_rows, None])[:, 0]).abs().max() <= 2.0 ** -16 * ref.abs().max()
    assert torch.equal(top_id[:, 0], logits[live_rows].argmax(-1)) and (top_lp - ref.topk(5).values).abs().max() <= 2.0 ** -16 * ref.abs().max()
    assert (ent + (ref.exp() * ref).sum(-1)).abs().max() <= 2.0 ** -14
