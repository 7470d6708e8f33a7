"""decoder_ops.token_logprobs against 64-bit torch.

Bounds: a log probability is (x - m) - log Z. x - m rounds by 2^-24 of itself, the final subtraction by 2^-24 of the result, log Z by
its sum's error and the logarithm's (2^-22 of its size, and of 1): Z's terms are exponentials whose argument t = (x - m) log2 e
rounds by 2^-23 |t|, so each is off by a factor 1 + |t| 2^-23 + 2^-22; weighted by p that is at most (H + 2) 2^-22, as
sum p |x - m| = log Z - ... <= H + log Z; the sum over n terms adds at most (n / 2048 + 64) 2^-24 (2048 accumulators or fewer
terms each). The entropy weighs the same errors by |x - m|.
"""
import math

import pytest
import torch

from palu_tt import decoder_ops as ops

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _exact(x, tokens, top):
    x = x.double()
    lp = torch.log_softmax(x, -1)
    p = lp.exp()
    ent = -(torch.where(p > 0, p * lp, 0)).sum(-1)
    ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
    return lp.gather(1, tokens[:, None])[:, 0], ent, lp.gather(1, ids), ids


def _check(x, tokens, top):
    lp, ent, tl, ids = ops.token_logprobs(x, tokens, top)
    e_lp, e_ent, e_tl, e_ids = _exact(x, tokens, top)
    n = x.shape[1]
    logz = torch.log(torch.exp(x.double() - x.double().amax(-1, keepdim=True)).sum(-1))
    sums = (e_ent + logz + 2) * 2.0 ** -22 + (n / 2048 + 64) * 2.0 ** -24
    off = lambda got, exp: torch.where(got == exp, 0, (got - exp).abs())            # (equal infinities are no distance apart)
    bound = lambda e, z, s: 2.0 ** -22 * (e.abs() + z) + s + 2.0 ** -22
    assert torch.equal(ids, e_ids)
    assert (off(lp, e_lp) <= bound(e_lp, logz, sums)).all()
    assert (off(tl, e_tl) <= bound(e_tl, logz[:, None], sums[:, None])).all()
    assert (off(ent, e_ent) <= bound(e_ent, logz, sums) * (2 + logz)).all()
    assert lp.dtype == ent.dtype == tl.dtype == torch.float32 and ids.dtype == torch.int64


def _case(rows, n, dtype, dev, seed=0, std=2.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, n, generator=g) * std).to(dev, dtype), torch.randint(0, n, (rows,), generator=g).to(dev)


@pytest.mark.parametrize("dtype", [BF, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 7), (2, 64), (5, 1000), (1, 2049), (600, 129), (17, 32000), (3, 128256), (2, 151_937),
                                    (520, 5001)])
def test_scores(gpu, dtype, rows, n):
    x, t = _case(rows, n, dtype, gpu, seed=n)
    for top in sorted({0, 1, min(5, n), min(64, n)}):
        _check(x, t, top)


@pytest.mark.parametrize("dtype", [BF, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("lead,ld", [(0, 1003), (1, 1003), (3, 1009), (5, 2000)])
def test_rows_that_start_anywhere(gpu, dtype, lead, ld):
    """Column slices of wider rows: row starts off every 16-byte boundary."""
    wide, t = _case(9, ld, dtype, gpu)
    _check(wide[:, lead:lead + 998], t % 998, 7)


@pytest.mark.parametrize("dtype", [BF, torch.float32], ids=["bf16", "f32"])
def test_orders_of_the_logits(gpu, dtype):
    """Rising and falling rows, rows of few different values (ties: the lower id first) and of one."""
    n = 40_000
    up = torch.linspace(-20, 20, n, device=gpu).to(dtype)
    few = torch.randint(0, 3, (n,), generator=torch.Generator().manual_seed(1)).to(gpu, dtype)
    x = torch.stack([up, up.flip(0), few, torch.zeros_like(up), up * 0 - 3, few * 100])
    t = torch.tensor([0, n - 1, 5, 17, 39_999, 2], device=gpu)
    for top in (1, 20, 64):
        _check(x, t, top)


@pytest.mark.parametrize("dtype", [BF, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows,n", [(2, 50_000), (2100, 3001)])
def test_rows_that_are_masked_but_for_a_few(gpu, dtype, rows, n):
    """Fewer entries allowed than asked for, anywhere in the row: the others follow at -infinity, the lower id first."""
    x, t = _case(rows, n, dtype, gpu)
    keep = torch.randint(0, n, (rows, 6), generator=torch.Generator().manual_seed(2)).to(gpu)
    x = torch.full_like(x, -math.inf).scatter(1, keep, x.gather(1, keep))
    t = torch.where(t % 2 == 0, t, keep[:, 0])
    for top in (1, 20, 64):
        _check(x, t, top)


def test_far_and_peaked_logits(gpu):
    """Large offsets (the statistics are differences from the maximum), one certain token, and -infinity in masked places."""
    x, t = _case(4, 3001, torch.float32, gpu)
    x[0] += 3e4
    x[1, 77] = 200.0
    x[2, 100:] = -math.inf
    x[3] = -math.inf
    x[3, 9] = -5.0
    t[2], t[3] = 50, 9
    _check(x, t, 9)
    lp, ent, tl, ids = ops.token_logprobs(x, torch.tensor([0, 77, 200, 10], device=gpu), 3)
    assert lp[2:].tolist() == [-math.inf, -math.inf] and ent[3] == 0 and lp[1] == 0 and tl[3].tolist() == [0, -math.inf, -math.inf]
    assert ids[3].tolist() == [9, 0, 1]


def test_signed_zeros_tie(gpu):
    x = torch.full((1, 300), -1.0, device=gpu)
    x[0, 40], x[0, 90], x[0, 200] = -0.0, 0.0, -0.0
    assert ops.token_logprobs(x, torch.tensor([0], device=gpu), 3)[3].tolist() == [[40, 90, 200]]


def test_non_finite_rows(gpu):
    """NaN, +infinity or nothing but -infinity make a row NaN, and that row only; NaN orders above every number."""
    x, t = _case(5, 700, torch.float32, gpu)
    clean = ops.token_logprobs(x, t, 4)
    x[1, 30], x[1, 600] = math.nan, math.nan
    x[2, 5] = math.inf
    x[3] = -math.inf
    lp, ent, tl, ids = ops.token_logprobs(x, t, 4)
    for r in (1, 2, 3):
        assert lp[r].isnan() and ent[r].isnan() and tl[r].isnan().all()
    for r in (0, 4):
        assert all(torch.equal(a[r], b[r]) for a, b in zip((lp, ent, tl, ids), clean))
    assert ids[1, :2].tolist() == [30, 600] and ids[2, 0] == 5 and ids[3].tolist() == [0, 1, 2, 3]


def test_tokens_outside_the_row(gpu):
    x, t = _case(4, 100, BF, gpu)
    t = torch.tensor([-1, 99, 100, -100], device=gpu)
    lp, _, _, _ = ops.token_logprobs(x, t, 0)
    assert lp[0] == 0 and lp[3] == 0 and lp[2].isnan() and lp[1].isfinite()
    assert torch.equal(ops.token_logprobs(x[:2], t[:2].to(torch.int32), 0)[0], lp[:2])


def test_rows_past_32_bits(gpu):
    """More than 2^31 logits, the last rows scored."""
    rows, n = 17_000, 128_256
    x = torch.zeros(rows, n, dtype=BF, device=gpu)
    assert x.numel() > 2 ** 31
    tail, t = _case(3, n, BF, gpu)
    x[-3:] = tail
    tokens = torch.cat([torch.zeros(rows - 3, dtype=torch.int64, device=gpu), t])
    got = ops.token_logprobs(x, tokens, 2)
    exp = ops.token_logprobs(tail, t, 2)
    # (the split of a row over waves goes by the number of rows: other sums, each within its bound)
    assert torch.equal(got[3][-3:], exp[3]) and (got[0][-3:] - exp[0]).abs().max() <= 2.0 ** -16
    assert (got[0][:-3] + math.log(n)).abs().max() <= 2.0 ** -18 and (got[1][:-3] - math.log(n)).abs().max() <= 2.0 ** -16


def test_streams_and_graph_replays(gpu):
    x, t = _case(30, 9000, torch.float32, gpu)
    exp = ops.token_logprobs(x, t, 5)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(8):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(ops.token_logprobs(x, t, 5))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in outs for a, b in zip(o, exp))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.token_logprobs(x, t, 5)
    for seed in range(4):
        x.copy_(_case(30, 9000, torch.float32, gpu, seed=seed + 5)[0])
        graph.replay()
        exp = ops.token_logprobs(x, t, 5)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(y, exp))


def test_empty_rows_and_refusals(gpu):
    x, t = _case(4, 50, BF, gpu)
    assert [tuple(o.shape) for o in ops.token_logprobs(x[:0], t[:0], 3)] == [(0,), (0,), (0, 3), (0, 3)]
    for args, what in [((x.half(), t, 1), "bf16 or fp32"), ((x, t[:2], 1), "tokens"), ((x, t, 51), "top"), ((x, t, -1), "top"),
                       ((x, t.float(), 1), "integer"), ((x[:, ::2], t, 1), "row-strided"), ((x.cpu(), t, 1), "GPU")]:
        with pytest.raises(RuntimeError, match=what):
            ops.token_logprobs(*args)
    with pytest.raises(RuntimeError, match="backward"):
        ops.token_logprobs(x.float().requires_grad_(), t, 1)
