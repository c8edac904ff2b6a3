"""Corners of the 8-bit pool and of the paged attention that a serving program
meets: zero rows, slices of a batch, rows that are missing, scales of any size,
and what a page that only later queries see may hold.  Against 64 bits, with
the bounds of _attnutil.attention_bound where values are rounded."""
import pytest
import torch

import yllang_b200 as yl
from _attnutil import attention_reference, e4m3, make_index, page_scale, store_reference
from test_paged_attention_gpu import _check, _pool

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("kind", ["warm-up", "zero queries", "tiny queries"])
def test_rows_whose_scores_vanish_give_the_mean_of_the_values(cuda, dtype, D, kind):
    """A warm-up prompt of zeros goes through the store (K's scales are 2^-100
    then) and the attention; and zero or the smallest queries meet K scales of
    2^-30.  All scores are 0 or next to it: every row gives the mean of the
    values it sees, decode and prefill alike."""
    H, G, ps, P = 2, 4, 16, 16
    prior, new = [0, 45, 70], [50, 33, 1]
    idx, pages = make_index(prior, new, ps, P, 1)
    (k, v, ks, vs), (kx, vx) = _pool(P, ps, H, D, dtype, "e4m3", cuda, 2)
    N = sum(new)
    q = torch.zeros(N, H * G, D, dtype=dtype)
    if kind == "warm-up":
        pool = yl.quant_kv_pool(P, ps, H, D, device=cuda)
        whole, _ = make_index([0] * 3, [a + b for a, b in zip(prior, new)], ps, P, 1)
        rows = torch.zeros(int(whole.qo_indptr[-1]), H, D, dtype=dtype, device=cuda)
        yl.store_kv_cache_quant(rows, rows, pool, whole)
        k, ks, kx = pool.k, pool.k_scale, torch.zeros_like(kx)
    else:
        kx = kx / ks.double().cpu()[:, None, :, None] * 2.0 ** -30
        ks.fill_(2.0 ** -30)
        if kind == "tiny queries":
            q += torch.finfo(dtype).smallest_normal
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    got = yl.paged_attention(q.to(cuda), k, v, idx, k_scale=ks, v_scale=vs, error_word=err)
    assert int(err.item()) == 0
    want, spread, reach = attention_reference(q, kx, vx, prior, new, pages)
    _check(got, want, spread, reach, dtype, "e4m3", D)


@pytest.mark.parametrize("batch", [([0, 17, 5, 200, 3, 14, 33, 1], [1] * 8),
                                   ([0, 7, 16, 31, 0, 64, 3], [50, 1, 16, 2, 1, 0, 13])], ids=["decode", "ragged"])
@pytest.mark.parametrize("ps", [1, 4, 16, 64])
@pytest.mark.parametrize("part", [(1, 3), (3, 7), (0, 4), (5, 7), (5, 6)])
def test_a_slice_of_a_batch_over_all_of_its_rows(cuda, batch, ps, part):
    """Page arrays of the sequences [lo, hi) beside the rows of the whole batch:
    those sequences' tokens and nothing else are stored, and attended."""
    lo, hi = part
    H, G, D = 3, 2, 64
    prior, new = batch
    P = sum(-(-(a + b) // ps) for a, b in zip(prior, new)) + 2
    whole, pages = make_index(prior, new, ps, P, 1)
    idx = yl.BatchIndex(whole.kv_indptr[lo:hi + 1], whole.kv_indices, whole.kv_last_page_len[lo:hi],
                        whole.qo_indptr[lo:hi + 1], None)
    first, last = sum(new[:lo]), sum(new[:hi])
    g = torch.Generator().manual_seed(ps)
    x = torch.randn(2, sum(new), H, D, generator=g) * torch.exp2(torch.randint(-3, 4, (2, sum(new), 1, 1), generator=g))
    x = x.to(torch.float16)
    pool = yl.quant_kv_pool(P, ps, H, D, device=cuda)
    want = [t.double().cpu() for t in pool]
    for i in range(2):
        store_reference(x[i, first:last].double(), want[i], want[2 + i], prior[lo:hi], new[lo:hi], pages[lo:hi], ps)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    yl.store_kv_cache_quant(x[0].to(cuda), x[1].to(cuda), pool, idx, error_word=err)
    assert int(err.item()) == 0
    for got, w in zip(pool, want):
        assert torch.equal(got.double().cpu(), w)
    q = torch.randn(sum(new), H * G, D, generator=g).to(torch.float16)
    out = torch.full_like(q, 7.0, device=cuda)
    yl.paged_attention(q.to(cuda), pool.k, pool.v, idx, k_scale=pool.k_scale, v_scale=pool.v_scale, out=out,
                       error_word=err)
    assert int(err.item()) == 0
    kx, vx = (w * s[:, None, :, None] for w, s in zip(want[:2], want[2:]))
    o, spread, reach = attention_reference(q[first:last], kx, vx, prior[lo:hi], new[lo:hi], pages[lo:hi])
    _check(out[first:last], o, spread, reach, torch.float16, "e4m3", D)
    assert bool((out[:first] == 7.0).all()) and bool((out[last:] == 7.0).all())


@pytest.mark.parametrize("batch", [([4, 0, 9], [1, 1, 1]), ([4, 0, 9], [20, 9, 1]), ([4, 0], [20, 8]), ([0, 3], [8, 16])],
                         ids=["decode", "ragged", "two", "whole pages"])
@pytest.mark.parametrize("ps", [1, 4, 8, 32])
def test_store_reports_every_missing_row(cuda, batch, ps):
    """K and V have fewer rows than the batch: the bit, and the rows that there are."""
    H, D, P = 2, 64, 48
    idx, _ = make_index(*batch, ps, P, 1)
    n = sum(batch[1])
    for rows in range(1, n + 2):
        pool = yl.quant_kv_pool(P, ps, H, D, device=cuda)
        err = torch.zeros(1, dtype=torch.int32, device=cuda)
        k = torch.ones(rows, H, D, dtype=torch.bfloat16, device=cuda)
        yl.store_kv_cache_quant(k, k, pool, idx, error_word=err)
        written = int((pool.k.float() != 0).any(-1).any(-1).sum())
        assert (int(err.item()), written) == (yl.DEVERR_TOKEN_COUNT if rows < n else 0, min(rows, n)), rows


@pytest.mark.parametrize("kv", ["e4m3", "16"])
@pytest.mark.parametrize("new,have", [(10, 5), (3, 1), (90, 60), (90, 3), (90, 89)])
@pytest.mark.parametrize("window", [0, 9])
def test_rows_that_are_there_keep_their_positions(cuda, kv, new, have, window):
    """q and o end inside the sequence's rows: the bit, and the rows that there
    are give what they give beside the others."""
    H, G, D, ps, prior = 2, 2, 64, 16, 21
    P = 12
    idx, pages = make_index([prior], [new], ps, P, 1)
    (k, v, ks, vs), (kx, vx) = _pool(P, ps, H, D, torch.float16, kv, cuda, 2)
    q = torch.randn(new, H * G, D, generator=torch.Generator().manual_seed(3)).to(torch.float16)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    got = yl.paged_attention(q[:have].to(cuda), k, v, idx, k_scale=ks, v_scale=vs, window=window, sinks=2, error_word=err)
    assert int(err.item()) == yl.DEVERR_TOKEN_COUNT
    want, spread, reach = attention_reference(q, kx, vx, [prior], [new], pages, window, 2)
    _check(got, want[:have], spread[:have], reach[:have], torch.float16, kv, D)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kv", ["e4m3", "16"])
def test_items_of_one_row_tile_behind_items_of_two(cuda, D, kv):
    """Sequences of 296 query rows (one item of one row tile, one of two, per
    head, several items to an SM) whose last value is no number: the rows in
    front of it give bit for bit what they give where it is 0, each time."""
    H, ps, B, new = 3, 16, 60, 296
    P = B * 20
    idx, pages = make_index([7] * B, [new] * B, ps, P, 1)
    (k, v, ks, vs), _ = _pool(P, ps, H, D, torch.bfloat16, kv, cuda, 2)
    q = torch.randn(B * new, H, D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(cuda)
    last = torch.tensor([mine[(7 + new - 1) // ps] for mine in pages], device=cuda), (7 + new - 1) % ps
    call = lambda: yl.paged_attention(q, k, v, idx, k_scale=ks, v_scale=vs)  # noqa: E731
    place, zero, nan = (v.view(torch.uint8), 0, 0x7F) if kv == "e4m3" else (v, 0.0, float("nan"))
    place[last] = zero
    want = call().view(B, new, H, D)
    assert bool(torch.isfinite(want).all())
    place[last] = nan
    for _ in range(8):
        got = call().view(B, new, H, D)
        assert torch.equal(got[:, :-1], want[:, :-1])
        assert bool(torch.isnan(got[:, -1]).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ps,count", [(16, 1), (16, 9), (64, 1), (64, 50), (4, 1), (4, 3)])
@pytest.mark.parametrize("scale", [7.0, 0.3, 1.0, 15 * 2.0 ** -7, 1e-3])
def test_store_beside_a_scale_that_is_no_power_of_two(cuda, dtype, ps, count, scale):
    """A page whose scale another program chose keeps it while it is large
    enough, and codes are of the product with its fp32 reciprocal: off from x by
    half a step of e4m3 (2^-4 of the value, 2^-10 below its normal numbers) and
    the reciprocal's and the product's roundings.  Louder tokens bring the power
    of two that they need, and the held codes are multiplied by the quotient."""
    H, D, P, held = 3, 64, 2, 1
    idx, pages = make_index([held], [count], ps, P, 1)
    page = pages[0][0]
    g = torch.Generator().manual_seed(count)
    s = torch.tensor(scale)
    for grow in (False, True):
        pool = yl.quant_kv_pool(P, ps, H, D, device=cuda)
        for t in (pool.k, pool.v):
            t.view(torch.uint8).copy_(torch.randint(0, 127, t.shape, generator=g, dtype=torch.uint8))
        pool.k_scale.fill_(scale)
        pool.v_scale.fill_(scale)
        before = pool.k[page, :held].cpu().float()
        x = torch.randint(-255, 256, (count, H, D), generator=g).float()
        x[..., :4] = torch.tensor([175.0, -203.0, 119.0, 77.0])  # borders of a scale of 7
        x = (x * (s / 7)).to(dtype)
        if grow:
            x[0, :, 5] = 1000 * s
        yl.store_kv_cache_quant(x.to(cuda), x.to(cuda), pool, idx)
        after = page_scale(float(x[0, 0].double().abs().max())) if grow else s
        after = torch.as_tensor(after, dtype=torch.float32)
        assert bool((pool.k_scale[page] == after).all())
        codes = pool.k[page].cpu()
        assert torch.equal(codes[held:held + count].double(), e4m3((x.float() * (1 / after)).double()))
        off = (codes[held:held + count].double() * after.double() - x.double()).abs()
        assert bool((off <= x.double().abs() * (2.0 ** -4 + 2.0 ** -23) + 2.0 ** -10 * after.double()).all())
        want = e4m3((before * (s / after)).double()) if grow else before.double()
        assert torch.equal(codes[:held].double(), want)


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("prior,new", [(31, 2), (26, 12), (3, 40)])
def test_scales_of_unseen_pages_do_not_reach_a_query(cuda, which, bad, prior, new):
    """The last page's scale is no finite number: the queries in front of the
    page give what they give without it, the others no number."""
    H, G, D, ps, P = 2, 2, 128, 16, 10
    idx, pages = make_index([prior], [new], ps, P, 1)
    (k, v, ks, vs), (kx, vx) = _pool(P, ps, H, D, torch.bfloat16, "e4m3", cuda, 2)
    q = torch.randn(new, H * G, D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    (ks if which == "k" else vs)[pages[0][2]] = bad
    got = yl.paged_attention(q.to(cuda), k, v, idx, k_scale=ks, v_scale=vs)
    want, spread, reach = attention_reference(q, kx, vx, [prior], [new], pages)
    before = 2 * ps - prior
    _check(got, want, spread, reach, torch.bfloat16, "e4m3", D, rows=slice(0, before))
    if which == "v" or bad != bad:
        assert not bool(torch.isfinite(got[before:]).all(-1).any())
