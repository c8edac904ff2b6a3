"""Corners of the 8-bit pool and of the paged attention that a serving program
meets: zero rows, slices of a batch, rows that are missing, scales of any size,
and what a page that only later queries see may hold.  Against 64 bits, with
the bounds of _attnutil.attention_bound where values are rounded."""
import pytest
import torch

import yllang_b200 as yl
from _attnutil import attention_bound, attention_reference, e4m3, make_index, page_scale, store_reference
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


@pytest.mark.parametrize("new", [[1, 1, 1], [20, 9, 1], [40, 30, 16]])
@pytest.mark.parametrize("ps", [1, 8, 32])
def test_store_reports_a_batch_far_behind_the_rows(cuda, ps, new):
    """A slice of a batch all of whose rows lie behind those of K and V: the bit,
    and nothing written."""
    H, D, P = 2, 64, 100
    idx, _ = make_index([0] * len(new), new, ps, P, 1)
    idx = idx._replace(qo_indptr=idx.qo_indptr + 5000)
    for rows in (1, 3, 100):
        pool = yl.quant_kv_pool(P, ps, H, D, device=cuda)
        err = torch.zeros(1, dtype=torch.int32, device=cuda)
        k = torch.ones(rows, H, D, dtype=torch.bfloat16, device=cuda)
        yl.store_kv_cache_quant(k, k, pool, idx, error_word=err)
        assert int(err.item()) == yl.DEVERR_TOKEN_COUNT
        assert not bool(pool.k.float().any())


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


def _wide_bound(want, spread, reach, dtype, D, scores, values, sums):
    """attention_bound where scores are off by `scores` more, values by a part
    of `values`, and the result by `sums`."""
    grown = torch.exp(2 * scores) - 1  # of a weight over the sum of weights
    return attention_bound(want, spread * (1 + grown), reach, dtype, torch.float16, D) + spread * (grown + values) + sums


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("ps", [5, 16, 128])
@pytest.mark.parametrize("window", [0, 60])
def test_scales_that_are_no_powers_of_two(cuda, dtype, D, ps, window):
    """Any fp32 scales, decode and prefill: the elements of a page are off by
    2^-10 at most (prefill rounds scale and product to fp16, half a step of
    2^-11 each), so scores by 2^-10 of the sum of |q| |k|."""
    H, G = 2, 4
    prior, new = [0, 37, 100], [60, 20, 1]
    P = sum(-(-(a + b) // ps) for a, b in zip(prior, new)) + 2
    idx, pages = make_index(prior, new, ps, P, 1)
    (k, v, ks, vs), (kx, vx) = _pool(P, ps, H, D, dtype, "e4m3", cuda, 2)
    g = torch.Generator().manual_seed(4)
    for s, x in ((ks, kx), (vs, vx)):
        other = s.cpu() * (1 + torch.rand(s.shape, generator=g))
        x.mul_((other.double() / s.double().cpu())[:, None, :, None])
        s.copy_(other)
    q = (torch.randn(sum(new), H * G, D, generator=g) / 2).to(dtype)
    got = yl.paged_attention(q.to(cuda), k, v, idx, k_scale=ks, v_scale=vs, window=window, sinks=3).cpu().double()
    want, spread, reach = attention_reference(q, kx, vx, prior, new, pages, window, 3)
    bound = _wide_bound(want, spread, reach, dtype, D, 2.0 ** -10 * reach, 2.0 ** -10, 0)
    assert float(((got - want).abs() / bound).max()) <= 1
    rows = slice(sum(new) - 1, None)  # decode: scales stay in fp32, weights are rounded once
    bound = attention_bound(want, spread, reach, dtype, torch.float16, D)
    assert float(((got - want).abs() / bound)[rows].max()) <= 1


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("place", [0, 1, 3])
@pytest.mark.parametrize("far", [0, 8, 15, 16, 20, 24, 40])
def test_a_page_of_small_values_with_all_the_weight(cuda, new, place, far):
    """One page's V scale lies 2^far under the others', and all of the weight on
    its tokens: down to 2^-15 the result is as exact as ever, and below off by
    2^-25 of the largest scale.  The page may be the first, the last or between."""
    H, G, D, ps, P, total = 2, 2, 64, 64, 6, 256
    idx, pages = make_index([0], [total], ps, P, 1)
    idx = idx._replace(qo_indptr=torch.tensor([0, new], dtype=torch.int32, device=cuda))
    (k, v, ks, vs), (_, vx) = _pool(P, ps, H, D, torch.float16, "e4m3", cuda, 2)
    codes = vx / vs.double().cpu()[:, None, :, None]
    page = pages[0][place]
    vs.fill_(1.0)
    vs[page] = 2.0 ** -far
    ks.fill_(2.0 ** -3)
    kx = torch.full((P, ps, H, D), -1.0, dtype=torch.float64)  # scores of about 20, the page's, and -20
    kx[page] = 1.0 + torch.arange(ps)[:, None, None].double() % 3 / 8
    k.view(torch.uint8).copy_((kx * 8).to(torch.float8_e4m3fn).view(torch.uint8).to(cuda))
    vx = codes * vs.double().cpu()[:, None, :, None]
    q = 2.5 + torch.rand(new, H * G, D, generator=torch.Generator().manual_seed(3)) / 4
    q = q.to(torch.float16)
    got = yl.paged_attention(q.to(cuda), k, v, idx, k_scale=ks, v_scale=vs).double().cpu()
    want, spread, reach = attention_reference(q, kx, vx, [total - new], [new], pages)
    seen = torch.arange(total - new, total) >= place * ps + ps - 1  # queries that see all of the page
    size = codes.abs()[pages[0]].sum((0, 1)).repeat_interleave(G, 0)  # sum of |codes| of the sequence's tokens
    small = codes.abs()[page].sum(0).repeat_interleave(G, 0)
    # (the others' weights are e^-40 and less: lost or not, 2^-36 of their codes bounds them)
    sums = 2.0 ** -36 * size + 2.0 ** (-28 - far) * small + (2.0 ** -25 if far > 15 else 0)
    sums = sums + 2.0 ** -25  # half of fp16's smallest step, of the result
    bound = _wide_bound(want, spread, reach, torch.float16, D, 0 * reach, 0, sums)
    assert bool(seen.any())
    assert float(((got - want).abs() / bound)[seen].max()) <= 1
    if far <= 8:  # and the bound is one that a lost page would not pass
        assert float((want.abs() / bound)[seen].median()) > 16


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("far", [0, 15, 18, 22])
def test_a_page_of_small_keys_with_all_the_weight(cuda, new, far):
    """A page whose K scale lies 2^far above the others' and whose scores lie far
    below theirs: the others' keep their precision down to 2^-15, and elements
    are off by 2^-25 of the largest scale below."""
    H, G, D, ps, P, total = 2, 2, 64, 16, 8, 64
    idx, pages = make_index([0], [total], ps, P, 1)
    idx = idx._replace(qo_indptr=torch.tensor([0, new], dtype=torch.int32, device=cuda))
    (k, v, ks, vs), (kx, vx) = _pool(P, ps, H, D, torch.bfloat16, "e4m3", cuda, 2)
    page = pages[0][0]
    kx = kx / ks.double().cpu()[:, None, :, None]
    kx[page] = -kx[page].abs().clamp(min=16)
    k.view(torch.uint8).copy_(kx.to(torch.float8_e4m3fn).view(torch.uint8).to(cuda))
    ks.fill_(2.0 ** -8)
    ks[page] = 2.0 ** (far - 8)
    kx = kx * ks.double().cpu()[:, None, :, None]
    q = (1 + torch.rand(new, H * G, D, generator=torch.Generator().manual_seed(3))).to(torch.bfloat16)
    got = yl.paged_attention(q.to(cuda), k, v, idx, k_scale=ks, v_scale=vs).double().cpu()
    want, spread, _ = attention_reference(q, kx, vx, [total - new], [new], pages)
    if far:
        kx[page] = 0  # scores of -2^15 and less, whose own error does not matter
    _, _, reach = attention_reference(q, kx, vx, [total - new], [new], pages)
    scores = 2.0 ** -25 * float(ks.max()) * q.double().abs().sum(-1, keepdim=True) * D ** -0.5 if far > 15 else 0 * reach
    bound = _wide_bound(want, spread, reach, torch.bfloat16, D, scores, 0, 0)
    assert float(((got - want).abs() / bound).max()) <= 1


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("kv", ["e4m3", "16"])
def test_values_near_the_largest_allowed(cuda, new, kv):
    """V elements just under 2^80 come through."""
    H, G, D, ps, P = 2, 2, 64, 16, 8
    idx, pages = make_index([60], [new], ps, P, 1)
    (k, v, ks, vs), (kx, vx) = _pool(P, ps, H, D, torch.bfloat16, kv, cuda, 2)
    up = 2.0 ** 70
    (v if kv == "16" else vs).mul_(up)
    vx = vx * up
    assert float(vx.abs().max()) < 2.0 ** 80
    q = torch.randn(new, H * G, D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    got = yl.paged_attention(q.to(cuda), k, v, idx, k_scale=ks, v_scale=vs)
    want, spread, reach = attention_reference(q, kx, vx, [60], [new], pages)
    _check(got, want, spread, reach, torch.bfloat16, kv, D)


@pytest.mark.parametrize("kv,dtype", [("e4m3", torch.bfloat16), ("e4m3", torch.float16), ("16", torch.bfloat16)])
@pytest.mark.parametrize("window", [0, 700])
def test_a_mixed_batch_repeats_itself_bit_for_bit(cuda, kv, dtype, window):
    """Prompts, chunks and decode steps in one call, with work for every SM: the
    joins' order and the items' way to the SMs do not show in the results."""
    H, G, D, ps = 8, 4, 128, 16
    prior = [0, 3000, 511, 4095, 0, 77] + [37 * i % 4000 for i in range(60)]
    new = [1500, 512, 100, 17, 1, 300] + [1] * 60
    P = sum(-(-(a + b) // ps) for a, b in zip(prior, new)) + 1
    idx, _ = make_index(prior, new, ps, P, 1)
    (k, v, ks, vs), _ = _pool(P, ps, H, D, dtype, kv, cuda, 2)
    q = torch.randn(sum(new), H * G, D, generator=torch.Generator().manual_seed(3)).to(dtype).to(cuda)
    other = torch.empty(1 << 26, dtype=torch.uint8, device=cuda)
    first = None
    for i in range(12):
        out = torch.full_like(q, float("nan"))
        yl.paged_attention(q, k, v, idx, k_scale=ks, v_scale=vs, window=window, sinks=4, out=out)
        other.fill_(i)  # (something else in the caches and on the SMs)
        first = out if first is None else first
        assert bool(torch.isfinite(out).all()) and torch.equal(out, first)
