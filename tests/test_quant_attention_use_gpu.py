"""The 8-bit pool and the paged attention as a serving loop uses them, beyond
the shape tables: captured and replayed steps, other streams, a workspace that
holds anything, prompts over many tiles, scores far apart, pools past 2^32
bytes, page tables that name a page twice, and batches that mix prompts with
decode steps."""
import pytest
import torch

import yllang_b200 as yl
from _attnutil import HALF_STEP, attention_reference, make_index, store_reference
from test_paged_attention_gpu import _check, _pool, _run
from test_quant_pool_gpu import _filled_pool, _host, _loud, _store_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("kv", ["e4m3", "16"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (200, 4)])
def test_prompts_over_many_tiles(cuda, D, kv, window, sinks):
    """Queries over more than one tile of rows and keys, odd lengths."""
    _run(cuda, [0, 333], [401, 170], H=1, G=3, D=D, kv=kv, window=window, sinks=sinks, dtype=torch.float16, seed=D)


@pytest.mark.parametrize("kv", ["e4m3", "16"])
@pytest.mark.parametrize("new", [1, 300])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scores_far_apart(cuda, kv, new, dtype):
    """Scores with a spread of tens: the running maximum moves often, and late."""
    _run(cuda, [500], [new], H=1, G=2, D=128, kv=kv, dtype=dtype, scale=0.9, seed=4)


@pytest.mark.parametrize("kv", ["e4m3", "16"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (130, 7)])
def test_prompts_and_decode_steps_together(cuda, kv, window, sinks):
    """One call over sequences of both kinds, empty ones between them, the last
    sequence a decode step."""
    _run(cuda, [0, 900, 0, 64, 511, 0, 17, 1023], [260, 1, 0, 17, 2, 1, 130, 1], H=2, G=4, kv=kv, window=window,
         sinks=sinks, pad=3, seed=6)


def _direct(q, k, v, ks, vs, idx, **kw):
    return yl.paged_attention(q, k, v, idx, k_scale=ks, v_scale=vs, **kw)


def test_workspace_holding_anything(cuda):
    """A call leaves nothing in the workspace that the next one relies on."""
    H, G, D, ps, P = 2, 4, 128, 16, 200
    (k, v, ks, vs), _ = _pool(P, ps, H, D, torch.bfloat16, "e4m3", cuda, 2)
    for prior, new in (([0, 700], [300, 150]), ([900, 3], [1, 1]), ([800, 3, 40], [1, 200, 4])):
        idx, _ = make_index(prior, new, ps, P, 1)
        q = torch.randn(sum(new), H * G, D, device=cuda).to(torch.bfloat16)
        want = _direct(q, k, v, ks, vs, idx)
        need = yl.paged_attention_workspace(q, k, v, idx, k_scale=ks, v_scale=vs)
        work = torch.full((need,), 0xFF, dtype=torch.uint8, device=cuda)
        for fill in (0xFF, 0x00, 0x3C, None, None):
            if fill is not None:
                work.fill_(fill)
            assert torch.equal(want, _direct(q, k, v, ks, vs, idx, workspace=work))


def test_results_are_the_same_every_time(cuda):
    """Items are handed out by a counter; no result depends on who takes them."""
    H, G, D, ps, P = 4, 4, 128, 16, 900
    (k, v, ks, vs), _ = _pool(P, ps, H, D, torch.bfloat16, "e4m3", cuda, 2)
    idx, _ = make_index([0, 5000, 17, 3000], [1500, 1, 700, 2], ps, P, 1)
    q = torch.randn(2203, H * G, D, device=cuda).to(torch.bfloat16)
    want = _direct(q, k, v, ks, vs, idx)
    for _ in range(20):
        assert torch.equal(want, _direct(q, k, v, ks, vs, idx))


def test_a_captured_serving_step(cuda):
    """Store, attention and read-back of one step captured in a graph; replays
    follow the rows, lengths and pages, a prompt's replay among them."""
    H, G, D, ps, P, B, N = 2, 4, 128, 16, 120, 3, 200
    pool = _filled_pool(P, ps, H, D, None, cuda, 1)
    idx, _ = make_index([700, 3, 40], [1, 1, 1], ps, P, 1, spare=60)
    q = torch.zeros(N, H * G, D, dtype=torch.bfloat16, device=cuda)
    k, v = (torch.zeros(N, H, D, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    slots = torch.zeros(N, dtype=torch.int64, device=cuda)
    out, back = torch.zeros_like(q), (torch.zeros_like(k), torch.zeros_like(k))

    def step():
        yl.store_kv_cache_quant(k, v, pool, idx)
        _direct(q, pool.k, pool.v, pool.k_scale, pool.v_scale, idx, out=out)
        yl.load_kv_cache_quant(pool, slots, out=back)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed, (prior, new) in enumerate([([700, 3, 40], [1, 1, 1]), ([0, 600, 5], [150, 1, 40]), ([33, 0, 64], [1, 0, 1])]):
        at, pages = make_index(prior, new, ps, P, seed)
        n, g = sum(new), torch.Generator().manual_seed(seed)
        for name in ("kv_indptr", "kv_last_page_len", "qo_indptr"):
            getattr(idx, name).copy_(getattr(at, name))
        idx.kv_indices[:at.kv_indices.numel()].copy_(at.kv_indices)
        slots.fill_(-1)
        slots[:n].copy_(at.slot_mapping)
        qh = torch.randn(N, H * G, D, generator=g).to(torch.bfloat16)
        kh, vh = (_loud((N, H, D), g, torch.bfloat16) for _ in range(2))
        q.copy_(qh), k.copy_(kh), v.copy_(vh)
        want = _host(pool)
        store_reference(kh[:n].double(), want[0], want[2], prior, new, pages, ps)
        store_reference(vh[:n].double(), want[1], want[3], prior, new, pages, ps)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(_host(pool), want):
            assert torch.equal(a, b)
        kx, vx = (c * s[:, None, :, None] for c, s in ((want[0], want[2]), (want[1], want[3])))
        o, spread, reach = attention_reference(qh[:n], kx, vx, prior, new, pages)
        _check(out[:n], o, spread, reach, torch.bfloat16, "e4m3", D)
        s = at.slot_mapping.cpu()
        assert torch.equal(back[0][:n].cpu().double(), kx[s // ps, s % ps].to(torch.bfloat16).double())
        assert not bool(back[1][n:].any())


def test_two_graphs_of_one_workspace_each(cuda):
    """Two captured decode steps, each with its own workspace, replayed on two
    streams at once."""
    H, G, D, ps, P = 4, 4, 128, 16, 600
    (k, v, ks, vs), _ = _pool(P, ps, H, D, torch.bfloat16, "e4m3", cuda, 2)
    cases = []
    for prior, new in (([4000, 100, 2500], [1, 1, 1]), ([1000, 3000], [90, 1])):
        idx, _ = make_index(prior, new, ps, P, 1)
        q = torch.randn(sum(new), H * G, D, device=cuda).to(torch.bfloat16)
        out = torch.zeros_like(q)
        work = torch.empty(yl.paged_attention_workspace(q, k, v, idx, k_scale=ks, v_scale=vs), dtype=torch.uint8,
                           device=cuda)
        want = _direct(q, k, v, ks, vs, idx)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            _direct(q, k, v, ks, vs, idx, out=out, workspace=work)
        cases.append((graph, out, want, torch.cuda.Stream()))
    for _ in range(10):
        for graph, out, _, stream in cases:
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, out, want, _ in cases:
        assert torch.equal(out, want)


def test_store_and_load_on_another_stream(cuda):
    """Rows made on a stream and stored on it; the pool is read there too."""
    H, D, ps, P = 2, 128, 16, 40
    prior, new = [5, 0, 100], [1, 200, 3]
    idx, pages = make_index(prior, new, ps, P, 1)
    pool = _filled_pool(P, ps, H, D, None, cuda, 1)
    want = _host(pool)
    g = torch.Generator().manual_seed(1)
    kh, vh = (_loud((204, H, D), g, torch.bfloat16).pin_memory() for _ in range(2))
    store_reference(kh.double(), want[0], want[2], prior, new, pages, ps)
    store_reference(vh.double(), want[1], want[3], prior, new, pages, ps)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        k, v = (torch.empty(204, H, D, dtype=torch.bfloat16, device=cuda) for _ in range(2))
        torch.cuda._sleep(10_000_000)
        k.copy_(kh, non_blocking=True), v.copy_(vh, non_blocking=True)
        yl.store_kv_cache_quant(k, v, pool, idx)
        back, _ = yl.load_kv_cache_quant(pool, idx.slot_mapping)
    stream.synchronize()
    for a, b in zip(_host(pool), want):
        assert torch.equal(a, b)
    s = idx.slot_mapping.cpu()
    assert torch.equal(back.cpu().double(), (want[0][s // ps, s % ps] * want[2][s // ps][..., None])
                       .to(torch.bfloat16).double())


@pytest.mark.parametrize("ps", [16, 17, 64, 128, 200])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_store_long_chunks(cuda, ps, dtype):
    """Chunks over whole pages of every mode's size, starting and ending inside one."""
    _store_case(cuda, [0, 3 * ps - 1, 5, ps], [4 * ps + 1, ps + 2, 2 * ps, 1], ps=ps, D=128, H=3, dtype=dtype, seed=ps)


@pytest.mark.parametrize("ps", [17, 64, 200])
def test_store_nonfinite_in_long_pages(cuda, ps):
    """An infinity and NaN in rows of different warps of one page; the other
    head, plane and pages are as without them."""
    H, D, P = 2, 64, 4
    n = 2 * ps
    x = torch.randn(n, H, D, generator=torch.Generator().manual_seed(ps)).to(torch.bfloat16)
    clean = x.clone()
    for t, d, bad in ((0, 1, float("inf")), (ps // 2, 2, float("nan")), (ps - 1, 3, float("-inf"))):
        x[t, 1, d], clean[t, 1, d] = bad, 0
    idx, pages = make_index([0], [n], ps, P, 1)
    pool, other = (yl.quant_kv_pool(P, ps, H, D, device=cuda) for _ in range(2))
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    yl.store_kv_cache_quant(clean.to(cuda), x.to(cuda), pool, idx, error_word=err)
    assert int(err.item()) == yl.DEVERR_NONFINITE
    yl.store_kv_cache_quant(clean.to(cuda), clean.to(cuda), other, idx)
    assert torch.equal(pool.v_scale, other.v_scale) and torch.equal(pool.k.float(), other.k.float())
    a, b, page = pool.v.float().cpu(), other.v.float().cpu(), pages[0][0]
    assert a[page, 0, 1, 1] == 448 and torch.isnan(a[page, ps // 2, 1, 2]) and a[page, ps - 1, 1, 3] == -448
    for t, d in ((0, 1), (ps // 2, 2), (ps - 1, 3)):
        a[page, t, 1, d] = 0
    assert torch.equal(a, b)


@pytest.mark.parametrize("count", [1, 31, 2500])
@pytest.mark.parametrize("H", [1, 8])
def test_load_counts(cuda, count, H):
    """From one slot to more than the grid holds, one slot named many times."""
    D, ps, P = 128, 16, 60
    pool = _filled_pool(P, ps, H, D, 2, cuda, 3)
    slots = torch.randint(0, P * ps, (count,), generator=torch.Generator().manual_seed(count))
    slots[:count // 2] = 77
    k, v = yl.load_kv_cache_quant(pool, slots.to(cuda))
    host = _host(pool)
    for got, x, s in ((k, host[0], host[2]), (v, host[1], host[3])):
        want = x[:, slots // ps, slots % ps] * s[:, slots // ps][..., None]
        assert torch.equal(got.cpu().double(), want.to(torch.bfloat16).double())


def test_pages_named_again_and_again(cuda):
    """A million tokens through a table that names 64 pages over and over: a
    decode step weighs every key as often as its page is named, so the result
    is the 64 pages' own.  Prefix sharing is the common case of it."""
    H, G, D, ps, P, named = 2, 4, 128, 16, 64, 1 << 16
    (k, v, ks, vs), (kx, vx) = _pool(P, ps, H, D, torch.bfloat16, "e4m3", cuda, 2)
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device=cuda)  # noqa: E731
    ids = torch.arange(P, dtype=torch.int32, device=cuda).repeat(named // P)
    idx = yl.BatchIndex(i32(0, named), ids, i32(ps), i32(0, 1), None)
    q = torch.randn(1, H * G, D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    got = _direct(q.to(cuda), k, v, ks, vs, idx)
    want, spread, reach = attention_reference(q, kx, vx, [P * ps - 1], [1], [list(range(P))])
    # fp32 sums, in parts of at most 2^8 steps of 16 tokens, each step off by 2^-23 of the sum so far, for the
    # products and for the sum of weights: 2^-14 in all; the bound is widened by 2^-13 of the spread
    bound_spread = spread * (1 + 2.0 ** -13 / HALF_STEP[torch.float16])
    _check(got, want, bound_spread, reach, torch.bfloat16, "e4m3", D)


@pytest.mark.parametrize("kv", ["e4m3", "16"])
def test_pool_past_32_bits(cuda, kv):
    """Pages whose first byte lies past 2^32: attention, store and read-back."""
    H, G, D, ps = 8, 2, 128, 16
    P = (1 << 32) // (H * D * ps * (1 if kv == "e4m3" else 2)) + 40
    prior, new = [100, 0], [1, 90]
    idx, pages = make_index(prior, new, ps, 20, 1)
    (k0, v0, ks0, vs0), (kx, vx) = _pool(20, ps, H, D, torch.bfloat16, kv, cuda, 2)

    def far(x):
        shape = (P, H, ps, D)
        big = torch.empty(shape, dtype=torch.uint8 if kv == "e4m3" else x.dtype, device=cuda).transpose(1, 2)
        big[P - 20:].copy_(x.view(torch.uint8) if kv == "e4m3" else x)
        return big.view(torch.float8_e4m3fn) if kv == "e4m3" else big

    def far_scale(s):
        big = torch.ones(P, H, device=cuda)
        big[P - 20:] = s
        return big

    idx = idx._replace(kv_indices=idx.kv_indices + (P - 20))
    pages = [[p + P - 20 for p in mine] for mine in pages]
    k, v = far(k0), far(v0)
    q = torch.randn(91, H * G, D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    near = [[p - (P - 20) for p in mine] for mine in pages]
    want, spread, reach = attention_reference(q, kx, vx, prior, new, near)
    ks, vs = (far_scale(ks0), far_scale(vs0)) if kv == "e4m3" else (None, None)
    got = _direct(q.to(cuda), k, v, ks, vs, idx)
    _check(got, want, spread, reach, torch.bfloat16, kv, D)
    if kv == "e4m3":
        pool = yl.QuantKVPool(k, v, ks, vs)
        rows = _loud((91, H, D), torch.Generator().manual_seed(5), torch.bfloat16)
        codes, scale = k0.cpu().double(), ks0.cpu().double()
        store_reference(rows.double(), codes, scale, prior, new, near, ps)
        yl.store_kv_cache_quant(rows.to(cuda), rows.to(cuda), pool, idx)
        assert torch.equal(pool.k[P - 20:].cpu().double(), codes) and torch.equal(pool.k_scale[P - 20:].cpu().double(), scale)
        slots = idx.slot_mapping + (P - 20) * ps
        back, _ = yl.load_kv_cache_quant(pool, slots)
        s = idx.slot_mapping.cpu()
        assert torch.equal(back.cpu().double(), (codes[s // ps, s % ps] * scale[s // ps][..., None]).to(torch.bfloat16).double())


def test_refusals_on_the_device(cuda):
    """Tensors of a wrong kind are refused before a launch, by name."""
    H, G, D, ps, P = 2, 2, 64, 16, 6
    pool = yl.quant_kv_pool(P, ps, H, D, device=cuda)
    idx, _ = make_index([0, 20], [1, 1], ps, P, 1)
    q = torch.zeros(2, H * G, D, dtype=torch.bfloat16, device=cuda)
    rows = q[:, :H].contiguous()
    scales = dict(k_scale=pool.k_scale, v_scale=pool.v_scale)
    bad = [
        lambda: yl.paged_attention(q.float(), pool.k, pool.v, idx, **scales),
        lambda: yl.paged_attention(q, pool.k, pool.v, idx),  # 8-bit pages without scales
        lambda: yl.paged_attention(q, q.new_zeros(P, ps, H, D), q.new_zeros(P, ps, H, D), idx, **scales),
        lambda: yl.paged_attention(q, pool.k, pool.v[:3], idx, **scales),
        lambda: yl.paged_attention(q[:, :3], pool.k, pool.v, idx, **scales),
        lambda: yl.paged_attention(q, pool.k, pool.v, idx, k_scale=pool.k_scale.double(), v_scale=pool.v_scale),
        lambda: yl.paged_attention(q, pool.k, pool.v, idx, window=-1, **scales),
        lambda: yl.paged_attention(q, pool.k, pool.v, idx, sm_scale=float("nan"), **scales),
        lambda: yl.paged_attention(q, pool.k, pool.v, idx, out=q.half(), **scales),
        lambda: yl.paged_attention(q, pool.k, pool.v, idx, out=q.transpose(1, 2).contiguous().transpose(1, 2), **scales),
        lambda: yl.paged_attention(q, pool.k, pool.v, idx._replace(kv_indptr=idx.kv_indptr.long()), **scales),
        lambda: yl.paged_attention(q, pool.k, pool.v, idx._replace(kv_last_page_len=idx.kv_last_page_len[:1]), **scales),
        lambda: yl.paged_attention(q, pool.k, pool.v, idx._replace(qo_indptr=idx.qo_indptr.cpu()), **scales),
        lambda: yl.store_kv_cache_quant(rows, rows.half(), pool, idx),
        lambda: yl.store_kv_cache_quant(rows, rows[:1], pool, idx),
        lambda: yl.store_kv_cache_quant(rows[:, :1], rows[:, :1], pool, idx),
        lambda: yl.store_kv_cache_quant(rows.float(), rows.float(), pool, idx),
        lambda: yl.store_kv_cache_quant(rows, rows, pool._replace(k=pool.k.view(torch.uint8)), idx),
        lambda: yl.store_kv_cache_quant(rows, rows, pool._replace(k_scale=pool.k_scale[:2]), idx),
        lambda: yl.load_kv_cache_quant(pool, torch.zeros(3, device=cuda)),
        lambda: yl.load_kv_cache_quant(pool, torch.zeros(3, dtype=torch.int64, device=cuda), dtype=torch.float32),
        lambda: yl.load_kv_cache_quant(pool, torch.zeros(3, dtype=torch.int64, device=cuda), out=(rows, rows)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((yl.PanicError, TypeError, ValueError)):
            call()
            pytest.fail(f"call {i} was accepted")
    torch.cuda.synchronize()
    assert not bool((pool.k.float() != 0).any())


@pytest.mark.parametrize("kv", ["e4m3", "16"])
@pytest.mark.parametrize("new", [1, 3, 150])
def test_queries_that_are_not_finite(cuda, kv, new):
    """NaN and infinities in some query heads: every other row is right (rows share when their
    reference moves, so not the same bits)."""
    H, G, D, ps, P, prior = 2, 4, 128, 16, 70, [130, 0, 400]
    idx, pages = make_index(prior, [new] * 3, ps, P, 1)
    (k, v, ks, vs), (kx, vx) = _pool(P, ps, H, D, torch.bfloat16, kv, cuda, 2)
    q = torch.randn(3 * new, H * G, D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    want, spread, reach = attention_reference(q, kx, vx, prior, [new] * 3, pages)
    q = q.to(cuda)
    bad = torch.zeros(3 * new, H * G, dtype=torch.bool, device=cuda)
    for row, head, d, value in ((0, 1, 0, float("nan")), (2 * new, 5, 17, float("inf")), (new, 6, 127, float("-inf"))):
        q[row, head, d], bad[row, head] = value, True
    got = _direct(q, k, v, ks, vs, idx)
    _check(got, want, spread, reach, torch.bfloat16, kv, D, rows=~bad.cpu())
    assert bool(torch.isnan(got[0, 1]).all())


@pytest.mark.parametrize("new", [1, 90])
@pytest.mark.parametrize("window,sinks", [(2 ** 31 - 1, 0), (5, 2 ** 31 - 1), (2 ** 31 - 1, 2 ** 31 - 1), (0, 9)])
def test_the_largest_windows(cuda, new, window, sinks):
    _run(cuda, [130, 0, 40], [new] * 3, H=1, G=2, D=64, window=window, sinks=sinks, dtype=torch.float16)


def test_a_batch_of_thousands(cuda):
    """More sequences than any block has threads, of up to four tokens; some
    with more query rows than the decode kernel takes."""
    new = [1 if i % 977 else 70 for i in range(9000)]
    prior = [(i * 7) % 4 for i in range(9000)]
    _run(cuda, prior, new, H=1, G=1, D=64, ps=4, pad=2, kv="16", dtype=torch.float16)
    _run(cuda, prior, new, H=1, G=1, D=64, ps=4, pad=2, hint=False)


def test_padded_batch_of_empty_sequences(cuda):
    """Rows of padding only: no page, an empty kv_indices, nothing written."""
    H, G, D, ps, P = 2, 2, 64, 16, 4
    pool = yl.quant_kv_pool(P, ps, H, D, device=cuda)
    i32 = lambda n: torch.zeros(n, dtype=torch.int32, device=cuda)  # noqa: E731
    idx = yl.BatchIndex(i32(3), i32(0), i32(2), i32(3), None)
    rows = torch.ones(5, H, D, dtype=torch.bfloat16, device=cuda)
    q = torch.ones(5, H * G, D, dtype=torch.bfloat16, device=cuda)
    err, out = i32(1), torch.full_like(q, 7.0)
    yl.store_kv_cache_quant(rows, rows, pool, idx, error_word=err)
    _direct(q, pool.k, pool.v, pool.k_scale, pool.v_scale, idx, out=out, error_word=err)
    assert int(err.item()) == 0 and not bool((pool.k.float() != 0).any()) and bool((out == 7.0).all())
    assert bool((pool.k_scale == 1).all())


@pytest.mark.parametrize("new", [1, 100])
def test_queries_as_heads_major_memory(cuda, new):
    """q and out in [heads, tokens, D] memory, the strides of rows below those of heads."""
    H, G, D, ps, P = 2, 4, 128, 16, 60
    prior = [200, 33]
    idx, pages = make_index(prior, [new, new], ps, P, 1)
    (k, v, ks, vs), (kx, vx) = _pool(P, ps, H, D, torch.bfloat16, "e4m3", cuda, 2)
    q = torch.randn(2 * new, H * G, D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    mem = q.to(cuda).transpose(0, 1).contiguous().transpose(0, 1)
    out = torch.zeros_like(q.transpose(0, 1).contiguous(), device=cuda).transpose(0, 1)
    got = _direct(mem, k, v, ks, vs, idx, out=out)
    want, spread, reach = attention_reference(q, kx, vx, prior, [new, new], pages)
    _check(got, want, spread, reach, torch.bfloat16, "e4m3", D)


@pytest.mark.parametrize("kv", ["e4m3", "16"])
def test_scores_that_fall_and_rise(cuda, kv):
    """Keys whose loudness grows along the sequence, then falls: the reference
    moves at nearly every tile, in decode and in prefill."""
    H, G, D, ps, P = 1, 4, 128, 16, 40
    for prior, new in (([600], [1]), ([300], [301])):
        idx, pages = make_index(prior, new, ps, P, 1)
        (k, v, ks, vs), (kx, vx) = _pool(P, ps, H, D, torch.float16, kv, cuda, 2)
        for j, page in enumerate(pages[0]):
            f = 2.0 ** (min(j, 37 - j) // 6 - 2)
            if kv == "e4m3":
                ks[page] *= f
            else:
                k[page] *= f
            kx[page] *= f
        q = torch.randn(sum(new), H * G, D, generator=torch.Generator().manual_seed(3)).to(torch.float16)
        got = _direct(q.to(cuda), k, v, ks, vs, idx)
        want, spread, reach = attention_reference(q, kx, vx, prior, new, pages)
        _check(got, want, spread, reach, torch.float16, kv, D)
