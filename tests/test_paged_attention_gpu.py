"""yl.paged_attention (yl_paged_attention) against 64-bit attention on the host:
decode, prefill and mixed batches, 16-bit and 8-bit pools, windows with first
tokens, page sizes, head layouts, ragged and empty sequences, and what the call
must leave alone.  The bound of each element counts the roundings (see
_attnutil.attention_bound)."""
import numpy as np
import pytest
import torch

import yllang_b200 as yl
from _attnutil import attention_bound, attention_reference, make_index

pytestmark = pytest.mark.gpu

NAN8 = 0x7F


def _pool(P, ps, H, D, dtype, kv, dev, seed, head_major=True):
    """(k, v, k_scale, v_scale) on the device and the values they stand for on the host."""
    g = torch.Generator().manual_seed(seed)
    shape = (P, H, ps, D) if head_major else (P, ps, H, D)
    out, values = [], []
    for _ in range(2):
        x = torch.randn(shape, generator=g)
        if kv == "e4m3":
            x = (x * 64).clamp(-448, 448).to(torch.float8_e4m3fn)
            s = torch.exp2(torch.randint(-9, -3, (P, H), generator=g).float())
            x = x.transpose(1, 2) if head_major else x
            values.append(x.to(torch.float64) * s.double()[:, None, :, None])
            d = torch.empty(shape, dtype=torch.uint8, device=dev)
            d = d.transpose(1, 2) if head_major else d
            d.copy_(x.view(torch.uint8).to(dev))
            out.append((d.view(torch.float8_e4m3fn), s.to(dev)))
        else:
            x = x.to(dtype)
            x = x.transpose(1, 2) if head_major else x
            values.append(x.double())
            d = torch.empty(shape, dtype=dtype, device=dev)
            d = d.transpose(1, 2) if head_major else d
            d.copy_(x.to(dev))
            out.append((d, None))
    return (out[0][0], out[1][0], out[0][1], out[1][1]), values


def _check(got, want, spread, reach, dtype, kv, D, rows=slice(None)):
    weights = torch.bfloat16 if dtype == torch.bfloat16 and kv == "16" else torch.float16
    bound = attention_bound(want, spread, reach, dtype, weights, D)
    err = (got.double().cpu() - want).abs()
    over = (err - bound)[rows]
    assert torch.isfinite(got[rows]).all()
    assert float(over.max() if over.numel() else 0) <= 0, (
        f"largest excess {float(over.max())}, worst ratio {float((err / bound)[rows].max()):.2f}")


def _run(cuda, prior, new, *, H=2, G=4, D=128, ps=16, dtype=torch.bfloat16, kv="e4m3", window=0, sinks=0, seed=0,
         head_major=True, hint=True, pad=0, scale=None, spare_pages=5, fill=None):
    P = int(sum(-(-(a + b) // ps) for a, b in zip(prior, new))) + spare_pages
    idx, pages = make_index(prior, new, ps, P, seed)
    (k, v, ks, vs), (kx, vx) = _pool(P, ps, H, D, dtype, kv, cuda, seed + 1, head_major)
    N = sum(new) + pad
    q = (torch.randn(N, H * G, D, generator=torch.Generator().manual_seed(seed + 2)) * 1.5).to(dtype)
    out = torch.full((N, H * G, D), 7.0, dtype=dtype, device=cuda)
    if fill is not None:
        fill(k, v, pages)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    got = yl.paged_attention(q.to(cuda), k, v, idx, k_scale=ks, v_scale=vs, window=window, sinks=sinks, sm_scale=scale,
                             max_new_len=max(new, default=0) if hint else 0, out=out, error_word=err)
    torch.cuda.synchronize()
    assert got is out and int(err.item()) == 0
    n = sum(new)
    want, spread, reach = attention_reference(q[:n], kx, vx, prior, new, pages, window, sinks, scale)
    _check(got[:n], want, spread, reach, dtype, kv, D)
    assert bool((got[n:] == 7.0).all())
    return got


MIXED = ([0, 1, 15, 16, 17, 63, 64, 130, 300, 0], [1, 1, 1, 1, 1, 1, 1, 1, 1, 0])
CHUNKS = ([0, 37, 150, 0, 1, 64, 300], [120, 1, 16, 3, 33, 0, 5])


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kv", ["e4m3", "16"])
@pytest.mark.parametrize("batch", [MIXED, CHUNKS], ids=["decode", "chunks"])
def test_types_and_head_dims(cuda, D, dtype, kv, batch):
    _run(cuda, *batch, D=D, dtype=dtype, kv=kv)


@pytest.mark.parametrize("ps", [1, 5, 8, 32, 64, 128, 200])
@pytest.mark.parametrize("kv", ["e4m3", "16"])
@pytest.mark.parametrize("batch", [MIXED, CHUNKS], ids=["decode", "chunks"])
def test_page_sizes(cuda, ps, kv, batch):
    _run(cuda, *batch, ps=ps, kv=kv, H=3, G=2, D=64, head_major=kv == "e4m3")


@pytest.mark.parametrize("G", [1, 3, 5, 7, 8, 16, 24, 80])
@pytest.mark.parametrize("new", [1, 2, 4, 9])
def test_groups(cuda, G, new):
    """Query heads per KV head and new tokens around the 16-row and 64-row tiles."""
    _run(cuda, [40, 0, 129], [new, new, new], H=1 + (G < 8), G=G, D=64, dtype=torch.float16)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (7, 0), (64, 4), (64, 70), (100, 16), (1000, 4), (128, 64)])
@pytest.mark.parametrize("kv", ["e4m3", "16"])
@pytest.mark.parametrize("batch", [MIXED, CHUNKS], ids=["decode", "chunks"])
def test_windows(cuda, window, sinks, kv, batch):
    _run(cuda, *batch, window=window, sinks=sinks, kv=kv, H=2, G=2)


@pytest.mark.parametrize("kv", ["e4m3", "16"])
def test_long_sequences(cuda, kv):
    """Sequences over many units of work beside short ones: the parts of one
    result lie in many blocks."""
    _run(cuda, [4999, 3, 1200, 2047], [1, 1, 1, 2], H=1, G=4, kv=kv, dtype=torch.bfloat16, ps=16)


@pytest.mark.parametrize("kv", ["e4m3", "16"])
def test_long_prompts(cuda, kv):
    _run(cuda, [0, 400, 0], [517, 260, 129], H=2, G=2, kv=kv, window=0)
    _run(cuda, [0, 400, 0], [517, 260, 129], H=1, G=3, kv=kv, window=150, sinks=5)


@pytest.mark.parametrize("hint", [False, True])
def test_hint_changes_nothing(cuda, hint):
    got = _run(cuda, [5, 90, 33], [1, 40, 2], hint=hint, seed=3)
    again = _run(cuda, [5, 90, 33], [1, 40, 2], hint=hint, seed=3)
    assert torch.equal(got, again)


def test_many_sequences(cuda):
    """More sequences than threads of a block, some of them empty."""
    rng = np.random.default_rng(5)
    new = rng.integers(0, 2, 700).tolist()
    prior = [int(x) * n for x, n in zip(rng.integers(0, 40, 700), new)]
    _run(cuda, prior, new, H=2, G=2, D=64, ps=8)


def test_rows_behind_the_last_sequence_stay(cuda):
    _run(cuda, [3, 20], [1, 1], pad=9)
    _run(cuda, [3, 20], [50, 1], pad=70)
    _run(cuda, [3, 20], [1, 1], pad=9, hint=False)


@pytest.mark.parametrize("kv", ["e4m3", "16"])
@pytest.mark.parametrize("new", [1, 3, 30])
def test_unseen_places_hold_nan(cuda, kv, new):
    """Every slot that no query may see holds NaN (codes, and infinities in a
    16-bit pool): behind the ends, in other pages, before the window, and, for
    each query, in the positions after it."""
    prior, ps, window, sinks = [37, 100, 0], 16, 20, 3

    def fill(k, v, pages):
        seen = torch.zeros(k.shape[:2], dtype=torch.bool)
        for p, mine in zip(prior, pages):
            for t in range(new):
                for j in range(p + t + 1):
                    if j > p + t - window or j < sinks:
                        seen[mine[j // ps], j % ps] = True
        hide = ~seen.to(k.device)
        for x in (k, v):
            if kv == "e4m3":
                x.view(torch.uint8)[hide] = NAN8
            else:
                x[hide] = float("nan")

    _run(cuda, prior, [new] * 3, kv=kv, window=window, sinks=sinks, fill=fill)


@pytest.mark.parametrize("kv,bad", [("e4m3", float("nan")), ("16", float("nan")), ("16", float("inf"))])
@pytest.mark.parametrize("new", [2, 12, 40])
def test_values_after_a_query_do_not_reach_it(cuda, kv, bad, new):
    """K and V of the last new token hold NaN or infinities: every earlier
    query's result is as without them, the last one's is not finite."""
    H, G, D, ps, prior = 2, 2, 128, 16, 21
    P = 10
    idx, pages = make_index([prior], [new], ps, P, 1)
    (k, v, ks, vs), (kx, vx) = _pool(P, ps, H, D, torch.bfloat16, kv, cuda, 2)
    q = torch.randn(new, H * G, D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    pos = prior + new - 1
    page, slot = pages[0][pos // ps], pos % ps
    want, spread, reach = attention_reference(q, kx, vx, [prior], [new], pages)
    for which in (k, v):
        keep = which[page, slot].clone()
        if kv == "e4m3":
            which.view(torch.uint8)[page, slot] = NAN8
        else:
            which[page, slot] = bad
        got = yl.paged_attention(q.to(cuda), k, v, idx, k_scale=ks, v_scale=vs)
        _check(got, want, spread, reach, torch.bfloat16, kv, D, rows=slice(0, new - 1))
        assert not bool(torch.isfinite(got[new - 1]).all())
        which[page, slot] = keep


def test_pages_outside_the_window_are_not_read(cuda):
    """Entries of pages that no query sees may hold anything."""
    H, G, D, ps, window, sinks = 2, 4, 128, 16, 40, 4
    for new in (1, 2, 40):
        prior, P = [200, 77], 40
        idx, pages = make_index(prior, [new, new], ps, P, 4)
        (k, v, ks, vs), (kx, vx) = _pool(P, ps, H, D, torch.float16, "e4m3", cuda, 5)
        q = torch.randn(2 * new, H * G, D, generator=torch.Generator().manual_seed(6)).to(torch.float16)
        ids = idx.kv_indices.cpu()
        at = 0
        for p in prior:
            n = -(-(p + new) // ps)
            for j in range(n):
                first, last = j * ps, j * ps + ps - 1
                if last <= p - window and first >= sinks:
                    ids[at + j] = 1 << 30
            at += n
        idx = idx._replace(kv_indices=ids.to(cuda))
        err = torch.zeros(1, dtype=torch.int32, device=cuda)
        got = yl.paged_attention(q.to(cuda), k, v, idx, k_scale=ks, v_scale=vs, window=window, sinks=sinks,
                                 error_word=err)
        assert int(err.item()) == 0
        want, spread, reach = attention_reference(q, kx, vx, prior, [new, new], pages, window, sinks)
        _check(got, want, spread, reach, torch.float16, "e4m3", D)


def test_strided_rows_and_token_major_pool(cuda):
    """q as a view of a packed projection, o as a view of a wider buffer, the
    pool as the framework's 16-bit token-major one."""
    H, G, D, ps, P = 2, 4, 64, 16, 30
    prior, new = [50, 0, 131], [1, 60, 2]
    idx, pages = make_index(prior, new, ps, P, 7)
    (k, v, _, _), (kx, vx) = _pool(P, ps, H, D, torch.bfloat16, "16", cuda, 8, head_major=False)
    N = sum(new)
    packed = torch.randn(N, (H * G + 2 * H) * D, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16).to(cuda)
    q = packed[:, :H * G * D].view(N, H * G, D)
    wide = torch.zeros(N, H * G, 2 * D, dtype=torch.bfloat16, device=cuda)
    got = yl.paged_attention(q, k, v, idx, out=wide[..., :D])
    want, spread, reach = attention_reference(q.cpu(), kx, vx, prior, new, pages)
    _check(got, want, spread, reach, torch.bfloat16, "16", D)
    assert not bool(wide[..., D:].any())


def test_scale_argument_and_loud_queries(cuda):
    """Scores far apart (one key takes all the weight) and a given sm_scale;
    queries of very large and very small rows over an 8-bit pool."""
    _run(cuda, [70, 9], [1, 20], scale=2.0)
    H, G, D, ps, P = 1, 4, 128, 16, 12
    idx, pages = make_index([90], [1], ps, P, 1)
    (k, v, ks, vs), (kx, vx) = _pool(P, ps, H, D, torch.bfloat16, "e4m3", cuda, 2)
    q = torch.randn(1, G, D, generator=torch.Generator().manual_seed(3))
    q = (q * torch.tensor([1e30, 1e-30, 3e4, 0.0])[None, :, None]).to(torch.bfloat16)
    for scale, rows in ((1e-30, [0, 1, 3]), (1.0, [1, 3]), (1e-5, [2])):
        got = yl.paged_attention(q.to(cuda), k, v, idx, k_scale=ks, v_scale=vs, sm_scale=scale)
        want, spread, reach = attention_reference(q, kx, vx, [90], [1], pages, sm_scale=scale)
        for r in rows:
            _check(got[:, r], want[:, r], spread[:, r], reach[:, r], torch.bfloat16, "e4m3", D)


def test_value_scales_far_apart(cuda):
    """Pages whose V scales differ by 2^30 and more: a small page that takes
    the weight keeps its precision beside a large one that takes little."""
    H, G, D, ps, P = 1, 2, 64, 16, 8
    for new in (1, 40):
        idx, pages = make_index([0], [100], ps, P, 1)
        idx = idx._replace(qo_indptr=torch.tensor([0, new], dtype=torch.int32, device=cuda))
        (k, v, ks, vs), (kx, vx) = _pool(P, ps, H, D, torch.float16, "e4m3", cuda, 2)
        factor = torch.ones(P)
        factor[pages[0][1]] = 2.0 ** 12
        factor[pages[0][2]] = 2.0 ** -30
        factor[pages[0][3]] = 0.0
        vs.mul_(factor.to(cuda)[:, None])
        vx = vx * factor.double()[:, None, None, None]
        q = torch.randn(new, H * G, D, generator=torch.Generator().manual_seed(3)).to(torch.float16)
        got = yl.paged_attention(q.to(cuda), k, v, idx, k_scale=ks, v_scale=vs)
        want, spread, reach = attention_reference(q, kx, vx, [100 - new], [new], pages)
        _check(got, want, spread, reach, torch.float16, "e4m3", D)


def test_replayed_graph_follows_the_lengths(cuda):
    """A captured call reads lengths, pages and queries anew at each replay."""
    H, G, D, ps, P, B = 2, 4, 128, 16, 200, 3
    (k, v, ks, vs), (kx, vx) = _pool(P, ps, H, D, torch.bfloat16, "e4m3", cuda, 2)
    first, _ = make_index([700, 3, 40], [1, 1, 1], ps, P, 1, spare=40)
    q = torch.zeros(B, H * G, D, dtype=torch.bfloat16, device=cuda)
    out = torch.zeros_like(q)
    call = lambda: yl.paged_attention(q, k, v, first, k_scale=ks, v_scale=vs, max_new_len=1, out=out)  # noqa: E731
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for seed, prior in enumerate([[700, 3, 40], [0, 900, 16], [64, 63, 62]]):
        idx, pages = make_index(prior, [1, 1, 1], ps, P, seed)
        for name in ("kv_indptr", "kv_last_page_len", "qo_indptr"):
            getattr(first, name).copy_(getattr(idx, name))
        first.kv_indices[:idx.kv_indices.numel()].copy_(idx.kv_indices)
        qh = torch.randn(B, H * G, D, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)
        q.copy_(qh)
        graph.replay()
        torch.cuda.synchronize()
        want, spread, reach = attention_reference(qh, kx, vx, prior, [1, 1, 1], pages)
        _check(out, want, spread, reach, torch.bfloat16, "e4m3", D)


def test_two_streams_at_once(cuda):
    """Calls on two streams, each with the workspace it allocates, and results
    the same as one after the other."""
    H, G, D, ps, P = 4, 4, 128, 16, 600
    idx, _ = make_index([4000, 100, 2500], [1, 1, 1], ps, P, 1)
    (k, v, ks, vs), _ = _pool(P, ps, H, D, torch.bfloat16, "e4m3", cuda, 2)
    qs = [torch.randn(3, H * G, D, device=cuda, generator=torch.Generator(device=cuda).manual_seed(i)).to(torch.bfloat16)
          for i in range(2)]
    alone = [yl.paged_attention(q, k, v, idx, k_scale=ks, v_scale=vs, max_new_len=1) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i in range(2):
            got[i].append(yl.paged_attention(qs[i], k, v, idx, k_scale=ks, v_scale=vs, max_new_len=1,
                                             stream=streams[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for o in got[i]:
            assert torch.equal(o, alone[i])


def test_device_checks(cuda):
    H, G, D, ps, P = 2, 4, 128, 16, 20
    (k, v, ks, vs), (kx, vx) = _pool(P, ps, H, D, torch.bfloat16, "e4m3", cuda, 2)

    def call(idx, n, **kw):
        err = torch.zeros(1, dtype=torch.int32, device=cuda)
        q = torch.ones(n, H * G, D, dtype=torch.bfloat16, device=cuda)
        out = torch.full_like(q, 7.0)
        yl.paged_attention(q, k, v, idx, k_scale=ks, v_scale=vs, out=out, error_word=err, **kw)
        torch.cuda.synchronize()
        return int(err.item()), out

    for new in (1, 40):
        prior = [60, 30]
        idx, pages = make_index(prior, [new, new], ps, P, 1)
        n = 2 * new
        # a page id outside the pool: that page counts as not seen
        ids = idx.kv_indices.clone()
        ids[1] = P
        bits, out = call(idx._replace(kv_indices=ids), n)
        assert bits == yl.DEVERR_PAGE_RANGE
        good = call(idx, n)[1]
        assert torch.equal(out[new:], good[new:]) and bool(torch.isfinite(out).all())
        # entries past the capacity
        short = idx._replace(kv_indices=idx.kv_indices[:5].contiguous())
        bits, out = call(short, n)
        assert bits == yl.DEVERR_INDICES_CAP and bool(torch.isfinite(out).all())
        # rows past q
        bits, out = call(idx, n - 1)
        assert bits == yl.DEVERR_TOKEN_COUNT
        # more new tokens than the hint says: those rows are left alone
        if new > 1:
            bits, out = call(idx, n, max_new_len=new - 1)
            assert bits == yl.DEVERR_TOKEN_COUNT and bool((out == 7.0).all())
    # more new tokens than the sequence has: rows before its first position are zero
    idx, pages = make_index([0], [5], ps, P, 1)
    idx = idx._replace(qo_indptr=torch.tensor([0, 8], dtype=torch.int32, device=cuda))
    bits, out = call(idx, 8)
    assert bits == 0 and not bool(out[:3].any()) and bool(out[3:].any())
    # a length of zero
    empty = yl.BatchIndex(*[torch.zeros(n, dtype=torch.int32, device=cuda) for n in (2, 1, 1)],
                          torch.tensor([0, 1], dtype=torch.int32, device=cuda), None)
    bits, out = call(empty, 1)
    assert bits == 0 and not bool(out.any())


def test_no_work_is_a_no_op(cuda):
    k = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16, device=cuda)
    idx, _ = make_index([], [], 16, 4)
    q = torch.zeros(0, 4, 64, dtype=torch.bfloat16, device=cuda)
    assert yl.paged_attention(q, k, k, idx).shape == (0, 4, 64)
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16, device=cuda)
    out = torch.full_like(q, 7.0)
    yl.paged_attention(q, k, k, idx, out=out)
    assert bool((out == 7.0).all())


def test_workspace(cuda):
    H, G, D, ps, P = 2, 4, 128, 16, 40
    idx, pages = make_index([300, 200], [1, 1], ps, P, 1)
    (k, v, ks, vs), _ = _pool(P, ps, H, D, torch.bfloat16, "e4m3", cuda, 2)
    q = torch.randn(2, H * G, D, device=cuda).to(torch.bfloat16)
    need = yl.paged_attention_workspace(q, k, v, idx, k_scale=ks, v_scale=vs)
    want = yl.paged_attention(q, k, v, idx, k_scale=ks, v_scale=vs)
    dirty = torch.full((need,), 0xFF, dtype=torch.uint8, device=cuda)
    assert torch.equal(want, yl.paged_attention(q, k, v, idx, k_scale=ks, v_scale=vs, workspace=dirty))
    with pytest.raises(yl.PanicError, match="workspace"):
        yl.paged_attention(q, k, v, idx, k_scale=ks, v_scale=vs, workspace=dirty[:need - 1].contiguous())
