"""The 8-bit pool on the GPU: yl.store_kv_cache_quant and yl.load_kv_cache_quant
against a 64-bit restatement.  Scales are powers of two and each code is
rounded once, so codes and scales are compared exactly; a read-back value is
the exact product rounded once, compared exactly too."""
import numpy as np
import pytest
import torch

import yllang_b200 as yl
from _attnutil import make_index, page_scale, store_reference

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


def _filled_pool(P, ps, H, D, L, dev, seed, token_major=False):
    """A pool with contents; token_major: [.., ps, H, D] in memory."""
    g = torch.Generator().manual_seed(seed)
    pool = yl.quant_kv_pool(P, ps, H, D, L, device=dev)
    if token_major:
        pool = pool._replace(k=torch.zeros(pool.k.shape, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn),
                             v=torch.zeros(pool.k.shape, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn))
    for t in (pool.k, pool.v):
        x = (torch.randn(t.shape, generator=g) * 90).clamp(-448, 448).to(torch.float8_e4m3fn)
        t.view(torch.uint8).copy_(x.view(torch.uint8).to(dev))
    for t in (pool.k_scale, pool.v_scale):
        t.copy_(torch.exp2(torch.randint(-9, -3, t.shape, generator=g).float()))
    return pool


def _host(pool):
    return [t.cpu().to(torch.float64) for t in (pool.k, pool.v)] + [t.cpu().double() for t in (pool.k_scale, pool.v_scale)]


def _loud(shape, g, dtype):
    """Rows whose largest elements differ by powers of two up to 2^6."""
    x = torch.randn(shape, generator=g)
    return (x * torch.exp2(torch.randint(-3, 4, (*shape[:-1], 1), generator=g).float())).to(dtype)


def _store_case(cuda, prior, new, *, H=2, D=128, ps=16, L=None, dtype=torch.bfloat16, seed=0, token_major=False, pad=0):
    P = int(sum(-(-(a + b) // ps) for a, b in zip(prior, new))) + 3
    idx, pages = make_index(prior, new, ps, P, seed)
    pool = _filled_pool(P, ps, H, D, L, cuda, seed + 1, token_major)
    g = torch.Generator().manual_seed(seed + 2)
    N, lead = sum(new), () if L is None else (L,)
    k, v = (_loud((*lead, N + pad, H, D), g, dtype) for _ in range(2))
    want = _host(pool)
    for layer in range(L or 1):
        at = (lambda t: t) if L is None else (lambda t: t[layer])  # noqa: B023
        store_reference(at(k).double(), at(want[0]), at(want[2]), prior, new, pages, ps)
        store_reference(at(v).double(), at(want[1]), at(want[3]), prior, new, pages, ps)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    yl.store_kv_cache_quant(k.to(cuda).reshape(*lead, N + pad, H * D), v.to(cuda), pool, idx, error_word=err)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    for got, w, name in zip(_host(pool), want, ("k", "v", "k_scale", "v_scale")):
        assert torch.equal(got, w), f"{name}: {int((got != w).sum())} of {w.numel()} differ"


DECODE = ([0, 1, 15, 16, 31, 47, 5, 200], [1] * 8)
RAGGED = ([0, 7, 16, 31, 0, 64, 3], [50, 1, 16, 2, 1, 0, 13])


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch", [DECODE, RAGGED], ids=["decode", "ragged"])
def test_store_types_and_head_dims(cuda, D, dtype, batch):
    _store_case(cuda, *batch, D=D, dtype=dtype, seed=D)


@pytest.mark.parametrize("ps", [1, 2, 5, 8, 17, 32, 64, 100])
@pytest.mark.parametrize("batch", [DECODE, RAGGED], ids=["decode", "ragged"])
def test_store_page_sizes(cuda, ps, batch):
    _store_case(cuda, *batch, ps=ps, D=64, H=3, seed=ps)


@pytest.mark.parametrize("H", [1, 2, 3, 5, 8])
@pytest.mark.parametrize("L", [None, 1, 3, 9])
def test_store_heads_and_layers(cuda, H, L):
    _store_case(cuda, [0, 21, 16], [33, 1, 1], H=H, L=L, D=64, seed=H)
    _store_case(cuda, [9, 21, 16], [1, 1, 1], H=H, L=L, D=128, seed=H)


def test_store_token_major_pool_and_padding_rows(cuda):
    _store_case(cuda, *RAGGED, token_major=True, pad=7)


def test_store_many_sequences(cuda):
    rng = np.random.default_rng(3)
    new = rng.integers(0, 3, 1500).tolist()
    prior = rng.integers(0, 30, 1500).tolist()
    _store_case(cuda, prior, new, H=1, D=64, ps=8)


def test_a_page_filled_token_by_token(cuda):
    """Sixteen steps of one token that grows louder: each step gives the
    restated codes, and the scale follows the loudest token so far."""
    H, D, ps, P = 2, 64, 16, 2
    pool = yl.quant_kv_pool(P, ps, H, D, device=cuda)
    want = _host(pool)
    g = torch.Generator().manual_seed(0)
    loudest = torch.zeros(H)
    for t in range(ps):
        idx, pages = make_index([t], [1], ps, P, 3)
        k, v = ((torch.randn(1, H, D, generator=g) * 2.0 ** (t // 3)).to(torch.bfloat16) for _ in range(2))
        yl.store_kv_cache_quant(k.to(cuda), v.to(cuda), pool, idx)
        store_reference(k.double(), want[0], want[2], [t], [1], pages, ps)
        store_reference(v.double(), want[1], want[3], [t], [1], pages, ps)
        for a, b in zip(_host(pool), want):
            assert torch.equal(a, b)
        loudest = torch.maximum(loudest, k[0].float().abs().amax(-1))
        assert pool.k_scale[pages[0][0]].tolist() == [page_scale(float(x)) for x in loudest]


@pytest.mark.parametrize("dtype", DTYPES)
def test_store_extremes(cuda, dtype):
    """Zeros, the smallest and largest magnitudes, exact powers of two around
    448, and signed zeros: scale exponents at both clamps."""
    H, D, ps, P = 1, 64, 4, 8
    f = torch.finfo(dtype)
    rows = torch.zeros(7, H, D, dtype=dtype)
    rows[1, 0, 3] = f.tiny
    rows[2, 0, :2] = torch.tensor([f.max, -1.0])
    rows[3, 0, :2] = torch.tensor([448.0, -448.0])
    rows[4, 0, 0] = float(torch.tensor(448.0).to(dtype)) * (1 + f.eps)
    rows[5, 0, :3] = torch.tensor([-0.0, 2.0 ** -10, 1.0])
    rows[6, 0, 0] = f.smallest_normal * f.eps  # subnormal
    prior, new = [0] * 7, [1] * 7
    idx, pages = make_index(prior, new, ps, P, 1)
    pool = yl.quant_kv_pool(P, ps, H, D, device=cuda)
    want = _host(pool)
    for x, s in ((want[0], want[2]), (want[1], want[3])):
        store_reference(rows.double(), x, s, prior, new, pages, ps)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    yl.store_kv_cache_quant(rows.to(cuda), rows.to(cuda), pool, idx, error_word=err)
    assert int(err.item()) == 0
    for a, b in zip(_host(pool), want):
        assert torch.equal(a, b)
    k, _ = yl.load_kv_cache_quant(pool, idx.slot_mapping, dtype=dtype)
    assert bool(torch.isfinite(k).all())  # the largest value comes back finite


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("count", [1, 3, 40])
def test_store_nonfinite(cuda, dtype, count):
    """The scale comes from the finite elements; infinities become the largest
    code, NaN e4m3's NaN, the bit is set, and other heads are as ever."""
    H, D, ps, P = 2, 128, 64, 3
    g = torch.Generator().manual_seed(count)
    x = torch.randn(count, H, D, generator=g).to(dtype)
    clean = x.clone()
    x[0, 1, 5], x[count - 1, 1, 6], x[0, 1, 7] = float("inf"), float("-inf"), float("nan")
    clean[0, 1, 5] = clean[count - 1, 1, 6] = clean[0, 1, 7] = 0
    idx, pages = make_index([0], [count], ps, P, 1)
    pool, other = (yl.quant_kv_pool(P, ps, H, D, device=cuda) for _ in range(2))
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    yl.store_kv_cache_quant(x.to(cuda), clean.to(cuda), pool, idx, error_word=err)
    assert int(err.item()) == yl.DEVERR_NONFINITE
    yl.store_kv_cache_quant(clean.to(cuda), clean.to(cuda), other, idx)
    a, b = pool.k.float().cpu(), other.k.float().cpu()
    page = pages[0][0]
    assert torch.equal(pool.k_scale, other.k_scale) and torch.equal(pool.v.float(), other.v.float())
    assert a[page, 0, 1, 5] == 448 and a[page, count - 1, 1, 6] == -448 and torch.isnan(a[page, 0, 1, 7])
    for t, d in ((0, 5), (count - 1, 6), (0, 7)):
        a[page, t, 1, d] = 0
    assert torch.equal(a, b)


def test_store_bad_held_scale(cuda):
    """A held page whose scale is no positive finite number: the bit, the new
    tokens' own scale, and the earlier codes as they were."""
    H, D, ps, P = 4, 64, 8, 2
    idx, pages = make_index([3], [2], ps, P, 1)
    pool = _filled_pool(P, ps, H, D, None, cuda, 2)
    page = pages[0][0]
    pool.k_scale[page] = torch.tensor([float("nan"), 0.0, -1.0, float("inf")], device=cuda)
    before = pool.k[page, :3].float().cpu()
    k = torch.randn(2, H, D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    yl.store_kv_cache_quant(k.to(cuda), k.to(cuda), pool, idx, error_word=err)
    assert int(err.item()) == yl.DEVERR_SCALE
    assert pool.k_scale[page].tolist() == [page_scale(float(k[:, h].float().abs().max())) for h in range(H)]
    assert torch.equal(pool.k[page, :3].float().cpu(), before)


def test_store_checks_on_the_device(cuda):
    H, D, ps, P = 2, 64, 8, 12

    def call(idx, n):
        pool = yl.quant_kv_pool(P, ps, H, D, device=cuda)
        err = torch.zeros(1, dtype=torch.int32, device=cuda)
        k = torch.ones(n, H, D, dtype=torch.bfloat16, device=cuda)
        yl.store_kv_cache_quant(k, k, pool, idx, error_word=err)
        return int(err.item()), int((pool.k.float() != 0).any(-1).any(-1).sum())

    for prior, new in (([4, 0], [1, 1]), ([4, 0], [20, 9])):
        n = sum(new)
        idx, pages = make_index(prior, new, ps, P, 1)
        assert call(idx, n) == (0, n)
        ids = idx.kv_indices.clone()
        ids[0] = P
        bits, written = call(idx._replace(kv_indices=ids), n)
        assert bits == yl.DEVERR_PAGE_RANGE and written < n
        ids[0] = -1
        assert call(idx._replace(kv_indices=ids), n)[0] == yl.DEVERR_PAGE_RANGE
        bits, written = call(idx._replace(kv_indices=idx.kv_indices[:1].contiguous()), n)
        assert bits == yl.DEVERR_INDICES_CAP and written < n
        assert call(idx, n + 5) == (0, n)  # rows behind the last sequence
        bits, written = call(idx, n - 1)
        assert written == n - 1 and bits in (0, yl.DEVERR_TOKEN_COUNT)
    # more new tokens than the sequence's pages hold: the last ones are those stored
    idx, pages = make_index([0], [5], ps, P, 1)
    idx = idx._replace(qo_indptr=torch.tensor([0, 9], dtype=torch.int32, device=cuda))
    assert call(idx, 9) == (yl.DEVERR_ROW_OVERFLOW, 5)


def test_store_debug_mode_names_the_bits(cuda, monkeypatch):
    monkeypatch.setattr(yl.ops, "CHECK_DEVICE_ERRORS", True)
    idx, pages = make_index([0], [1], 4, 2, 1)
    pool = yl.quant_kv_pool(2, 4, 1, 64, device=cuda)
    k = torch.full((1, 1, 64), float("nan"), dtype=torch.bfloat16, device=cuda)
    with pytest.raises(yl.PanicError, match="NONFINITE"):
        yl.store_kv_cache_quant(k, k, pool, idx)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("L", [None, 2])
@pytest.mark.parametrize("slot_dtype", [torch.int32, torch.int64])
def test_load(cuda, D, dtype, L, slot_dtype):
    """Repeated, skipped and out-of-range slots; values beyond fp16's range."""
    H, ps, P = 3, 5, 23
    pool = _filled_pool(P, ps, H, D, L, cuda, D)
    if dtype == torch.float16:
        pool.k_scale.mul_(2.0 ** 14)  # some values pass 65504
    g = torch.Generator().manual_seed(1)
    slots = torch.randint(0, P * ps, (301,), generator=g)
    slots[7], slots[100], slots[300] = -1, P * ps, -5
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    k, v = yl.load_kv_cache_quant(pool, slots.to(slot_dtype).to(cuda), dtype=dtype, error_word=err)
    assert int(err.item()) == yl.DEVERR_SLOT_RANGE
    host = _host(pool)
    good = (slots >= 0) & (slots < P * ps)
    at = torch.where(good, slots, 0)
    for got, x, s in ((k, host[0], host[2]), (v, host[1], host[3])):
        want = x[..., at // ps, at % ps, :, :] * s[..., at // ps, :][..., None]
        lim = torch.finfo(dtype).max
        want = want.clamp(-lim, lim) * good.double()[:, None, None]
        assert torch.equal(got.cpu().double(), want.to(dtype).double())


def test_load_into_strided_outputs_and_empty(cuda):
    H, D, ps, P = 2, 64, 4, 9
    pool = _filled_pool(P, ps, H, D, None, cuda, 1)
    slots = torch.arange(20, device=cuda)
    k, v = yl.load_kv_cache_quant(pool, slots)
    wide = torch.full((20, 2 * H * D + 8), 3.0, dtype=torch.bfloat16, device=cuda)
    out = (wide[:, :H * D], wide[:, H * D:2 * H * D])
    got = yl.load_kv_cache_quant(pool, slots, out=out)
    assert got is out and torch.equal(out[0].reshape(20, H, D), k) and torch.equal(out[1].reshape(20, H, D), v)
    assert bool((wide[:, 2 * H * D:] == 3.0).all())
    e, _ = yl.load_kv_cache_quant(pool, slots[:0])
    assert e.shape == (0, H, D)


def test_store_then_attend_then_load(cuda):
    """A serving loop over the 8-bit pool with the framework's own index build
    and page pool: a prompt step, then decode steps, each stored and attended
    in one stream without a wait; results near 16-bit attention over the
    unquantised rows (a code is off by at most 2^-4 relative to its value, its
    e4m3 half step, so a result by that times the weights' spread, and a score
    by 2^-4 of the sum of |q| |k|)."""
    H, G, D, ps, P, B, W = 2, 4, 128, 16, 64, 3, 16
    pool = yl.quant_kv_pool(P, ps, H, D, device=cuda)
    pages = yl.DevicePagePool(P, device=cuda)
    table = torch.full((B, W), -1, dtype=torch.int32, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(0)
    prior = torch.zeros(B, dtype=torch.int32, device=cuda)
    rows_k, rows_v, have = [[] for _ in range(B)], [[] for _ in range(B)], [0] * B
    for step, new in enumerate([[40, 3, 17], [1, 1, 1], [1, 1, 1], [1, 30, 1]]):
        fresh = torch.tensor(new, dtype=torch.int32, device=cuda)
        pages.reserve(table, prior, fresh, ps)
        idx = yl.build_index(prior, fresh, table, ps, num_pages=P)
        N = sum(new)
        q = 0.3 * torch.randn(N, H * G, D, generator=g, device=cuda)
        k, v = (torch.randn(N, H, D, generator=g, device=cuda).to(torch.bfloat16) for _ in range(2))
        q = q.to(torch.bfloat16)
        yl.store_kv_cache_quant(k, v, pool, idx)
        out = yl.paged_attention(q, pool.k, pool.v, idx, k_scale=pool.k_scale, v_scale=pool.v_scale)
        back_k, back_v = yl.load_kv_cache_quant(pool, idx.slot_mapping)
        at = 0
        for i, n in enumerate(new):
            rows_k[i].append(k[at:at + n])
            rows_v[i].append(v[at:at + n])
            have[i] += n
            kk, vv = torch.cat(rows_k[i]).double(), torch.cat(rows_v[i]).double()
            for t in range(n):
                see = have[i] - n + t + 1
                for h in range(H):
                    qs = q[at + t, h * G:(h + 1) * G].double()
                    s = qs @ kk[:see, h].T / D ** 0.5
                    off = (qs.abs() @ kk[:see, h].abs().T / D ** 0.5).amax(-1, keepdim=True) * 2.0 ** -4
                    w = torch.softmax(s, -1)
                    want, spread = w @ vv[:see, h], w @ vv[:see, h].abs()
                    # requantisation may round a code once more
                    bound = spread * ((1 + 2.0 ** -4) ** 2 * torch.exp(4 * off) - 1) + 2.0 ** -7
                    assert bool(((out[at + t, h * G:(h + 1) * G].double() - want).abs() <= bound).all())
            at += n
        assert bool(((back_k.double() - k.double()).abs() <= k.double().abs() * 2.0 ** -4 + 0.02).all())
        prior = prior + fresh
