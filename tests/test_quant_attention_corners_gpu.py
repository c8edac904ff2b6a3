"""Corners of the 8-bit pool and of the paged attention that a serving program
meets: zero rows, slices of a batch, rows that are missing, scales of any size,
and what a page that only later queries see may hold.  Against 64 bits, with
the bounds of _attnutil.attention_bound where values are rounded."""
import pytest
import torch

import yllang_b200 as yl
from _attnutil import attention_reference, make_index
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
