"""Helpers of the 8-bit pool's and the paged attention's tests: batches with
scattered pages, and plain 64-bit restatements on the host."""
from __future__ import annotations

import math

import numpy as np
import torch

import yllang_b200 as yl

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # torch.finfo(t).eps / 2


def make_index(prior, new, page_size, num_pages, seed=0, device="cuda", spare=0):
    """Page arrays of a batch over a random permutation of the pool's pages
    (host lists of page ids too); `spare` unused entries follow kv_indices."""
    prior, new = np.asarray(prior, np.int64), np.asarray(new, np.int64)
    count = -(-(prior + new) // page_size)
    perm = np.random.default_rng(seed).permutation(num_pages)
    assert count.sum() <= num_pages
    indptr = np.concatenate([[0], np.cumsum(count)])
    ids = perm[:indptr[-1]]
    pages = [ids[a:b].tolist() for a, b in zip(indptr[:-1], indptr[1:])]
    last = np.where(count > 0, (prior + new - 1) % page_size + 1, 0)
    qo = np.concatenate([[0], np.cumsum(new)])
    slots = [pages[i][p // page_size] * page_size + p % page_size
             for i in range(len(prior)) for p in range(prior[i], prior[i] + new[i])]
    t = lambda a, d=torch.int32: torch.tensor(np.asarray(a, np.int64), dtype=d, device=device)  # noqa: E731
    idx = yl.BatchIndex(t(indptr), t(np.concatenate([ids, np.full(spare, -7)])), t(last), t(qo),
                        t(slots, torch.int64))
    return idx, pages


def e4m3(x: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 value of x (64 bits), ties to even, |x| > 448 to 448."""
    e = (torch.frexp(x)[1] - 1).clamp(min=-6).double()
    step = torch.exp2(e - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def page_scale(amax: float) -> float:
    """Least power of two s with amax / s <= 448, exponent in [-100, 120]."""
    if amax == 0:
        return 2.0 ** -100
    k = math.floor(math.log2(amax)) - 12
    while amax > 448 * 2.0 ** k:
        k += 1
    return 2.0 ** min(max(k, -100), 120)


def store_reference(x, codes, scale, prior, new, pages, page_size):
    """One plane in 64 bits, in place: x [N, H, D] (finite), codes [P, ps, H, D]
    as the values they stand for, scale [P, H]."""
    at = 0
    for p, n, mine in zip(prior, new, pages):
        for j in range(p // page_size, -(-(p + n) // page_size) if n else 0):
            a, b = max(p, j * page_size), min(p + n, (j + 1) * page_size)
            rows = x[at + a - p:at + b - p]
            held, page = a - j * page_size, mine[j]
            for h in range(x.shape[1]):
                want = page_scale(float(rows[:, h].abs().max()))
                if held:
                    old = float(scale[page, h])
                    want = max(want, old)
                    codes[page, :held, h] = e4m3(codes[page, :held, h] * (old / want))
                scale[page, h] = want
                codes[page, held:held + b - a, h] = e4m3(rows[:, h] / want)
        at += n


def attention_reference(q, k_pages, v_pages, prior, new, pages, window=0, sinks=0, sm_scale=None):
    """64-bit attention on host tensors: q [N, Hq, D], pages [P, ps, H, D].
    Returns (o, spread): spread is the sum of weight * |v| of each element,
    what a relative error of the weights multiplies, and `reach`, the largest
    sum of |q| |k| of a row's scores times sm_scale."""
    N, Hq, D = q.shape
    H, ps = k_pages.shape[2], k_pages.shape[1]
    G = Hq // H
    sm_scale = D ** -0.5 if sm_scale is None else sm_scale
    out = torch.zeros(N, Hq, D, dtype=torch.float64)
    spread, reach = torch.zeros_like(out), torch.zeros(N, Hq, 1, dtype=torch.float64)
    row = 0
    for p, n, mine in zip(prior, new, pages):
        total = p + n
        for t in range(n):
            pos = p + t
            see = [j for j in range(pos + 1) if window == 0 or j > pos - window or j < sinks]
            if see:
                at = torch.tensor([mine[j // ps] for j in see]), torch.tensor([j % ps for j in see])
                k, v = k_pages[at].double(), v_pages[at].double()  # [n, H, D]
                for h in range(H):
                    qs = q[row, h * G:(h + 1) * G].double()
                    s = qs @ k[:, h].T * sm_scale
                    w = torch.softmax(s, -1)
                    out[row, h * G:(h + 1) * G] = w @ v[:, h]
                    spread[row, h * G:(h + 1) * G] = w @ v[:, h].abs()
                    reach[row, h * G:(h + 1) * G, 0] = (qs.abs() @ k[:, h].abs().T * sm_scale).amax(-1)
            row += 1
        assert total >= n
    return out, spread, reach


def attention_bound(want, spread, reach, dtype, weights, head_dim):
    """How far a right kernel can be from the 64-bit result: the output's one
    rounding; the weights' one rounding to `weights`; and fp32 arithmetic of
    the scores, off by (head_dim + 4) half steps of 2^-24 times the sum of
    |q| |k|, which changes a weight and the sum of weights by that much each,
    with 2^-21 for the exponential and the sums; fp16 weights more than 2^-24
    below the largest may vanish (with their lift, 2^-27 and less)."""
    delta = 2 * reach * (head_dim + 4) * 2.0 ** -24 + 2.0 ** -20
    return HALF_STEP[dtype] * want.abs() + (HALF_STEP[weights] + 2 * delta) * spread * (1 + 2.0 ** -8) + 1e-7
