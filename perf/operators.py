"""Measured cases of the 8-bit KV cache and of the framework's own paged attention.

Four operators, in a plain form (elementary torch operations in 32 bits) and
through the public calls of yllang_b200:

* store: K/V rows quantised to e4m3 as they are written into the paged pool,
  with one power-of-two scale for each page and head;
* load: rows of that pool read back by slot in 16 bits;
* attention over the 8-bit pool, for new tokens of any number per sequence
  (one: decode; many: prefill), causal from each sequence's end;
* the same attention with a sliding window and a few first tokens that stay
  visible, over a 16-bit or an 8-bit pool.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
QMAX = 448.0                 # largest e4m3 value
KMIN, KMAX = -100, 120       # exponents a scale may have


def listed():
    return [
        # One decode step's store of the Llama-3-8B shape, all 32 layers in one call.
        dict(name="store_decode_256seq_32layers", op="store", layers=32, batch=256, lo=128, hi=8192, new=1, heads=8,
             dim=128, page=16, dtype="bf16", pages=512),
        # Ragged prompts written at prefill, two layers of the same model.
        dict(name="store_prefill_64prompts", op="store", layers=2, batch=64, lo=128, hi=4096, new=0, heads=8, dim=128,
             page=16, dtype="bf16", pages=0),
        # Chunks of a few hundred tokens behind cached ones, long pages, narrow heads.
        dict(name="store_chunks_page64", op="store", layers=4, batch=9, lo=1, hi=4607, new=511, heads=3, dim=64,
             page=64, dtype="fp16", pages=0),
        # Reading a batch of cached prompts back in 16 bits (moving them, or a 16-bit attention over them).
        dict(name="load_131k_tokens", op="load", layers=1, tokens=131072, heads=8, dim=128, page=16, dtype="bf16"),
        # One short cached prefix.
        dict(name="load_257_tokens", op="load", layers=1, tokens=257, heads=4, dim=256, page=1, dtype="fp16"),
        # One layer of a decode step, Llama-3-8B heads.
        dict(name="decode_256seq", op="attend", kv="e4m3", batch=256, lo=128, hi=8192, new=1, heads=8, group=4, dim=128,
             page=16, dtype="bf16", window=0, sinks=0),
        # One user's chat: a single sequence, where latency counts.
        dict(name="decode_1seq_8k", op="attend", kv="e4m3", batch=1, lo=8191, hi=8191, new=1, heads=8, group=4, dim=128,
             page=16, dtype="bf16", window=0, sinks=0),
        # Ragged prompts at prefill.
        dict(name="prefill_8prompts", op="attend", kv="e4m3", batch=8, lo=128, hi=4096, new=0, heads=8, group=4,
             dim=128, page=16, dtype="bf16", window=0, sinks=0),
        # Chunked prefill: 512 new tokens behind long histories, Qwen2-72B heads, long pages.
        dict(name="chunks_512_of_8k", op="attend", kv="e4m3", batch=8, lo=600, hi=8192, new=512, heads=8, group=8,
             dim=128, page=64, dtype="fp16", window=0, sinks=0),
        # Long chats with a window: only the window's and the first pages are in the 16-bit pool.
        dict(name="window_decode_128seq", op="attend", kv="16", batch=128, lo=512, hi=32768, new=1, heads=8, group=8,
             dim=128, page=16, dtype="bf16", window=4096, sinks=4),
        # A long prompt with a window.
        dict(name="window_prefill_8k", op="attend", kv="16", batch=1, lo=8192, hi=8192, new=0, heads=8, group=4,
             dim=128, page=16, dtype="bf16", window=1024, sinks=4),
        # A few short chats with a window over the 8-bit pool.
        dict(name="window_decode_5seq_8bit", op="attend", kv="e4m3", batch=5, lo=33, hi=3001, new=1, heads=2, group=7,
             dim=64, page=16, dtype="fp16", window=500, sinks=3),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["store", "load", "attend", "attend", "window", "window"])
    heads, dim = rng.choice([1, 2, 3, 4, 5, 8]), rng.choice([64, 128, 256])
    page, dtype = rng.choice([1, 5, 8, 16, 16, 32, 64, 128]), rng.choice(["bf16", "fp16"])
    row = heads * dim
    if op == "load":
        layers = rng.choice([1, 1, 2, 3])
        return dict(op=op, layers=layers, tokens=_log(rng, 1, max(2, (100 << 20) // (row * layers))), heads=heads,
                    dim=dim, page=page, dtype=dtype)
    if op == "store":
        layers = _log(rng, 1, 32)
        batch = _log(rng, 1, 256)
        new = rng.choice([1, 1, 2, 0, _log(rng, 2, 700)])
        hi = _log(rng, 2, 8192)
        if new == 0:
            hi = max(2, min(hi, (200 << 20) // (layers * row * batch)))
        elif new > 1:
            new = max(2, min(new, (200 << 20) // (layers * row * batch)))
        return dict(op=op, layers=layers, batch=batch, lo=max(1, hi // 8), hi=hi, new=new, heads=heads, dim=dim,
                    page=page, dtype=dtype, pages=0)
    group = rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 8, 16])
    kind = rng.choice(["decode", "decode", "prefill", "chunk", "few"])
    window = _log(rng, 1, 4096) if op == "window" else 0
    sinks = rng.choice([0, 1, 4, 17, 64]) if op == "window" else 0
    kv = rng.choice(["e4m3", "16"]) if op == "window" else "e4m3"
    if kind in ("decode", "few"):
        batch = _log(rng, 1, 256)
        hi = max(1, min(_log(rng, 1, 16384), (256 << 20) // (row * batch)))
        new = 1 if kind == "decode" else rng.choice([2, 3, 4])
    elif kind == "prefill":
        batch = _log(rng, 1, 16)
        hi, new = max(1, min(_log(rng, 16, 6000), int(math.sqrt((1 << 31) / (batch * heads * group)) * 128 / dim))), 0
    else:
        batch, new = _log(rng, 1, 8), _log(rng, 5, 700)
        hi = min(_log(rng, 16, 8192), max(16, (1 << 30) // (batch * heads * group * new)))
    return dict(op="attend", kv=kv, batch=batch, lo=max(1, hi // 8), hi=hi, new=new, heads=heads, group=group, dim=dim,
                page=page, dtype=dtype, window=window, sinks=sinks)


def _lengths(case):
    """prior and new tokens of each sequence; `new` 0: a whole prompt without cached tokens."""
    rng = np.random.default_rng(11 + case["batch"])
    total = rng.integers(case["lo"], case["hi"] + 1, case["batch"]).astype(np.int64)
    new = total.copy() if case["new"] == 0 else np.minimum(total, case["new"])
    return total - new, new


def _visible_from(total, new, window, sinks, page):
    """First page of the window and the number of first pages that some new token sees."""
    if window <= 0:
        return 0, 0
    first = max(0, total - new + 1 - window)
    return first // page, -(-min(sinks, total) // page)


def _index(case, rng, unique):
    """The page arrays of a batch with scattered pages; `unique`: the pages that a sequence needs, as (lo, hi)
    ranges of page ordinals. Other entries are -1 (pages given back, or never read)."""
    prior, new = _lengths(case)
    ps = case["page"]
    count = -(-(prior + new) // ps)
    indptr = np.concatenate([[0], np.cumsum(count)])
    own_page = np.zeros(int(indptr[-1]), bool)
    for i, (a, ranges) in enumerate(zip(indptr, unique(prior, new, count))):
        for lo, hi in ranges:
            own_page[a + lo:a + hi] = True
    need = int(own_page.sum())
    pages = max(need, case.get("pages", 0)) + 3
    ids = np.full(int(indptr[-1]), -1, np.int64)
    ids[own_page] = rng.permutation(pages)[:need]
    last = np.where(count > 0, (prior + new - 1) % ps + 1, 0)
    qo = np.concatenate([[0], np.cumsum(new)])
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(torch.int32).cuda()  # noqa: E731
    pos = np.concatenate([np.arange(p, p + n) for p, n in zip(prior, new)]) if len(new) else np.zeros(0, np.int64)
    seq = np.repeat(np.arange(len(new)), new)
    slot = ids[indptr[seq] + pos // ps] * ps + pos % ps
    return dict(kv_indptr=t(indptr), kv_indices=t(ids), kv_last_page_len=t(last), qo_indptr=t(qo),
                slot_mapping=torch.from_numpy(slot).cuda()), pages, prior.tolist(), new.tolist()


def _pool8(layers, pages, page, heads, dim, g):
    """An 8-bit pool with contents: [layers, pages, page, heads, dim] views of head-major pages."""
    shape = (layers, pages, heads, page, dim)
    out = []
    for _ in range(2):
        scale = torch.exp2(torch.randint(-8, -4, (layers, pages, heads), generator=g, device="cuda").float())
        codes = torch.empty(shape, dtype=torch.float8_e4m3fn, device="cuda")
        for layer in range(layers):
            codes[layer].copy_((torch.randn(shape[1:], generator=g, device="cuda") * 64).clamp_(-QMAX, QMAX))
        out += [codes.transpose(2, 3), scale]
    return dict(k=out[0], v=out[2], k_scale=out[1], v_scale=out[3])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    dtype, H, D, ps = DTYPES[case["dtype"]], case["heads"], case["dim"], case["page"]
    if case["op"] == "load":
        pages = -(-case["tokens"] // ps) + 2
        pool = _pool8(case["layers"], pages, ps, H, D, g)
        order = rng.permutation(pages)[:-(-case["tokens"] // ps)]
        slots = (order[:, None] * ps + np.arange(ps)[None]).reshape(-1)[:case["tokens"]]
        return dict(case=case, dtype=dtype, pool=pool, slots=torch.from_numpy(slots).cuda())
    if case["op"] == "store":
        def unique(prior, new, count):
            return [[(int(p) // ps, int(c))] for p, c in zip(prior, count)]
        index, pages, prior, new = _index(case, rng, unique)
        L, N = case["layers"], sum(new)
        # rows of different loudness, some elements far out, as keys have
        x = [torch.empty(L, N, H * D, dtype=dtype, device="cuda") for _ in range(2)]
        for t in x:
            loud = torch.exp2(torch.randn(N, H, 1, generator=g, device="cuda"))
            for layer in range(L):
                t[layer].copy_((torch.randn(N, H, D, generator=g, device="cuda") * loud).view(N, H * D))
        pool = _pool8(L, pages, ps, H, D, g)
        return dict(case=case, k=x[0], v=x[1], pool=pool, index=index,
                    prior=torch.tensor(prior, device="cuda"), new=torch.tensor(new, device="cuda"))

    def unique(prior, new, count):
        got = []
        for p, n, c in zip(prior.tolist(), new.tolist(), count.tolist()):
            first, head = _visible_from(p + n, n, case["window"], case["sinks"], ps)
            got.append([(0, min(head, c)), (first, c)])
        return got
    index, pages, prior, new = _index(case, rng, unique)
    N, Hq = sum(new), H * case["group"]
    q = (torch.randn(N, Hq, D, generator=g, device="cuda") * 1.5).to(dtype)
    if case["kv"] == "e4m3":
        pool = _pool8(1, pages, ps, H, D, g)
        pool = {k: v[0] for k, v in pool.items()}
    else:
        pool = dict(k=torch.randn(pages, ps, H, D, generator=g, device="cuda", dtype=dtype),
                    v=torch.randn(pages, ps, H, D, generator=g, device="cuda", dtype=dtype), k_scale=None, v_scale=None)
    return dict(case=case, dtype=dtype, q=q, pool=pool, index=index, prior=prior, new=new, most_new=max(new, default=0))


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _rows(pool, which, slots, page):
    """[..., n, heads, dim] values of the given slots in 32 bits; slots [n] or [a, b]."""
    x, s = pool[which], pool[which + "_scale"]
    at, off = slots // page, slots % page
    if x.dtype != torch.float8_e4m3fn:
        return x[at, off].float()
    codes = x.view(torch.uint8)
    if x.dim() == 4:
        return codes[at, off].view(torch.float8_e4m3fn).float() * s[at][..., None]
    return codes[:, at, off].view(torch.float8_e4m3fn).float() * s[:, at][..., None]


def _plain_load(s):
    page = s["case"]["page"]
    return {"k": _rows(s["pool"], "k", s["slots"], page).to(s["dtype"]),
            "v": _rows(s["pool"], "v", s["slots"], page).to(s["dtype"])}


def _two_to(k):
    return ((k + 127) << 23).to(torch.int32).view(torch.float32)


def _plain_store(s):
    case, idx, pool = s["case"], s["index"], s["pool"]
    L, H, D, ps = case["layers"], case["heads"], case["dim"], case["page"]
    prior, new = s["prior"], s["new"]
    N, P = s["k"].shape[1], pool["k"].shape[1]
    slot = idx["slot_mapping"]
    at, off = slot // ps, slot % ps
    # tokens that a touched page held before this call
    seq = torch.repeat_interleave(torch.arange(new.shape[0], device="cuda"), new, output_size=N)
    pos = prior[seq] + torch.arange(N, device="cuda") - idx["qo_indptr"][:-1].long()[seq]
    held = torch.full((P,), -1, dtype=torch.int64, device="cuda")
    held[at] = (prior[seq] - pos // ps * ps).clamp(0, ps)
    touched = torch.nonzero(held >= 0)[:, 0]
    held = held[touched]
    where = torch.zeros(P, dtype=torch.int64, device="cuda")
    where[touched] = torch.arange(touched.shape[0], device="cuda")
    for name in ("k", "v"):
        x = s[name].view(L, N, H, D).float()
        amax = torch.zeros(L, touched.shape[0], H, device="cuda")
        amax.index_reduce_(1, where[at], x.abs().amax(-1), "amax")
        m, e = torch.frexp(amax)
        need = _two_to((e - torch.where(m <= 0.875, 9, 8)).clamp(KMIN, KMAX).masked_fill(amax == 0, KMIN))
        scale, codes = pool[name + "_scale"], pool[name].view(torch.uint8)
        old = scale[:, touched]
        grown = torch.maximum(need, torch.where((held > 0)[None, :, None], old, torch.zeros_like(old)))
        # tokens that were there take the page's new scale
        mine = codes[:, touched]                                          # [L, T, ps, H, D]
        again = mine.view(torch.float8_e4m3fn).float() * (old / grown)[:, :, None, :, None]
        keep = torch.arange(ps, device="cuda")[None, :] < held[:, None]   # [T, ps]
        codes[:, touched] = torch.where(keep[None, :, :, None, None], again.to(torch.float8_e4m3fn).view(torch.uint8),
                                        mine)
        scale[:, touched] = grown
        codes[:, at, off] = (x / grown[:, where[at]][..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
    return dict(pool)


def _slots_of(idx, seq, pos, page):
    return idx["kv_indices"].long()[idx["kv_indptr"].long()[seq] + pos // page] * page + pos % page


def _seen(qpos, kpos, window, sinks):
    ok = kpos <= qpos
    if window > 0:
        ok = ok & ((kpos > qpos - window) | (kpos < sinks))
    return ok


def _plain_attend(s):
    case, idx, q = s["case"], s["index"], s["q"]
    H, G, D, ps, W, S = (case[k] for k in ("heads", "group", "dim", "page", "window", "sinks"))
    prior, new = s["prior"], s["new"]
    if s["most_new"] <= 1:  # every sequence at once, over the longest one's visible positions
        total = torch.tensor([p + n for p, n in zip(prior, new)], device="cuda")
        longest = max(p + n for p, n in zip(prior, new))
        if W > 0:
            start = (total - W).clamp(min=0)
            first = torch.arange(min(S, longest), device="cuda")
            run = torch.arange(min(W, longest), device="cuda")
            pos = torch.cat([first[None].expand(len(prior), -1), start[:, None] + run[None]], 1)
            ok = torch.cat([first[None] < torch.minimum(start, total)[:, None], (start[:, None] + run[None]) < total[:, None]], 1)
        else:
            pos = torch.arange(longest, device="cuda")[None].expand(len(prior), -1)
            ok = pos < total[:, None]
        pos = torch.where(ok, pos, (total - 1)[:, None])
        slots = _slots_of(idx, torch.arange(len(prior), device="cuda")[:, None], pos, ps)
        k, v = _rows(s["pool"], "k", slots, ps), _rows(s["pool"], "v", slots, ps)      # [B, n, H, D]
        a = torch.einsum("bhgd,bnhd->bhgn", q.float().view(-1, H, G, D), k) / math.sqrt(D)
        a = a.masked_fill(~ok[:, None, None], float("-inf"))
        a = torch.exp(a - a.amax(-1, keepdim=True))
        o = torch.einsum("bhgn,bnhd->bhgd", a, v) / a.sum(-1)[..., None]
        return o.reshape(-1, H * G, D).to(s["dtype"])
    out, at = torch.empty_like(q), 0
    for i, (p, n) in enumerate(zip(prior, new)):  # ragged: a sequence at a time
        pos = torch.arange(p + n, device="cuda")
        if W > 0:
            pos = torch.cat([pos[:min(S, max(0, p + 1 - W))], pos[max(0, p + 1 - W):]])
        slots = _slots_of(idx, torch.tensor(i, device="cuda"), pos, ps)
        k, v = _rows(s["pool"], "k", slots, ps), _rows(s["pool"], "v", slots, ps)      # [n, H, D]
        ok = _seen(torch.arange(p, p + n, device="cuda")[:, None], pos[None], W, S)
        a = torch.einsum("thgd,nhd->hgtn", q[at:at + n].float().view(n, H, G, D), k) / math.sqrt(D)
        a = a.masked_fill_(~ok, float("-inf"))
        a = a.sub_(a.amax(-1, keepdim=True)).exp_()
        o = torch.einsum("hgtn,nhd->thgd", a, v) / a.sum(-1).permute(2, 0, 1)[..., None]
        out[at:at + n] = o.reshape(n, H * G, D).to(s["dtype"])
        at += n
    return out


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _own(s):
    import yllang_b200 as yl

    case, p = s["case"], s["pool"]
    if case["op"] == "load":
        k, v = yl.load_kv_cache_quant(yl.QuantKVPool(**p), s["slots"], dtype=s["dtype"])
        return {"k": k, "v": v}
    index = yl.BatchIndex(**s["index"])
    if case["op"] == "store":
        yl.store_kv_cache_quant(s["k"], s["v"], yl.QuantKVPool(**p), index)
        return dict(p)
    return yl.paged_attention(s["q"], p["k"], p["v"], index, k_scale=p["k_scale"], v_scale=p["v_scale"],
                              window=case["window"], sinks=case["sinks"], max_new_len=s["most_new"])


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return (_plain_load if op == "load" else _plain_store if op == "store" else _plain_attend)(state)


# ---------------------------------------------------------------------------
# what a pass cannot do without, and the definition in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    H, D, ps = case["heads"], case["dim"], case["page"]
    row = H * D
    if case["op"] == "load":
        n = case["tokens"] * case["layers"]
        return {"bytes": 2 * (n * row * 3 + -(-case["tokens"] // ps) * case["layers"] * H * 4) + 8 * case["tokens"],
                "flops": 2 * n * row}
    prior, new = _lengths(case)
    total = prior + new
    if case["op"] == "store":
        n = int(new.sum()) * case["layers"]
        touched = int((-(-total // ps) - prior // ps).sum())
        return {"bytes": 2 * (n * row * 3 + touched * case["layers"] * H * 8) + 16 * len(new) + 4 * touched,
                "flops": 4 * n * row}
    W, S = case["window"], case["sinks"]
    read = pairs = pages = 0
    for t, n in zip(total.tolist(), new.tolist()):
        if n == 0:
            continue
        qpos = np.arange(t - n, t)
        low = np.maximum(0, qpos + 1 - W) if W > 0 else np.zeros(n, np.int64)
        pairs += int((qpos + 1 - low + np.minimum(low, S)).sum())
        tokens = t - int(low[0]) + min(int(low[0]), S)
        read += tokens
        pages += -(-tokens // ps)
    Hq = H * case["group"]
    item = 1 if case["kv"] == "e4m3" else 2
    return {"bytes": 2 * read * row * item + (pages * H * 8 if item == 1 else 0) + pages * 4 + 4 * int(new.sum()) * Hq * D,
            "flops": 4 * pairs * Hq * D}


def _e4m3(x):
    """Nearest e4m3 value, ties to even, of |x| <= 448 in 64 bits."""
    e = (torch.frexp(x)[1] - 1).clamp(min=-6).double()
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def _exact_store(s):
    """Page by page, from the definition: a page's scale is the least power of two that brings the largest of its new
    tokens, and of the scale that its earlier tokens have, within e4m3's range."""
    case, idx, pool = s["case"], s["index"], s["pool"]
    H, D, ps = case["heads"], case["dim"], case["page"]
    indptr, ids = idx["kv_indptr"].tolist(), idx["kv_indices"].tolist()
    prior, new, qo = s["prior"].tolist(), s["new"].tolist(), idx["qo_indptr"].tolist()
    got = {}
    for name in ("k", "v"):
        codes = pool[name].to(torch.float64).contiguous()
        scale = pool[name + "_scale"].double().clone()
        x = s[name].view(s[name].shape[0], -1, H, D)
        for i, (p, n) in enumerate(zip(prior, new)):
            for j in range(p // ps, -(-(p + n) // ps) if n else 0):
                a, b = max(p, j * ps), min(p + n, (j + 1) * ps)
                rows = x[:, qo[i] + a - p:qo[i] + b - p].double()              # [L, t, H, D]
                amax = rows.abs().amax((1, 3))
                k = torch.ceil(torch.log2(torch.where(amax > 0, amax, 1.0) / QMAX))
                k = torch.where(amax > torch.exp2(k) * QMAX, k + 1, k)
                k = torch.where(amax <= torch.exp2(k - 1) * QMAX, k - 1, k).clamp(KMIN, KMAX)
                want = torch.exp2(torch.where(amax > 0, k, torch.full_like(k, KMIN)))
                page, had = ids[indptr[i] + j], max(0, min(p - j * ps, ps))
                if had:
                    was = scale[:, page].clone()
                    want = torch.maximum(want, was)
                    codes[:, page, :had] = _e4m3(codes[:, page, :had] * (was / want)[:, None, :, None])
                scale[:, page] = want
                codes[:, page, a - j * ps:b - j * ps] = _e4m3(rows / want[:, None, :, None])
        got[name], got[name + "_scale"] = codes, scale
    return got


def exact(case, seed):
    w = work(case)
    if case["op"] == "store" and sum(-(-int(t) // case["page"]) + 1 for t in _lengths(case)[1]) > 12000:
        return None
    if w["flops"] > 4e12:
        return None
    s = prepare(case, seed)
    pool = s["pool"]
    if case["op"] == "store":
        return _exact_store(s)
    ps = case["page"]

    def rows(which, slots):
        x, sc = pool[which], pool[which + "_scale"]
        if sc is None:
            return x[slots // ps, slots % ps].double()
        x = x if x.dim() == 5 else x[None]
        sc = sc if sc.dim() == 3 else sc[None]
        got = x.view(torch.uint8)[:, slots // ps, slots % ps].view(torch.float8_e4m3fn).double()
        got = got * sc.double()[:, slots // ps][..., None]
        return got if case["op"] == "load" else got[0]

    if case["op"] == "load":
        return {"k": rows("k", s["slots"]), "v": rows("v", s["slots"])}
    H, G, D, W, S = (case[k] for k in ("heads", "group", "dim", "window", "sinks"))
    indptr, ids = s["index"]["kv_indptr"].tolist(), s["index"]["kv_indices"].long()
    out, at = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    for i, (p, n) in enumerate(zip(s["prior"], s["new"])):
        pos = np.arange(p + n)
        if W > 0:
            pos = pos[(pos > p - W) | (pos < S)]
        pos = torch.from_numpy(pos).cuda()
        slots = ids[indptr[i] + pos // ps] * ps + pos % ps
        k, v = rows("k", slots), rows("v", slots)
        qs = s["q"][at:at + n].double().view(n, H, G, D)
        qpos = torch.arange(p, p + n, device="cuda")[:, None]
        hidden = pos[None] > qpos
        if W > 0:
            hidden = hidden | ((pos[None] <= qpos - W) & (pos[None] >= S))
        for h in range(H):
            a = torch.matmul(qs[:, h].transpose(0, 1), k[:, h].t()) * D ** -0.5             # [G, n, len]
            a = torch.softmax(a.masked_fill(hidden, float("-inf")), -1)
            out[at:at + n].view(n, H, G, D)[:, h] = torch.matmul(a, v[:, h]).transpose(0, 1)
        at += n
    return out
