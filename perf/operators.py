"""Performance cases of the attention between a decoder layer's q/k/v and o linears, and of the 8-bit cache it reads.

Kinds of case:

  prompt   causal attention of packed prompts of different lengths with grouped heads: the prefill's attention.  A
           chunk of a prompt attends to all keys up to its own end (more keys than queries).
  append   new keys and values go into the paged int8 cache: 64 tokens a page, one scale per page, head and side.
  cache    attention of each sequence's last tokens over that cache: one token (decode), a verify block, a chunk.
  weights  the softmax weights that those tokens give to each cached token, summed over them and over the query heads of
           a key/value head, and added to what earlier calls gave.
  evict    each head of each sequence keeps its last `recent` tokens and those of the others with the largest summed
           weights, `keep` in all, moved together into new pages.

The cache is `k_cache` int8 [pages, kv heads, 64, d], `v_cache` int8 [pages, kv heads, d, 64] (a page's values are held
transposed) and float32 `k_scale`, `v_scale` [pages, kv heads]; a value is code * scale.  Page j of sequence b is
block_table[b, j].  The scale of a page is the absmax of what it holds / 127.  Where new tokens of a page are larger
than what it held, its codes are rounded to the new scale.
"""

import math

import torch

own = False

PAGE = 64
TINY = 2.0 ** -100     # a page with no larger value than this is held as zeros
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    # 32 query heads on 8 key/value heads of 128: the attention of this repository's decoder layer (4096 / 1024).
    layer = {"hq": 32, "hkv": 8, "d": 128}
    kv = {"hkv": 8, "d": 128}
    return [
        # three short requests in one call: latency
        {"name": "prompt_short", "kind": "prompt", "q": "45,1,17", "k": "45,1,17", "dtype": "bf16", **layer},
        # prompts and a chunk of one (behind 1500 tokens prefilled before) with as many key/value heads as query heads
        {"name": "prompt_ragged", "kind": "prompt", "q": "1999,700,1024,331", "k": "1999,700,1024,1831", "hq": 16,
         "hkv": 16, "d": 64, "dtype": "fp16"},
        # one long multimodal prompt
        {"name": "prompt_long", "kind": "prompt", "q": "8192", "k": "8192", "dtype": "bf16", **layer},
        # a decode step's new token of 32 sequences
        {"name": "append_decode", "kind": "append", "q": ",".join(["1"] * 32),
         "k": ",".join(str(1 + 251 * i) for i in range(32)), "dtype": "bf16", **kv},
        # a batch of long prompts, one of them behind a cached prefix
        {"name": "append_prompts", "kind": "append", "q": "8192,16001,5000,3100", "k": "0,0,100,0", "dtype": "fp16", **kv},
        # a decode step of one sequence: latency
        {"name": "cache_one", "kind": "cache", "q": "1", "k": "1733", "dtype": "bf16", **layer},
        # verify blocks of 16 drafted tokens
        {"name": "cache_verify", "kind": "cache", "q": "16,16,16,16,16,16,16,16",
         "k": "4112,3000,5111,2048,4000,6001,777,1300", "dtype": "fp16", **layer},
        # a large ragged decode batch
        {"name": "cache_batch", "kind": "cache", "q": ",".join(["1"] * 64),
         "k": ",".join(str(300 + 241 * i) for i in range(64)), "dtype": "bf16", **layer},
        # the weights that the last 16 tokens of a prompt give to what is cached
        {"name": "weights_window", "kind": "weights", "q": "16", "k": "4097", "dtype": "fp16", **layer},
        # a decode step's weights, added up for a later eviction
        {"name": "weights_batch", "kind": "weights", "q": ",".join(["1"] * 32),
         "k": ",".join(str(300 + 241 * i) for i in range(32)), "dtype": "bf16", **layer},
        # one sequence's cache cut to a budget
        {"name": "evict_one", "kind": "evict", "k": "4097", "keep": 1000, "recent": 100, "dtype": "bf16", **kv},
        # a batch whose sequences outgrew their budget, some of them not yet
        {"name": "evict_batch", "kind": "evict", "k": ",".join(str(1500 + 401 * i) for i in range(32)), "keep": 4096,
         "recent": 512, "dtype": "bf16", **kv},
    ]


def _spread(rng, lo, hi):
    """A whole number of lo..hi, spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = ((32, 8), (16, 16), (16, 4), (28, 4), (12, 2), (8, 1), (5, 5))


def draw(rng):
    kind = rng.choice(("prompt", "prompt", "append", "cache", "cache", "weights", "evict"))
    hq, hkv = rng.choice(HEADS)
    d = rng.choice((64, 128))
    case = {"kind": kind, "hkv": hkv, "d": d, "dtype": rng.choice(("bf16", "fp16"))}
    if kind == "prompt":
        b = _spread(rng, 1, 16)
        top = min(8192, int(8192 * math.sqrt(32.0 / (hq * b))))
        q = [_spread(rng, 1, top) for _ in range(b)]
        more = rng.random() < 0.4
        k = [min(top, n + (_spread(rng, 1, top) if more else 0)) for n in q]
        case.update(hq=hq, q=",".join(map(str, q)), k=",".join(map(str, k)))
    elif kind == "append":
        b = _spread(rng, 1, 128)
        step = rng.random() < 0.5
        q = [1 if step else _spread(rng, 1, max(2, 256000 // (b * hkv))) for _ in range(b)]
        k = [rng.choice((0, _spread(rng, 1, 8192))) for _ in range(b)]
        case.update(dtype=rng.choice(("bf16", "fp16", "fp32")), q=",".join(map(str, q)), k=",".join(map(str, k)))
    elif kind == "evict":
        b = _spread(rng, 1, 64)
        k = [_spread(rng, 1, min(65536, 2000000 // (b * hkv))) for _ in range(b)]
        keep = _spread(rng, 1, max(k))
        case.update(k=",".join(map(str, k)), keep=keep, recent=rng.choice((0, keep, rng.randint(0, keep))))
    else:
        b = _spread(rng, 1, 128)
        n = rng.choice((1, 1, rng.randint(2, 8), 16, rng.randint(17, 200)))
        n = min(n, max(1, 512 // b))
        q = [n if rng.random() < 0.8 else rng.randint(1, n) for _ in range(b)]
        top = min(131072, 480000 * 8 // (b * hkv), int(1.2e11 / (b * n * hq * d)))
        k = [max(m, _spread(rng, 1, top)) for m in q]
        case.update(hq=hq, q=",".join(map(str, q)), k=",".join(map(str, k)))
    return case


def _lens(text):
    return [int(s) for s in text.split(",")]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _cu(lens):
    return torch.tensor([0] + lens, dtype=torch.int32, device="cuda").cumsum(0, dtype=torch.int32)


def _values(gen, *shape):
    """Rows of keys, queries or values: normal, with a few channels of each head larger than the others."""
    x = torch.randn(*shape, generator=gen, device="cuda")
    amp = 1.0 + 3.0 * (torch.rand(shape[-2], shape[-1], generator=gen, device="cuda") < 0.03).float()
    return x.mul_(amp)


def _pages(x):
    """Codes and scales of full pages x [pages, heads, 64, d]."""
    top = x.abs().amax((-1, -2))
    codes = torch.round(x * (127.0 / top)[..., None, None]).to(torch.int8)
    return codes, top / 127.0


def _table(lens, gen, spare=3):
    """Pages of the sequences in a random order, with some pages that belong to none: (block_table, pages in all)."""
    need = [-(-n // PAGE) for n in lens]
    total = sum(need) + spare
    perm = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    idx = torch.arange(max(max(need), 1), device="cuda")
    need_t = torch.tensor(need, device="cuda")
    first = need_t.cumsum(0) - need_t
    at = (first[:, None] + idx[None]).clamp(max=total - 1)
    return torch.where(idx[None] < need_t[:, None], perm[at], torch.full_like(perm[at], -1)).contiguous(), total


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind, hkv, d, dt = case["kind"], case["hkv"], case["d"], DT[case["dtype"]]
    q, k = _lens(case["q"]) if kind != "evict" else [], _lens(case["k"])
    state = {"kind": kind, "lens_q": q, "lens_k": k, "scale": 1.0 / math.sqrt(d), "cu_q": _cu(q)}
    if kind == "prompt":
        # what the three linears of a layer return, seen as heads
        state["q"] = _values(gen, sum(q), case["hq"], d).to(dt)
        state["k"] = _values(gen, sum(k), hkv, d).to(dt)
        state["v"] = _values(gen, sum(k), hkv, d).to(dt)
        state["cu_k"] = _cu(k)
        return state
    after = k
    if kind == "append":
        after = [n + m for n, m in zip(q, k)]
        state["k"] = _values(gen, sum(q), hkv, d).to(dt)
        state["v"] = _values(gen, sum(q), hkv, d).to(dt)
        state["cached"] = torch.tensor(k, dtype=torch.int32, device="cuda")
    else:
        state["lens"] = torch.tensor(k, dtype=torch.int32, device="cuda")
    if kind in ("cache", "weights"):
        state["q"] = _values(gen, sum(q), case["hq"], d).to(dt)
    state["table"], pages = _table(after, gen)
    if kind == "evict":
        # pages of their own for what is kept
        state["keep"], state["recent"] = case["keep"], case["recent"]
        fresh, more = _table([min(m, case["keep"]) for m in k], gen, 0)
        state["new_table"] = torch.where(fresh >= 0, fresh + pages, fresh)
        pages += more
    state["k_cache"], state["k_scale"] = _pages(_values(gen, pages, hkv, PAGE, d))
    codes, state["v_scale"] = _pages(_values(gen, pages, hkv, PAGE, d))
    state["v_cache"] = codes.transpose(-1, -2).contiguous()
    if kind in ("weights", "evict"):
        # a few tokens hold most of the weight, and some none at all
        w = torch.randn(len(k), hkv, max(k), generator=gen, device="cuda").mul_(2.0).exp_()
        state["weights"] = w.mul_((w > 0.08).float())
    if kind == "weights":
        # from calls like this one before it
        w.mul_(case["hq"] // hkv * (sum(q) / len(q)) / w.sum(-1, keepdim=True))
        state["lse"] = _cache(state)["lse"]        # from the attention call before it
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    if own:
        return _own(state)
    return {"prompt": _prompt, "append": _append, "cache": _cache, "weights": _weights, "evict": _evict}[state["kind"]](state)


def _own(s):
    from alpamayo_amd import attention
    if s["kind"] == "prompt":
        out, lse = attention.prompt_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], scale=s["scale"])
        return {"out": out, "lse": lse}
    pools = (s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
    if s["kind"] == "append":
        attention.kv_append_i8(s["k"], s["v"], *pools, s["table"], s["cu_q"], s["cached"])
        return dict(zip(("k_codes", "v_codes", "k_scale", "v_scale"), pools))
    if s["kind"] == "weights":
        total = s["weights"].clone()
        attention.cache_weights_i8(s["q"], s["k_cache"], s["k_scale"], s["table"], s["cu_q"], s["lens"], s["lse"], total,
                                   scale=s["scale"])
        return {"weights": total}
    if s["kind"] == "evict":
        weights, lens, kept = attention.cache_evict_i8(*pools, s["weights"], s["table"], s["lens"], s["new_table"],
                                                       s["keep"], s["recent"])
        return {"weights": weights, "lens": lens, "kept": kept,
                **dict(zip(("k_codes", "v_codes", "k_scale", "v_scale"), pools))}
    out, lse = attention.cache_attention_i8(s["q"], *pools, s["table"], s["cu_q"], s["lens"], scale=s["scale"])
    return {"out": out, "lse": lse}


def _rows(cu, total):
    """Sequence and place in it of each packed row."""
    rows = torch.arange(total, device=cu.device)
    seq = torch.searchsorted(cu[1:].long(), rows, right=True)
    return seq, rows - cu[seq].long()


def _padded(x, seq, place, batch, most):
    """Packed rows x [rows, heads, d] as float32 [batch, heads, most, d], zeros behind each sequence."""
    y = torch.zeros(batch, most, *x.shape[1:], device=x.device)
    y[seq, place] = x.float()
    return y.transpose(1, 2)


def _attend(q, k, v, lens_q, lens_k, scale):
    """Softmax attention in float32, q [b, hq, n, d] on k, v [b, hkv, m, d], the last query on the last key: (out, lse)."""
    b, hq, n, d = q.shape
    hkv, m = k.shape[1:3]
    s = torch.matmul(q.reshape(b, hkv, hq // hkv * n, d) * scale, k.transpose(-1, -2)).view(b, hq, n, m)
    at_q = torch.arange(n, device=q.device)[None, :, None] + (lens_k - lens_q)[:, None, None]
    at_k = torch.arange(m, device=q.device)[None, None]
    s.masked_fill_((at_k > at_q)[:, None], -math.inf)
    top = s.amax(-1, keepdim=True).clamp_(min=-3e38)
    s.sub_(top).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(b, hkv, hq // hkv * n, m), v).view(b, hq, n, d)
    return o / total.clamp(min=1e-38), (top + torch.log(total)).squeeze(-1)


def _prompt(s):
    q, k, v = s["q"], s["k"], s["v"]
    b = len(s["lens_q"])
    sq, pq = _rows(s["cu_q"], q.shape[0])
    sk, pk = _rows(s["cu_k"], k.shape[0])
    nq, nk = max(s["lens_q"]), max(s["lens_k"])
    o, lse = _attend(_padded(q, sq, pq, b, nq), _padded(k, sk, pk, b, nk), _padded(v, sk, pk, b, nk),
                     s["cu_q"].diff(), s["cu_k"].diff(), s["scale"])
    return {"out": o.transpose(1, 2)[sq, pq].to(q.dtype), "lse": lse.transpose(0, 1)[:, sq, pq]}


def _append_side(x, cache, scale, transposed, seq, place, table):
    """One side of the cache: x [rows, heads, d] to places `place` of sequences `seq`."""
    pages, heads = scale.shape
    codes = cache.transpose(-1, -2) if transposed else cache               # [pages, heads, 64, d]
    page = table[seq, place // PAGE].long()
    x = x.float()
    fine = torch.isfinite(x)
    mag = torch.where(fine, x.abs(), torch.zeros_like(x)).amax(-1)         # [rows, heads]
    top = torch.zeros(pages, heads, device=x.device)
    top.scatter_reduce_(0, page[:, None].expand(-1, heads), mag, "amax")
    hit = torch.zeros(pages, dtype=torch.bool, device=x.device).index_fill_(0, page, True)
    # a page whose first token is among the new ones held nothing before
    held = hit.index_fill(0, page[place % PAGE == 0], False)
    n127 = torch.full((), 127.0, device=x.device)
    fresh = torch.where(top < TINY, torch.zeros_like(top), top / n127)
    old = torch.where(held[:, None], scale, torch.zeros_like(scale))
    new = torch.maximum(old, fresh)
    grown = held[:, None] & (fresh > old)
    ratio = torch.where(grown, old / torch.where(grown, new, torch.ones_like(new)), torch.ones_like(new))
    touched = torch.nonzero(hit).squeeze(1)
    was = codes[touched].float()
    # the tokens that a page holds are requantized; what lies behind them is left as it was
    start = torch.full((pages,), PAGE, device=x.device, dtype=torch.int64)
    start.scatter_reduce_(0, page, place % PAGE, "amin")
    keep = torch.arange(PAGE, device=x.device)[None] < start[touched][:, None]
    moved = torch.where(keep[:, None, :, None], torch.round(was * ratio[touched][..., None, None]), was)
    codes[touched] = moved.to(torch.int8)
    inv = torch.where(new > 0, torch.reciprocal(torch.where(new > 0, new, torch.ones_like(new))), torch.zeros_like(new))
    y = torch.nan_to_num(x, nan=0.0, posinf=3e38, neginf=-3e38) * inv[page][..., None]
    codes[page, :, place % PAGE] = torch.round(y).clamp(-127, 127).to(torch.int8)
    scale[touched] = new[touched]


def _append(s):
    seq, i = _rows(s["cu_q"], s["k"].shape[0])
    place = s["cached"].long()[seq] + i
    _append_side(s["k"], s["k_cache"], s["k_scale"], False, seq, place, s["table"])
    _append_side(s["v"], s["v_cache"], s["v_scale"], True, seq, place, s["table"])
    return {"k_codes": s["k_cache"], "v_codes": s["v_cache"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _cache(s):
    q, table = s["q"], s["table"].long().clamp(min=0)
    b = len(s["lens_q"])
    sq, pq = _rows(s["cu_q"], q.shape[0])
    k = s["k_cache"][table].float() * s["k_scale"][table][..., None, None]      # [b, pages, heads, 64, d]
    k = k.transpose(1, 2).reshape(b, k.shape[2], -1, k.shape[4])
    v = s["v_cache"][table].float() * s["v_scale"][table][..., None, None]      # [b, pages, heads, d, 64]
    v = v.permute(0, 2, 1, 4, 3).reshape(k.shape)
    o, lse = _attend(_padded(q, sq, pq, b, max(s["lens_q"])), k, v, s["cu_q"].diff(), s["lens"], s["scale"])
    return {"out": o.transpose(1, 2)[sq, pq].to(q.dtype), "lse": lse.transpose(0, 1)[:, sq, pq]}


def _weights(s):
    q, table = s["q"], s["table"].long().clamp(min=0)
    b, hq, d = len(s["lens_q"]), q.shape[1], q.shape[2]
    sq, pq = _rows(s["cu_q"], q.shape[0])
    k = s["k_cache"][table].float() * s["k_scale"][table][..., None, None]
    k = k.transpose(1, 2).reshape(b, k.shape[2], -1, d)
    hkv, m, n = k.shape[1], k.shape[2], max(s["lens_q"])
    score = torch.matmul(_padded(q, sq, pq, b, n).reshape(b, hkv, -1, d) * s["scale"], k.transpose(-1, -2))
    lse = torch.full((b, n, hq), math.inf, device=q.device)
    lse[sq, pq] = s["lse"].t()
    at_q = torch.arange(n, device=q.device)[None, :, None] + (s["lens"] - s["cu_q"].diff())[:, None, None]
    hidden = torch.arange(m, device=q.device)[None, None] > at_q
    w = torch.exp_(score.view(b, hq, n, m).sub_(lse.transpose(1, 2)[..., None])).masked_fill_(hidden[:, None], 0.0)
    total = s["weights"].clone()
    total += w.view(b, hkv, -1, m).sum(2)[..., :total.shape[-1]]
    return {"weights": total}


def _evict(s):
    w, lens, keep, recent = s["weights"], s["lens"].long(), s["keep"], s["recent"]
    b, hkv, most = w.shape
    at = torch.arange(most, device=w.device)
    left = lens.clamp(max=keep)
    # the recent tokens first, then the others by weight, the earlier one of equals first; what is no token last
    rank = torch.where((at >= (lens - recent)[:, None])[:, None], torch.full_like(w, math.inf), w)
    rank = torch.where((at < lens[:, None])[:, None], rank, torch.full_like(w, -math.inf))
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices
    chosen = torch.zeros(b, hkv, most, dtype=torch.bool, device=w.device)
    chosen.scatter_(-1, order, (at < left[:, None])[:, None].expand(b, hkv, most))
    kept = torch.sort((~chosen).to(torch.int8), dim=-1, stable=True).indices[..., :keep]     # the kept ones, in order
    there = (torch.arange(kept.shape[-1], device=w.device) < left[:, None])[:, None].expand_as(kept)
    seq, head, place = torch.nonzero(there, as_tuple=True)
    src = kept[seq, head, place]
    old, new = s["table"][seq, src // PAGE].long(), s["new_table"][seq, place // PAGE].long()
    for codes, scale in ((s["k_cache"], s["k_scale"]), (s["v_cache"].transpose(-1, -2), s["v_scale"])):
        x = codes[old, head, src % PAGE].float() * scale[old, head][:, None]
        top = torch.zeros_like(scale).view(-1)
        top.scatter_reduce_(0, new * hkv + head, x.abs().amax(-1), "amax")
        top = top.view_as(scale)
        fresh = torch.where(top < TINY, torch.zeros_like(top), top / torch.full((), 127.0, device=w.device))
        inv = torch.where(fresh > 0, torch.reciprocal(fresh), torch.zeros_like(fresh))
        codes[new, head, place % PAGE] = torch.round(x * inv[new, head][:, None]).clamp(-127, 127).to(torch.int8)
        scale[new, head] = fresh[new, head]
    out = torch.zeros_like(w)
    out[seq, head, place] = w[seq, head, src]
    where = torch.full((b, hkv, keep), -1, dtype=torch.int32, device=w.device)
    where[..., :kept.shape[-1]] = torch.where(there, kept, torch.full_like(kept, -1)).to(torch.int32)
    return {"weights": out, "lens": left.to(torch.int32), "kept": where, "k_codes": s["k_cache"], "v_codes": s["v_cache"],
            "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


# ---------------------------------------------------------------------------
# from the definition, in 64 bits, one sequence and head at a time
# ---------------------------------------------------------------------------

def _exact_head(q, k, v, scale):
    """One head of one sequence: q [n, d], k, v [m, d]."""
    n, m = q.shape[0], k.shape[0]
    s = (q.double() @ k.double().t()) * scale
    s = s.masked_fill(torch.ones(n, m, dtype=torch.bool, device=q.device).triu(m - n + 1), -math.inf)
    lse = torch.logsumexp(s, 1)
    return torch.exp(s - lse[:, None]) @ v.double(), lse


def exact(case, seed):
    s = prepare(case, seed)
    q, k = s["lens_q"], s["lens_k"]
    hkv, d = case["hkv"], case["d"]
    if case["kind"] == "append":
        return _exact_append(s)
    if case["kind"] == "evict":
        return _exact_evict(s)
    hq = case["hq"]
    # a pass in 64 bits at some 20 TFLOP/s, and a launch or ten for each head of each sequence
    if sum(4.0 * n * m * d * hq for n, m in zip(q, k)) > 2e13 or len(q) * hq > 20000:
        return None
    out = torch.zeros(sum(q), hq, d, dtype=torch.float64, device="cuda")
    lse = torch.zeros(hq, sum(q), dtype=torch.float64, device="cuda")
    total = s["weights"].double() if case["kind"] == "weights" else None
    at_q = at_k = 0
    for b, (n, m) in enumerate(zip(q, k)):
        if case["kind"] == "prompt":
            keys, vals = s["k"][at_k:at_k + m], s["v"][at_k:at_k + m]
        else:
            page = s["table"][b, :-(-m // PAGE)].long()
            keys = s["k_cache"][page].double() * s["k_scale"][page].double()[..., None, None]
            keys = keys.transpose(1, 2).reshape(-1, hkv, d)[:m]
            vals = s["v_cache"][page].double() * s["v_scale"][page].double()[..., None, None]
            vals = vals.permute(0, 3, 1, 2).reshape(-1, hkv, d)[:m]
        for h in range(hq):
            g = h // (hq // hkv)
            if total is not None:
                total[b, g, :m] += _exact_weights(s["q"][at_q:at_q + n, h], keys[:, g], s["lse"][h, at_q:at_q + n], s["scale"])
                continue
            o, z = _exact_head(s["q"][at_q:at_q + n, h], keys[:, g], vals[:, g], s["scale"])
            out[at_q:at_q + n, h], lse[h, at_q:at_q + n] = o, z
        at_q, at_k = at_q + n, at_k + m
    return {"out": out, "lse": lse} if total is None else {"weights": total}


def _exact_weights(q, k, lse, scale):
    """What the queries of one head of one sequence give to each of its keys, by the lse in hand."""
    n, m = q.shape[0], k.shape[0]
    w = torch.exp((q.double() @ k.double().t()) * scale - lse.double()[:, None])
    return w.tril(m - n).sum(0)


def _exact_evict(s):
    """The scales and weights; the kept positions and the codes are whole numbers."""
    k_scale, v_scale = s["k_scale"].double(), s["v_scale"].double()
    out = torch.zeros_like(s["weights"], dtype=torch.float64)
    # the tokens' magnitudes, [pages, heads, 64]
    k_top = s["k_cache"].double().abs().amax(-1) * k_scale[..., None]
    v_top = s["v_cache"].double().abs().amax(-2) * v_scale[..., None]
    for b, m in enumerate(s["lens_k"]):
        fixed = max(0, m - s["recent"])
        more = min(s["keep"], m) - (m - fixed)
        pages = s["table"][b].long()
        for h in range(out.shape[1]):
            w = s["weights"][b, h, :m]
            best = torch.argsort(-w[:fixed], stable=True)[:more]
            at = torch.cat([torch.sort(best).values, torch.arange(fixed, m, device="cuda")])
            out[b, h, :len(at)] = w[at].double()
            for top, scale in ((k_top, k_scale), (v_top, v_scale)):
                mag = top[pages[at // PAGE], h, at % PAGE]
                full = torch.zeros(-(-len(at) // PAGE) * PAGE, dtype=torch.float64, device="cuda")
                full[:len(at)] = mag
                scale[s["new_table"][b, :full.numel() // PAGE].long(), h] = full.view(-1, PAGE).amax(1) / 127.0
    return {"weights": out, "lens": None, "kept": None, "k_codes": None, "v_codes": None, "k_scale": k_scale,
            "v_scale": v_scale}


def _exact_append(s):
    """The scales; the codes are whole numbers."""
    scales = {}
    for side in ("k", "v"):
        x, scale = s[side].double().abs().amax(-1), s[side + "_scale"].double().clone()
        at = 0
        for b, (n, m) in enumerate(zip(s["lens_q"], s["lens_k"])):
            for j in range(m // PAGE, -(-(m + n) // PAGE)):
                page = int(s["table"][b, j])
                first, last = max(j * PAGE, m) - m, min((j + 1) * PAGE, m + n) - m
                top = x[at + first:at + last].amax(0) / 127.0
                scale[page] = torch.maximum(scale[page], top) if j * PAGE < m else top
            at += n
        scales[side + "_scale"] = scale
    return {"k_codes": None, "v_codes": None, **scales}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    q, k, d, hkv = _lens(case["q"]) if case["kind"] != "evict" else [], _lens(case["k"]), case["d"], case["hkv"]
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "append":
        # rows in, codes out; a scale for each page and head; no read of what the pages hold, which only growth needs
        pages = sum(-(-(m + n) // PAGE) - m // PAGE for n, m in zip(q, k))
        return {"bytes": 2 * sum(q) * hkv * d * (size + 1) + 2 * pages * hkv * 4, "flops": 4 * sum(q) * hkv * d}
    if case["kind"] == "evict":
        # weights in and out, what is kept read and written with its position
        left = sum(min(m, case["keep"]) for m in k)
        return {"bytes": hkv * (4 * sum(k) + 4 * len(k) * (max(k) + case["keep"]) + 4 * left * d), "flops": 6 * left * hkv * d}
    hq = case["hq"]
    # pairs that the causal rule leaves
    pairs = sum(n * m - n * (n - 1) // 2 if m >= n else m * (m + 1) // 2 for n, m in zip(q, k))
    if case["kind"] == "weights":
        return {"bytes": sum(q) * hq * (d * size + 4) + sum(k) * hkv * (d + 8), "flops": 2 * pairs * hq * d}
    rows = sum(q) * hq * (2 * d * size + 4)
    kv = 2 * sum(k) * hkv * (d * size if case["kind"] == "prompt" else d)
    if case["kind"] == "cache":
        kv += 2 * sum(-(-m // PAGE) for m in k) * hkv * 4
    return {"bytes": rows + kv, "flops": 4 * pairs * hq * d}
