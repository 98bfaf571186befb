"""Attention between a decoder layer's q/k/v and o linears, and the paged int8 cache that it reads.

torch custom ops over libparoquant_hip.so (namespace ``paroquant_attn``), each with a function of the same name here:

  prompt_attention(q, k, v, cu_seqlens_q, cu_seqlens_k=None, scale=None, causal=True) -> (out, lse)
      packed prompts of different lengths, grouped heads
  kv_append_i8(k, v, k_cache, v_cache, k_scale, v_scale, block_table, cu_seqlens, cached_lens)
      new tokens' keys and values into the cache
  cache_attention_i8(q, k_cache, v_cache, k_scale, v_scale, block_table, cu_seqlens_q, lens, scale=None) -> (out, lse)
      each sequence's last tokens over the cache: decode, verify blocks, chunks
  cache_weights_i8(q, k_cache, k_scale, block_table, cu_seqlens_q, lens, lse, weights, scale=None)
      adds the softmax weights of that call to a sum for each cached token
  cache_evict_i8(k_cache, v_cache, k_scale, v_scale, weights, block_table, lens, new_table, keep, recent)
          -> (weights, lens, kept)
      cuts each head's cache to the recent tokens and those with the largest sums

``PagedKVCacheI8`` holds a cache's tensors and has these calls as methods.

Packed rows: q is [tokens, query heads, d], k and v [tokens, key/value heads, d], d = 64 or 128, any strides of tokens and
heads (views of a fused projection need no copy while rows are 16-byte aligned).  Sequence b has rows
cu_seqlens[b] .. cu_seqlens[b + 1] - 1.  Query head h reads key/value head h // (query heads / key/value heads).  Rows
outside of the sequences, and rows that see no key, get zeros and lse = -inf.

The cache: k_cache int8 [pages, heads, 64, d], v_cache int8 [pages, heads, d, 64], k_scale and v_scale float32
[pages, heads]; a value is code * scale.  Token i of sequence b is in page block_table[b, i // 64]; a page number outside
of [0, pages) is no page: tokens that would go there are dropped, and attention does not see them.

Lengths and page numbers are int32 tensors on the device: nothing here reads them on the host, so the calls never wait
and a captured graph serves other lengths in the same buffers.  As everywhere in this package the kernels run on the
current stream of the tensors' device, outputs and scratch come from torch's allocator, and there is no CPU
implementation.  None of the ops has a backward pass: like the quantized linears around them they serve, and inputs
that record gradients are refused.
"""

from __future__ import annotations

import torch

from . import _lib
from .ops import _DT, _DeviceGuard, _same_device, _stream

PAGE = 64
_HALF = (torch.float16, torch.bfloat16)

_attn_lib = torch.library.Library("paroquant_attn", "DEF")
_attn_lib.define("prompt_attention(Tensor q, Tensor k, Tensor v, Tensor cu_seqlens_q, Tensor? cu_seqlens_k=None, "
                 "float? scale=None, bool causal=True) -> (Tensor, Tensor)")
_attn_lib.define("kv_append_i8(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scale, "
                 "Tensor(d!) v_scale, Tensor block_table, Tensor cu_seqlens, Tensor cached_lens) -> ()")
_attn_lib.define("cache_attention_i8(Tensor q, Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale, "
                 "Tensor block_table, Tensor cu_seqlens_q, Tensor lens, float? scale=None) -> (Tensor, Tensor)")
_attn_lib.define("cache_weights_i8(Tensor q, Tensor k_cache, Tensor k_scale, Tensor block_table, Tensor cu_seqlens_q, "
                 "Tensor lens, Tensor lse, Tensor(a!) weights, float? scale=None) -> ()")
_attn_lib.define("cache_evict_i8(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scale, Tensor(d!) v_scale, "
                 "Tensor weights, Tensor block_table, Tensor lens, Tensor new_table, int keep, int recent) "
                 "-> (Tensor, Tensor, Tensor)")


# ---------------------------------------------------------------------------
# checks
# ---------------------------------------------------------------------------

def _no_grad(who, *tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                raise RuntimeError(f"{who} has no backward pass: detach its inputs or call it under torch.no_grad()")


def _heads3(name, t, dtypes):
    """Checks packed rows [tokens, heads, d]; a copy where the kernels' 16-byte loads could not take t as it lies."""
    if t.dtype not in dtypes:
        raise RuntimeError(f"{name} must be one of {', '.join(str(d) for d in dtypes)}, got {t.dtype}")
    if t.dim() != 3 or t.size(2) not in (64, 128) or t.size(1) < 1:
        raise RuntimeError(f"{name} must be [tokens, heads, 64 or 128], got {tuple(t.shape)}")
    per = 16 // t.element_size()
    st = t.stride()
    if st[2] != 1 or st[0] % per or st[1] % per or t.data_ptr() % 16:
        t = t.contiguous() if not t.is_contiguous() else t.clone()
    return t


def _index(name, t, shape, dev):
    """An int32 tensor of this shape (None: any size) on the rows' device, contiguous."""
    if t.dtype != torch.int32:
        raise RuntimeError(f"{name} must be int32, got {t.dtype}")
    if t.dim() != len(shape) or any(n is not None and n != m for n, m in zip(shape, t.shape)):
        raise RuntimeError(f"{name} must be {[n if n is not None else '*' for n in shape]}, got {tuple(t.shape)}")
    _same_device(name, t, dev)
    return t.contiguous()


def _cu(name, t, dev):
    t = _index(name, t, (None,), dev)
    if t.numel() < 1:
        raise RuntimeError(f"{name} must hold batch + 1 offsets, got none")
    return t


def _codes(name, t, pages, heads, rows, cols, dev):
    shape = (pages, heads, rows, cols)
    if t.dtype != torch.int8 or tuple(t.shape) != shape:
        raise RuntimeError(f"{name} must be int8 {shape}, got {t.dtype} {tuple(t.shape)}")
    if not t.is_contiguous() or t.data_ptr() % 16:
        raise RuntimeError(f"{name} must be contiguous and 16-byte aligned")
    _same_device(name, t, dev)


def _scales(name, t, pages, heads, dev):
    if t.dtype != torch.float32 or tuple(t.shape) != (pages, heads) or not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous float32 {(pages, heads)}, got {t.dtype} {tuple(t.shape)}")
    _same_device(name, t, dev)


def _cache_dims(k_cache):
    if k_cache.dim() != 4 or k_cache.size(2) != PAGE or k_cache.size(3) not in (64, 128) or k_cache.size(1) < 1:
        raise RuntimeError(f"k_cache must be int8 [pages, heads, {PAGE}, 64 or 128], got {tuple(k_cache.shape)}")
    return k_cache.size(0), k_cache.size(1), k_cache.size(3)


def _pools(k_cache, v_cache, k_scale, v_scale, dev):
    pages, heads, d = _cache_dims(k_cache)
    _codes("k_cache", k_cache, pages, heads, PAGE, d, dev)
    _codes("v_cache", v_cache, pages, heads, d, PAGE, dev)
    _scales("k_scale", k_scale, pages, heads, dev)
    _scales("v_scale", v_scale, pages, heads, dev)
    return pages, heads, d


def _group(name, q, heads, d):
    if q.size(2) != d:
        raise RuntimeError(f"{name} has {q.size(2)} channels a head, the keys have {d}")
    if q.size(1) % heads:
        raise RuntimeError(f"{name} has {q.size(1)} heads, not a multiple of the {heads} key/value heads")
    return q.size(1) // heads


def _scale(scale, d):
    if scale is None:
        return d ** -0.5
    if not 0.0 < scale < float("inf"):
        raise RuntimeError(f"scale={scale} must be positive and finite")
    return float(scale)


def _ptr(t):
    return t.data_ptr() if t.numel() else None


# ---------------------------------------------------------------------------
# prompt_attention
# ---------------------------------------------------------------------------

def _prompt_impl(q, k, v, cu_seqlens_q, cu_seqlens_k=None, scale=None, causal=True):
    dev = q.device
    _no_grad("prompt_attention", q, k, v)
    q = _heads3("q", q, _HALF)
    k, v = _heads3("k", k, (q.dtype,)), _heads3("v", v, (q.dtype,))
    _same_device("k", k, dev)
    _same_device("v", v, dev)
    if k.shape != v.shape:
        raise RuntimeError(f"k and v must have one shape, got {tuple(k.shape)} and {tuple(v.shape)}")
    heads, d = k.size(1), k.size(2)
    group = _group("q", q, heads, d)
    cq = _cu("cu_seqlens_q", cu_seqlens_q, dev)
    if cu_seqlens_k is None:
        if k.size(0) != q.size(0):
            raise RuntimeError(f"q has {q.size(0)} rows and k {k.size(0)}: give cu_seqlens_k")
        ck = cq
    else:
        ck = _index("cu_seqlens_k", cu_seqlens_k, (cq.numel(),), dev)
    sc = _scale(scale, d)
    out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    lse = torch.empty((q.size(1), q.size(0)), dtype=torch.float32, device=dev)
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    with _DeviceGuard(dev):
        st = _lib.load().pq_attn_prompt(_ptr(q), _ptr(k), _ptr(v), _DT[q.dtype], qs[0], qs[1], ks[0], ks[1], vs[0],
                                        vs[1], cq.data_ptr(), ck.data_ptr(), _ptr(out), _ptr(lse), cq.numel() - 1,
                                        q.size(0), k.size(0), heads, group, d, sc, bool(causal), _stream(dev))
    _lib.check(st, "paroquant_attn::prompt_attention")
    return out, lse


_attn_lib.impl("prompt_attention", _prompt_impl, "CUDA")


@torch.library.register_fake("paroquant_attn::prompt_attention")
def _prompt_fake(q, k, v, cu_seqlens_q, cu_seqlens_k=None, scale=None, causal=True):
    return q.new_empty(q.shape), q.new_empty((q.size(1), q.size(0)), dtype=torch.float32)


def prompt_attention(q, k, v, cu_seqlens_q, cu_seqlens_k=None, scale=None, causal=True):
    """Attention of packed prompts: (out [tokens, query heads, d], lse float32 [query heads, tokens]).

    Causal: the last query of a sequence sees all of its keys, the one before all but the last, and so on; with fewer
    queries than keys (a chunk of a prompt) that is the chunk at the prompt's end, with more the first queries see
    nothing.  cu_seqlens_k: the keys' offsets where they differ from the queries'.  scale: 1 / sqrt(d) by default.
    lse is the natural logarithm of each row's sum of exp(scale * q . k).  A value of k or v that a row does not see
    has no effect on it, whatever it is."""
    return torch.ops.paroquant_attn.prompt_attention.default(q, k, v, cu_seqlens_q, cu_seqlens_k, scale, causal)


# ---------------------------------------------------------------------------
# kv_append_i8
# ---------------------------------------------------------------------------

def _append_impl(k, v, k_cache, v_cache, k_scale, v_scale, block_table, cu_seqlens, cached_lens):
    dev = k.device
    _no_grad("kv_append_i8", k, v)
    k = _heads3("k", k, tuple(_DT))
    v = _heads3("v", v, (k.dtype,))
    _same_device("v", v, dev)
    pages, heads, d = _pools(k_cache, v_cache, k_scale, v_scale, dev)
    if k.shape != v.shape or k.size(1) != heads or k.size(2) != d:
        raise RuntimeError(f"k and v must be [tokens, {heads}, {d}] as the cache, got {tuple(k.shape)} and {tuple(v.shape)}")
    cu = _cu("cu_seqlens", cu_seqlens, dev)
    batch = cu.numel() - 1
    table = _index("block_table", block_table, (batch, None), dev)
    cached = _index("cached_lens", cached_lens, (batch,), dev)
    ks, vs = k.stride(), v.stride()
    with _DeviceGuard(dev):
        st = _lib.load().pq_kv_append_i8(_ptr(k), _ptr(v), _DT[k.dtype], ks[0], ks[1], vs[0], vs[1], _ptr(k_cache),
                                         _ptr(v_cache), _ptr(k_scale), _ptr(v_scale), _ptr(table), cu.data_ptr(),
                                         _ptr(cached), batch, table.size(1), k.size(0), heads, d, pages, _stream(dev))
    _lib.check(st, "paroquant_attn::kv_append_i8")


_attn_lib.impl("kv_append_i8", _append_impl, "CUDA")


@torch.library.register_fake("paroquant_attn::kv_append_i8")
def _append_fake(k, v, k_cache, v_cache, k_scale, v_scale, block_table, cu_seqlens, cached_lens):
    return None


def kv_append_i8(k, v, k_cache, v_cache, k_scale, v_scale, block_table, cu_seqlens, cached_lens):
    """Puts row i of sequence b at place cached_lens[b] + i of its pages (float32, float16 or bfloat16 rows).

    A page's scale for a head is the absmax of what it holds / 127, a code round(x / scale).  Where new tokens are larger
    than what their page holds, its codes are rounded to the new scale; a page whose first token is new starts afresh.
    NaN is held as 0, infinities as the largest code.  The lengths are the caller's to advance.  A page may belong to
    one sequence of the call only."""
    torch.ops.paroquant_attn.kv_append_i8.default(k, v, k_cache, v_cache, k_scale, v_scale, block_table, cu_seqlens,
                                                  cached_lens)


# ---------------------------------------------------------------------------
# cache_attention_i8, cache_weights_i8
# ---------------------------------------------------------------------------

def _cache_attn_impl(q, k_cache, v_cache, k_scale, v_scale, block_table, cu_seqlens_q, lens, scale=None):
    dev = q.device
    _no_grad("cache_attention_i8", q)
    q = _heads3("q", q, _HALF)
    pages, heads, d = _pools(k_cache, v_cache, k_scale, v_scale, dev)
    group = _group("q", q, heads, d)
    cu = _cu("cu_seqlens_q", cu_seqlens_q, dev)
    batch, tokens = cu.numel() - 1, q.size(0)
    table = _index("block_table", block_table, (batch, None), dev)
    ln = _index("lens", lens, (batch,), dev)
    sc = _scale(scale, d)
    out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    lse = torch.empty((q.size(1), tokens), dtype=torch.float32, device=dev)
    lib = _lib.load()
    need = int(lib.pq_attn_cache_i8_workspace_size(batch, tokens, group, d))
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    qs = q.stride()
    with _DeviceGuard(dev):
        st = lib.pq_attn_cache_i8(_ptr(q), _DT[q.dtype], qs[0], qs[1], _ptr(k_cache), _ptr(v_cache), _ptr(k_scale),
                                  _ptr(v_scale), _ptr(table), cu.data_ptr(), _ptr(ln), _ptr(out), _ptr(lse), batch,
                                  table.size(1), tokens, heads, group, d, pages, sc,
                                  ws.data_ptr() if ws is not None else None, need, _stream(dev))
    _lib.check(st, "paroquant_attn::cache_attention_i8")
    return out, lse


_attn_lib.impl("cache_attention_i8", _cache_attn_impl, "CUDA")


@torch.library.register_fake("paroquant_attn::cache_attention_i8")
def _cache_attn_fake(q, k_cache, v_cache, k_scale, v_scale, block_table, cu_seqlens_q, lens, scale=None):
    return q.new_empty(q.shape), q.new_empty((q.size(1), q.size(0)), dtype=torch.float32)


def cache_attention_i8(q, k_cache, v_cache, k_scale, v_scale, block_table, cu_seqlens_q, lens, scale=None):
    """Attention of each sequence's last tokens over its cache: (out [tokens, query heads, d], lse float32
    [query heads, tokens]), in bfloat16 or float16.

    lens[b]: tokens of sequence b in the cache, the new ones among them.  Its last query sees all of them, the one
    before all but the last, and so on."""
    return torch.ops.paroquant_attn.cache_attention_i8.default(q, k_cache, v_cache, k_scale, v_scale, block_table,
                                                               cu_seqlens_q, lens, scale)


def _cache_weights_impl(q, k_cache, k_scale, block_table, cu_seqlens_q, lens, lse, weights, scale=None):
    dev = q.device
    _no_grad("cache_weights_i8", q, lse, weights)
    q = _heads3("q", q, _HALF)
    pages, heads, d = _cache_dims(k_cache)
    _codes("k_cache", k_cache, pages, heads, PAGE, d, dev)
    _scales("k_scale", k_scale, pages, heads, dev)
    group = _group("q", q, heads, d)
    cu = _cu("cu_seqlens_q", cu_seqlens_q, dev)
    batch, tokens = cu.numel() - 1, q.size(0)
    table = _index("block_table", block_table, (batch, None), dev)
    ln = _index("lens", lens, (batch,), dev)
    if lse.dtype != torch.float32 or tuple(lse.shape) != (q.size(1), tokens):
        raise RuntimeError(f"lse must be float32 {(q.size(1), tokens)}, got {lse.dtype} {tuple(lse.shape)}")
    _same_device("lse", lse, dev)
    lse = lse.contiguous()
    _check_weights(weights, batch, heads, dev)
    if not weights.is_contiguous():
        raise RuntimeError("weights must be contiguous")
    sc = _scale(scale, d)
    qs = q.stride()
    with _DeviceGuard(dev):
        st = _lib.load().pq_attn_cache_weights_i8(_ptr(q), _DT[q.dtype], qs[0], qs[1], _ptr(k_cache), _ptr(k_scale),
                                                  _ptr(table), cu.data_ptr(), _ptr(ln), _ptr(lse), _ptr(weights), batch,
                                                  table.size(1), weights.size(2), tokens, heads, group, d, pages, sc,
                                                  _stream(dev))
    _lib.check(st, "paroquant_attn::cache_weights_i8")


def _check_weights(weights, batch, heads, dev):
    if weights.dtype != torch.float32 or weights.dim() != 3 or weights.size(0) != batch or weights.size(1) != heads:
        raise RuntimeError(f"weights must be float32 [{batch}, {heads}, tokens], got {weights.dtype} {tuple(weights.shape)}")
    _same_device("weights", weights, dev)


_attn_lib.impl("cache_weights_i8", _cache_weights_impl, "CUDA")


@torch.library.register_fake("paroquant_attn::cache_weights_i8")
def _cache_weights_fake(q, k_cache, k_scale, block_table, cu_seqlens_q, lens, lse, weights, scale=None):
    return None


def cache_weights_i8(q, k_cache, k_scale, block_table, cu_seqlens_q, lens, lse, weights, scale=None):
    """weights[b, head, j] += sum of exp(scale * q . k_j - lse) over sequence b's rows of the head that see token j.

    q, lengths and scale are those of a cache_attention_i8 call and lse what it returned, so the sum is over its softmax
    weights.  weights: float32 [batch, key/value heads, tokens], contiguous; tokens past its end are left out.  Sums
    are taken in a fixed order."""
    torch.ops.paroquant_attn.cache_weights_i8.default(q, k_cache, k_scale, block_table, cu_seqlens_q, lens, lse, weights,
                                                      scale)


# ---------------------------------------------------------------------------
# cache_evict_i8
# ---------------------------------------------------------------------------

def _evict_impl(k_cache, v_cache, k_scale, v_scale, weights, block_table, lens, new_table, keep, recent):
    dev = k_cache.device
    _no_grad("cache_evict_i8", weights)
    pages, heads, d = _pools(k_cache, v_cache, k_scale, v_scale, dev)
    ln = _index("lens", lens, (None,), dev)
    batch = ln.numel()
    table = _index("block_table", block_table, (batch, None), dev)
    new = _index("new_table", new_table, (batch, None), dev)
    _check_weights(weights, batch, heads, dev)
    if not 0 <= recent <= keep or keep < 1:
        raise RuntimeError(f"keep={keep} must be at least 1 and recent={recent} within 0..keep")
    w = weights.contiguous()
    out = torch.empty_like(w)
    new_lens = torch.empty_like(ln)
    kept = torch.empty((batch, heads, keep), dtype=torch.int32, device=dev)
    with _DeviceGuard(dev):
        st = _lib.load().pq_kv_evict_i8(_ptr(k_cache), _ptr(v_cache), _ptr(k_scale), _ptr(v_scale), _ptr(w), _ptr(table),
                                        _ptr(ln), _ptr(new), _ptr(out), _ptr(new_lens), _ptr(kept), batch, table.size(1),
                                        new.size(1), w.size(2), heads, d, pages, keep, recent, _stream(dev))
    _lib.check(st, "paroquant_attn::cache_evict_i8")
    return out, new_lens, kept


_attn_lib.impl("cache_evict_i8", _evict_impl, "CUDA")


@torch.library.register_fake("paroquant_attn::cache_evict_i8")
def _evict_fake(k_cache, v_cache, k_scale, v_scale, weights, block_table, lens, new_table, keep, recent):
    return (weights.new_empty(weights.shape), lens.new_empty(lens.shape),
            lens.new_empty((weights.size(0), weights.size(1), keep)))


def cache_evict_i8(k_cache, v_cache, k_scale, v_scale, weights, block_table, lens, new_table, keep, recent):
    """Cuts the cache of each sequence and head to `keep` tokens, its last `recent` ones and those before them with the
    largest weights (of equals the earlier ones; NaN counts as the lowest): (weights, lens, kept).

    What is kept moves in order to the front of the pages that new_table names, which no sequence of the call may be
    using; the old pages are the caller's to free.  Codes are rounded to the new pages' scales.  Returned: the kept
    tokens' weights in their new places with zeros behind, as large as `weights`; the new lengths; and the kept tokens'
    old places, int32 [batch, heads, keep], -1 behind the last.  A sequence of `keep` tokens or fewer is moved whole.
    Tokens past the end of block_table or of `weights` do not count."""
    return torch.ops.paroquant_attn.cache_evict_i8.default(k_cache, v_cache, k_scale, v_scale, weights, block_table, lens,
                                                           new_table, keep, recent)


class PagedKVCacheI8:
    """The tensors of a paged int8 cache of one layer, and the calls that write and read them.

    Pages are the caller's to hand out: block_table int32 [batch, pages a sequence may have] names each sequence's."""

    def __init__(self, pages: int, kv_heads: int, head_dim: int, device="cuda"):
        if head_dim not in (64, 128) or kv_heads < 1 or pages < 0:
            raise RuntimeError(f"pages={pages} kv_heads={kv_heads} head_dim={head_dim} (64 or 128)")
        self.k_cache = torch.zeros((pages, kv_heads, PAGE, head_dim), dtype=torch.int8, device=device)
        self.v_cache = torch.zeros((pages, kv_heads, head_dim, PAGE), dtype=torch.int8, device=device)
        self.k_scale = torch.zeros((pages, kv_heads), dtype=torch.float32, device=device)
        self.v_scale = torch.zeros((pages, kv_heads), dtype=torch.float32, device=device)

    @property
    def pools(self):
        return self.k_cache, self.v_cache, self.k_scale, self.v_scale

    @staticmethod
    def pages_for(tokens: int) -> int:
        return -(-tokens // PAGE)

    def append(self, k, v, block_table, cu_seqlens, cached_lens) -> None:
        kv_append_i8(k, v, *self.pools, block_table, cu_seqlens, cached_lens)

    def attention(self, q, block_table, cu_seqlens_q, lens, scale=None):
        return cache_attention_i8(q, *self.pools, block_table, cu_seqlens_q, lens, scale)

    def add_weights(self, q, block_table, cu_seqlens_q, lens, lse, weights, scale=None) -> None:
        cache_weights_i8(q, self.k_cache, self.k_scale, block_table, cu_seqlens_q, lens, lse, weights, scale)

    def evict(self, weights, block_table, lens, new_table, keep, recent):
        return cache_evict_i8(*self.pools, weights, block_table, lens, new_table, keep, recent)
