"""prompt_attention, the paged int8 cache and what reads it, against the float64 / bit-exact oracle (oracle/attention.py).

Tolerances: u is half a step of the type (bf16 2^-8, fp16 2^-11).  An output is a sum of p v with p rounded once (u of the
type p is held in, and 2^-25 of the largest weight where an fp16 p is subnormal) and rounded once itself; a score is a
float32 sum of d products and p its exponential, which turns an absolute error of the score into a relative one of p,
once in the sum above and once in the sum below."""

import numpy as np
import pytest
import torch

import alpamayo_amd  # noqa: F401
from alpamayo_amd import attention
from oracle import attention as oatt

pytestmark = pytest.mark.gpu

PAGE = 64
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
BF, HF = torch.bfloat16, torch.float16


def _np(t):
    return t.detach().cpu().float().numpy() if t.is_floating_point() else t.detach().cpu().numpy()


def _rand(gen, *shape, dtype=BF, amp=1.0):
    return (torch.randn(*shape, generator=gen) * amp).to(dtype)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _cu(lens):
    return torch.tensor(np.cumsum([0] + list(lens)), dtype=torch.int32)


def _score_error(qn, kn, scale):
    """Bound of a float32 score's error: d products and sums, and the roundings of scaling and exponential."""
    d = qn.shape[-1]
    top = np.abs(qn).max() * np.abs(kn[np.isfinite(kn)]).max() * d * scale if kn.size and qn.size else 0.0
    return (d + 16) * 2.0 ** -24 * top + 2.0 ** -20


def _check(out, lse, ref, dtype, p_type, delta, vmax, n):
    o, z, mag = ref
    got, gz = _np(out).astype(np.float64), _np(lse).astype(np.float64)
    up, uo = U[p_type], U[dtype]
    tol = (up + 3 * delta + n * 2.0 ** -23) * mag + uo * np.abs(o) + 2.0 ** -25 * n * vmax + 1e-30
    tol *= 1 + uo
    bad = ~(np.abs(got - o) <= tol)
    assert not bad.any(), f"{bad.sum()} of {bad.size} out by up to {np.abs(got - o)[bad].max():.3e}, e.g. at {np.argwhere(bad)[0]}"
    inf = np.isneginf(z)
    assert np.array_equal(inf, np.isneginf(gz))
    dz = np.abs(gz[~inf] - z[~inf])
    assert (dz <= delta + n * 2.0 ** -23 + 2.0 ** -21 * np.abs(z[~inf])).all(), dz.max()


def _prompt_case(lens_q, lens_k, hq, hkv, d, dtype, causal=True, scale=None, seed=0, amp=1.0, tail=0, strided=False):
    g = _gen(seed)
    tq, tk = sum(lens_q) + tail, sum(lens_k) + tail
    if strided:
        # q, k, v as slices of one fused projection, the heads of k and v interleaved
        fused = _rand(g, tq, (hq + 2 * hkv) * d, dtype=dtype, amp=amp).cuda()
        q = fused[:, :hq * d].view(tq, hq, d)
        k = fused[:, hq * d:].view(tq, hkv, 2, d)[:, :, 0]
        v = fused[:, hq * d:].view(tq, hkv, 2, d)[:, :, 1]
        assert lens_q == lens_k
    else:
        q, k, v = (_rand(g, t, h, d, dtype=dtype, amp=amp).cuda() for t, h in ((tq, hq), (tk, hkv), (tk, hkv)))
    cq, ck = _cu(lens_q), _cu(lens_k)
    sc = d ** -0.5 if scale is None else scale
    print(f"prompt q={lens_q} k={lens_k} heads {hq}/{hkv} d={d} {dtype} causal={causal} tail={tail}", flush=True)
    out, lse = attention.prompt_attention(q, k, v, cq.cuda(), ck.cuda(), scale=scale, causal=causal)
    torch.cuda.synchronize()
    qn, kn, vn = _np(q), _np(k), _np(v)
    ref = oatt.packed_attention(qn, kn, vn, cq.numpy(), ck.numpy(), sc, causal)
    _check(out, lse, ref, dtype, dtype, _score_error(qn, kn, sc), np.abs(vn).max(), max(lens_k + [1]))
    if tail:
        assert (out[sum(lens_q):] == 0).all() and torch.isneginf(lse[:, sum(lens_q):]).all()
    return q, k, v, cq, ck, out, lse


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens,hq,hkv", [
    ([1], 1, 1), ([2, 1, 3], 4, 2), ([63, 64, 65], 4, 1), ([31, 0, 33, 97], 6, 2), ([129, 1, 128], 2, 2), ([200], 7, 1),
    ([5] * 70, 2, 1),
])
def test_prompt_lengths_and_heads(lens, hq, hkv, d, dtype):
    _prompt_case(lens, lens, hq, hkv, d, dtype, seed=len(lens) + d)


@pytest.mark.parametrize("lens_q,lens_k", [([1], [300]), ([64, 7], [65, 200]), ([100], [37]), ([3, 4], [0, 2]), ([150, 20], [150, 0])])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_other_key_lengths(lens_q, lens_k, causal):
    """Chunks of prompts, and more queries than keys: the first rows see nothing."""
    _prompt_case(lens_q, lens_k, 4, 2, 128, BF, causal=causal, seed=3)


@pytest.mark.parametrize("d,dtype", [(64, BF), (128, HF)])
@pytest.mark.parametrize("lens_q,lens_k", [([5], [3000]), ([130, 1], [1990, 4003]), ([64, 0, 3], [2500, 700, 2600]), ([900], [900])])
def test_prompt_keys_split_over_workgroups(lens_q, lens_k, d, dtype):
    """Few rows on many keys: parts of the keys, joined; some rows see nothing of the later parts."""
    need = attention._lib.load().pq_attn_prompt_workspace_size(len(lens_q), sum(lens_q) + 2, sum(lens_k) + 2, 2, 2, d)
    assert need > 0, "the case is meant to be split"
    _prompt_case(lens_q, lens_k, 4, 2, d, dtype, tail=2, seed=sum(lens_q))


def test_prompt_rows_outside_sequences():
    _prompt_case([40, 30], [40, 30], 4, 2, 128, BF, tail=37, seed=5)
    _prompt_case([0], [0], 4, 2, 64, HF, tail=200, seed=5)


def test_prompt_strided_views():
    _prompt_case([70, 65], [70, 65], 4, 2, 128, BF, strided=True, seed=6)
    _prompt_case([33], [33], 3, 3, 64, HF, strided=True, seed=7)


@pytest.mark.parametrize("amp,scale", [(30.0, None), (0.01, None), (4.0, 3.0)])
def test_prompt_sharp_and_flat_scores(amp, scale):
    """Scores of thousands (one weight takes all), and of nothing (all alike)."""
    _prompt_case([150], [150], 2, 1, 64, HF, amp=amp, scale=scale, seed=8)


def test_prompt_long_row_maximum_moves():
    """Keys that grow along the prompt: the running maximum moves in every tile, by more than exp can hold."""
    g, d, n = _gen(9), 64, 400
    q = torch.ones(n, 1, d, dtype=HF)
    k = (torch.arange(n, dtype=torch.float32)[:, None, None] * 0.05 * torch.ones(1, 1, d)).to(HF)
    v = _rand(g, n, 1, d, dtype=HF)
    cu = _cu([n])
    for kk in (k, k.flip(0)):
        out, lse = attention.prompt_attention(q.cuda(), kk.cuda(), v.cuda(), cu.cuda())
        ref = oatt.packed_attention(_np(q), _np(kk), _np(v), cu.numpy(), cu.numpy(), d ** -0.5)
        _check(out, lse, ref, HF, HF, _score_error(_np(q), _np(kk), d ** -0.5), _np(v).max(), n)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_prompt_what_a_row_does_not_see_has_no_effect(bad, dtype):
    """Key and value `at` hold values that are not finite: rows before it, other sequences and other heads keep their bits."""
    lens, d, at = [100, 90], 128, 75
    g = _gen(11)
    q, k, v = (_rand(g, 190, h, d, dtype=dtype).cuda() for h in (4, 2, 2))
    cu = _cu(lens).cuda()
    good, _ = attention.prompt_attention(q, k, v, cu)
    k2, v2 = k.clone(), v.clone()
    k2[at, 0, 5] = bad
    v2[at, 0, 7] = bad
    out, _ = attention.prompt_attention(q, k2, v2, cu)
    assert torch.equal(out[:at, :2], good[:at, :2]) and torch.equal(out[:, 2:], good[:, 2:])
    assert torch.equal(out[100:], good[100:])
    v3 = v.clone()
    v3[at, 0, 7] = bad
    out, _ = attention.prompt_attention(q, k, v3, cu)
    seen = out[at:100, :2, 7].float()
    assert (seen.isnan() if bad != bad else seen == bad).all()
    keep = torch.ones(d, dtype=torch.bool)
    keep[7] = False
    assert torch.equal(out[:, :, keep], good[:, :, keep])


# ---------------------------------------------------------------------------
# the cache
# ---------------------------------------------------------------------------

def _pools(gen, pages, heads, d, garbage=True):
    """Pools that hold something in every byte."""
    k = torch.randint(-127, 128, (pages, heads, PAGE, d), generator=gen, dtype=torch.int8)
    v = torch.randint(-127, 128, (pages, heads, d, PAGE), generator=gen, dtype=torch.int8)
    ks, vs = (torch.rand(pages, heads, generator=gen) * 0.02 + 0.005 for _ in range(2))
    return k, v, ks, vs


def _table(gen, batch, width, pages):
    assert batch * width <= pages
    return torch.randperm(pages, generator=gen)[:batch * width].view(batch, width).to(torch.int32)


def _cuda(*ts):
    return tuple(t.cuda() for t in ts)


def _same_cache(pools, ref):
    for got, want, name in zip(pools, (ref.k, ref.v, ref.ks, ref.vs), ("k_cache", "v_cache", "k_scale", "v_scale")):
        assert np.array_equal(got.cpu().numpy(), want), f"{name}: {(got.cpu().numpy() != want).sum()} differ"


@pytest.mark.parametrize("dtype", [torch.float32, HF, BF])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads", [1, 3])
def test_append_bits(dtype, d, heads):
    """Fresh pages, pages in the middle, growth and no growth, one token and several pages: every byte of the pools."""
    new, held = [1, 64, 130, 0, 5, 63, 1], [0, 0, 10, 7, 63, 64, 127]
    g = _gen(d + heads)
    pools = _pools(g, 40, heads, d)
    table = _table(g, 7, 4, 40)
    ref = oatt.Cache(*(p.numpy() for p in pools))
    dev = _cuda(*pools)
    cached = torch.tensor(held, dtype=torch.int32)
    cu = _cu(new)
    for step, amp in enumerate((0.1, 1.0, 20.0)):       # below, about and above what the pages hold
        k, v = (_rand(g, sum(new) + 3, heads, d, dtype=dtype, amp=amp) for _ in range(2))
        print(f"append d={d} heads={heads} {dtype} amp={amp}", flush=True)
        attention.kv_append_i8(*_cuda(k, v), *dev, *_cuda(table, cu, cached))
        ref.append(_np(k), _np(v), table.numpy(), cu.numpy(), cached.numpy())
        _same_cache(dev, ref)


def test_append_values_that_are_not_finite_and_tiny_ones():
    g, d = _gen(2), 64
    pools = _pools(g, 6, 2, d)
    ref = oatt.Cache(*(p.numpy() for p in pools))
    dev = _cuda(*pools)
    table = torch.tensor([[3, 1], [0, 5]], dtype=torch.int32)
    k, v = _rand(g, 80, 2, d, dtype=torch.float32), _rand(g, 80, 2, d, dtype=torch.float32)
    k[3, 0, 1], k[4, 0, 2], k[5, 1, 3], v[6, 0, 1] = float("nan"), float("inf"), -float("inf"), float("nan")
    k[70:80], v[70:80, 0] = 0.0, 1e-38
    v[70:80, 1] = float("nan")
    cu, cached = _cu([70, 10]), torch.tensor([0, 64], dtype=torch.int32)
    attention.kv_append_i8(*_cuda(k, v), *dev, *_cuda(table, cu, cached))
    ref.append(k.numpy(), v.numpy(), table.numpy(), cu.numpy(), cached.numpy())
    _same_cache(dev, ref)
    assert np.isfinite(ref.ks).all()


def test_append_pages_that_do_not_exist_and_ends_of_the_table():
    g, d = _gen(4), 128
    pools = _pools(g, 5, 2, d)
    ref = oatt.Cache(*(p.numpy() for p in pools))
    dev = _cuda(*pools)
    table = torch.tensor([[2, -1], [9, 4]], dtype=torch.int32)        # -1 and 9 are no pages
    k, v = _rand(g, 300, 2, d), _rand(g, 300, 2, d)
    cu, cached = _cu([200, 100]), torch.tensor([30, -4], dtype=torch.int32)
    attention.kv_append_i8(*_cuda(k, v), *dev, *_cuda(table, cu, cached))
    ref.append(_np(k), _np(v), table.numpy(), cu.numpy(), cached.numpy())
    _same_cache(dev, ref)


def test_append_strided_rows():
    g, d = _gen(5), 128
    pools = _pools(g, 8, 2, d)
    ref = oatt.Cache(*(p.numpy() for p in pools))
    dev = _cuda(*pools)
    fused = _rand(g, 100, 6 * d).cuda()
    k, v = fused[:, 2 * d:4 * d].view(100, 2, d), fused[:, 4 * d:].view(100, 2, d)
    table, cu, cached = _table(g, 2, 2, 8), _cu([37, 63]), torch.tensor([20, 0], dtype=torch.int32)
    attention.kv_append_i8(k, v, *dev, *_cuda(table, cu, cached))
    ref.append(_np(k), _np(v), table.numpy(), cu.numpy(), cached.numpy())
    _same_cache(dev, ref)


def _cache_case(new, lens, hq, hkv, d, dtype, seed=0, tail=0, amp=1.0, table=None, pages=None, scale=None):
    g = _gen(seed)
    width = max(1, -(-max(lens) // PAGE))
    pages = pages or len(new) * width + 2
    pools = _pools(g, pages, hkv, d)
    table = _table(g, len(new), width, pages) if table is None else table
    q = _rand(g, sum(new) + tail, hq, d, dtype=dtype, amp=amp)
    cu, ln = _cu(new), torch.tensor(lens, dtype=torch.int32)
    sc = d ** -0.5 if scale is None else scale
    print(f"cache new={new} lens={lens} heads {hq}/{hkv} d={d} {dtype}", flush=True)
    dev = _cuda(*pools)
    dt = _cuda(table, cu, ln)
    out, lse = attention.cache_attention_i8(q.cuda(), *dev, *dt, scale=scale)
    torch.cuda.synchronize()
    ref = oatt.Cache(*(p.numpy() for p in pools))
    r = ref.attention(_np(q), table.numpy(), cu.numpy(), ln.numpy(), sc)
    kmax = float(pools[2].max()) * 127
    delta = _score_error(_np(q), np.full((1, d), kmax), sc)
    _check(out, lse, r, dtype, HF, delta, float(pools[3].max()) * 127, max(lens + [1]))
    if tail:
        assert (out[sum(new):] == 0).all() and torch.isneginf(lse[:, sum(new):]).all()
    return q, dev, dt, ref, table, cu, ln, out, lse, sc, delta


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new,lens,hq,hkv", [
    ([1], [1], 4, 1), ([1, 1, 1], [65, 1, 400], 8, 2), ([1], [1000], 7, 1), ([16, 16], [200, 77], 4, 1),
    ([4, 1, 0, 8], [130, 64, 50, 8], 4, 2), ([70], [300], 5, 1), ([1] * 70, list(range(1, 71)), 2, 1),
])
def test_cache_attention(new, lens, hq, hkv, d, dtype):
    _cache_case(new, lens, hq, hkv, d, dtype, seed=d + len(new))


def test_cache_attention_rows_that_see_nothing():
    """Empty caches, more new tokens than the cache holds, and rows outside of the sequences."""
    _cache_case([1, 2, 9], [0, 0, 5], 4, 2, 128, BF, tail=5, seed=1)
    _cache_case([3], [0], 2, 1, 64, HF, seed=2)


def test_cache_attention_large_and_small_queries():
    """Rows of q far from 1: their largest value is brought to the same power of two."""
    for amp in (1e-6, 300.0):
        _cache_case([2], [150], 4, 2, 64, BF, amp=amp, seed=3, scale=0.125 / amp)


def test_cache_attention_split_over_many_workgroups():
    """One sequence and head over thousands of tokens, so that its pages are cut into many shares."""
    _cache_case([1], [20000], 4, 1, 64, BF, seed=4)
    _cache_case([2, 1], [9001, 3], 2, 1, 128, HF, seed=5)


def test_cache_attention_more_parts_than_lanes():
    """One key/value head and row tile whose pages make a share for each of hundreds of workgroups."""
    _cache_case([1], [131072], 2, 1, 64, BF, seed=8)
    _cache_case([17], [60000], 2, 1, 128, HF, seed=9)


def test_cache_attention_pages_that_do_not_exist():
    table = torch.tensor([[1, -1, 3], [50, 2, 0]], dtype=torch.int32)
    _cache_case([2, 1], [190, 100], 4, 2, 128, BF, seed=6, table=table, pages=5)


def test_cache_attention_shared_pages():
    """Two sequences with the same first pages."""
    table = torch.tensor([[4, 1, 3], [4, 1, 0]], dtype=torch.int32)
    _cache_case([1, 1], [190, 150], 4, 2, 128, BF, seed=7, table=table, pages=6)


@pytest.mark.parametrize("d,dtype", [(64, HF), (128, BF)])
@pytest.mark.parametrize("new,lens,span", [([1, 1], [65, 300], 300), ([16], [200], 150), ([3, 0, 40], [9, 50, 129], 200), ([4], [2], 64)])
def test_cache_weights(new, lens, span, d, dtype):
    q, dev, dt, ref, table, cu, ln, _, lse, sc, delta = _cache_case(new, lens, 4, 2, d, dtype, seed=9)
    start = torch.rand(len(new), 2, span, generator=_gen(1))
    w = start.cuda()
    attention.cache_weights_i8(q.cuda(), dev[0], dev[2], *dt, lse, w)
    want = ref.weights(_np(q), table.numpy(), cu.numpy(), ln.numpy(), _np(lse), sc, span)
    got = _np(w).astype(np.float64)
    terms = 2 * max(new)
    # a weight's relative error: the score's, that of lse in base 2 and the exponential's; then the sums'
    tol = (2 * delta + 2.0 ** -20 * (1 + np.abs(_np(lse)[np.isfinite(_np(lse))]).max(initial=0.0)) + terms * 2.0 ** -24) * want
    tol = tol + 2.0 ** -23 * (start.numpy() + want)
    assert (np.abs(got - (start.numpy() + want)) <= tol).all()
    none = torch.arange(span)[None] >= ln[:, None]
    assert torch.equal(w.cpu()[none[:, None].expand_as(start)], start[none[:, None].expand_as(start)])
    again = start.cuda()
    attention.cache_weights_i8(q.cuda(), dev[0], dev[2], *dt, lse, again)
    assert torch.equal(again, w)


def _evict_case(lens, keep, recent, heads, d, weights, seed=0, span=None, table=None, pages=None):
    g = _gen(seed)
    b, width = len(lens), max(1, -(-max(lens) // PAGE))
    new_width = -(-min(keep, width * PAGE) // PAGE)
    pages = pages or b * (width + new_width) + 1
    pools = _pools(g, pages, heads, d)
    both = _table(g, b, width + new_width, pages) if table is None else table
    old, new = both[:, :width].contiguous(), both[:, width:].contiguous()
    ln = torch.tensor(lens, dtype=torch.int32)
    dev = _cuda(*pools)
    print(f"evict lens={lens} keep={keep} recent={recent} heads={heads} d={d}", flush=True)
    w, left, kept = attention.cache_evict_i8(*dev, *_cuda(weights, old, ln, new), keep, recent)
    torch.cuda.synchronize()
    ref = oatt.Cache(*(p.numpy() for p in pools))
    rw, rl, rk = ref.evict(weights.numpy(), old.numpy(), ln.numpy(), new.numpy(), keep, recent)
    assert np.array_equal(left.cpu().numpy(), rl)
    assert np.array_equal(kept.cpu().numpy(), rk)
    assert np.array_equal(w.cpu().numpy(), rw, equal_nan=True)
    _same_cache(dev, ref)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens,keep,recent", [
    ([200, 64, 1, 0, 90], 65, 10), ([300], 1, 0), ([300], 1, 1), ([130, 131], 130, 130), ([2500], 1111, 64), ([70], 500, 3),
])
def test_evict(lens, keep, recent, d):
    g = _gen(keep)
    w = torch.randn(len(lens), 2, max(lens), generator=g).exp()
    _evict_case(lens, keep, recent, 2, d, w, seed=d + keep)


@pytest.mark.parametrize("n", [4096, 4097, 8192, 8200, 16384, 40001])
def test_evict_long_rows(n):
    """Rows of one and of several blocks of weights, with ties across their ends."""
    w = torch.randint(0, 50, (1, 1, n), generator=_gen(n)).float()
    _evict_case([n], n // 3, 100, 1, 64, w, seed=n)
    _evict_case([n - 1], n - 2, 0, 1, 64, w[:, :, :n - 1].contiguous(), seed=n)


def test_evict_ties_and_strange_weights():
    """Equal weights go to the earlier token; signed zeros are equal; NaN is lowest, infinities are the ends."""
    g = _gen(3)
    _evict_case([1500, 1100], 700, 50, 2, 64, torch.zeros(2, 2, 1500), seed=1)
    w = torch.randint(0, 3, (2, 2, 1500), generator=g).float()
    _evict_case([1500, 1100], 700, 50, 2, 64, w, seed=2)
    w = torch.randn(2, 2, 1500, generator=g)
    w[:, :, ::7], w[:, :, 3::11], w[:, :, 5::13] = float("nan"), float("inf"), -float("inf")
    w[:, :, 2::5] = 0.0
    w[:, 1, 2::10] = -0.0
    for keep in (100, 700, 1400):
        _evict_case([1500, 1300], keep, 50, 2, 64, w, seed=keep)


@pytest.mark.parametrize("d", [64, 128])
def test_evict_pages_whose_scale_is_not_finite_or_zero_or_large(d):
    """What such a page stands for: NaN is held as 0, infinities as the largest code, and the scale is that of the rest."""
    g = _gen(d)
    pools = _pools(g, 12, 2, d)
    top = float(np.finfo(np.float32).max)
    for i, bad in enumerate((float("nan"), float("inf"), 0.0, top / 127, 1e-42, -0.25)):
        pools[2][i, i % 2] = pools[3][i, (i + 1) % 2] = bad
    table, new = torch.arange(8, dtype=torch.int32)[None], torch.tensor([[8, 9, 10, 11]], dtype=torch.int32)
    ln, w = torch.tensor([500], dtype=torch.int32), torch.rand(1, 2, 500, generator=g)
    dev = _cuda(*pools)
    got = attention.cache_evict_i8(*dev, *_cuda(w, table, ln, new), 230, 20)
    ref = oatt.Cache(*(p.numpy() for p in pools))
    with np.errstate(all="ignore"):
        want = ref.evict(w.numpy(), table.numpy(), ln.numpy(), new.numpy(), 230, 20)
    assert all(np.array_equal(_np(a), b) for a, b in zip(got, want))
    _same_cache([p[8:] for p in dev], oatt.Cache(*(p[8:] for p in (ref.k, ref.v, ref.ks, ref.vs))))


def test_evict_span_shorter_than_the_cache_and_missing_pages():
    g = _gen(6)
    _evict_case([300, 100], 120, 20, 2, 128, torch.rand(2, 2, 150, generator=g), seed=4)
    table = torch.tensor([[0, -1, 2, 7, 8], [3, 99, 4, -5, 9]], dtype=torch.int32)
    _evict_case([190, 180], 100, 20, 2, 128, torch.rand(2, 2, 190, generator=g), seed=5, table=table, pages=10)
