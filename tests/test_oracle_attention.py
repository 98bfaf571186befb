"""The attention oracle against torch's own attention in float64, and the cache's definitions on small examples."""

import numpy as np
import torch

from oracle import attention as oatt


def _rand(*shape, seed=0):
    return np.random.default_rng(seed).standard_normal(shape)


def test_attention_against_torch():
    q, k, v = _rand(7, 4, 16, seed=1), _rand(9, 2, 16, seed=2), _rand(9, 2, 16, seed=3)
    for causal in (True, False):
        out, lse, mag = oatt.packed_attention(q, k, v, [0, 7], [0, 9], 0.3, causal)
        t = [torch.from_numpy(x).transpose(0, 1) for x in (q, k.repeat(2, 1), v.repeat(2, 1))]
        mask = torch.ones(7, 9, dtype=torch.bool).tril(2) if causal else None
        want = torch.nn.functional.scaled_dot_product_attention(*t, attn_mask=mask, scale=0.3)
        assert np.allclose(out, want.transpose(0, 1).numpy(), rtol=1e-12, atol=1e-12)
        s = t[0] @ t[1].transpose(1, 2) * 0.3
        s = s if mask is None else s.masked_fill(~mask, -np.inf)
        assert np.allclose(lse, s.logsumexp(-1).numpy(), rtol=1e-12)
        assert (mag >= np.abs(out) - 1e-12).all()


def test_packed_sequences_are_their_own():
    q, k, v = (_rand(10, 2, 8, seed=s) for s in range(3))
    both = oatt.packed_attention(q, k, v, [0, 4, 10], [0, 4, 10], 1.0)
    for a, e in ((0, 4), (4, 10)):
        one = oatt.packed_attention(q[a:e], k[a:e], v[a:e], [0, e - a], [0, e - a], 1.0)
        assert np.array_equal(both[0][a:e], one[0]) and np.array_equal(both[1][:, a:e], one[1])


def test_rows_that_see_nothing():
    q, k = _rand(5, 1, 8), _rand(2, 1, 8)
    out, lse, _ = oatt.packed_attention(q, k, k, [0, 5], [0, 2], 1.0)
    assert (out[:3] == 0).all() and np.isneginf(lse[:, :3]).all() and np.isfinite(lse[:, 3:]).all()


def test_codes():
    x = np.array([1.0, -1.0, 0.5, 1 / 254, 3 / 254, np.nan, np.inf, -np.inf], np.float32)
    s = oatt.page_scale(x)
    assert s == np.float32(1) / np.float32(127)
    assert oatt.encode(x, s).tolist()[:3] == [127, -127, 64] and oatt.encode(x, s).tolist()[5:] == [0, 127, -127]
    assert oatt.page_scale(np.full(4, 1e-38, np.float32)) == 0
    assert (oatt.encode(np.array([1e-38, np.inf], np.float32), np.float32(0)) == 0).all()


def _cache(pages=4, heads=1, d=4):
    return oatt.Cache(np.zeros((pages, heads, 64, d), np.int8), np.zeros((pages, heads, d, 64), np.int8),
                      np.zeros((pages, heads), np.float32), np.zeros((pages, heads), np.float32))


def test_append_holds_what_was_put():
    c = _cache()
    x = _rand(100, 1, 4, seed=5).astype(np.float32)
    table = np.array([[2, 0]])
    for a, e in ((0, 1), (1, 64), (64, 70), (70, 100)):
        c.append(x[a:e], -x[a:e], table, [0, e - a], [a])
    for side, sign in ((0, 1), (1, -1)):
        got, there = c.values(side, table[0], 100, 0, 4)
        assert there.all()
        # each growth of a scale adds half a step of it, and the scales grow: two steps of the last bound them all
        step = np.repeat((c.ks, c.vs)[side][table[0], 0], 64)[:100, None]
        assert (np.abs(got - sign * x[:, 0]) <= 2 * step).all()
    assert (c.ks[[1, 3]] == 0).all() and np.array_equal(c.k[2, 0], -c.v[2, 0].T)


def test_attention_over_the_cache_is_attention_of_its_values():
    c = _cache(heads=2)
    x = _rand(90, 2, 4, seed=6).astype(np.float32)
    table = np.array([[3, 1]])
    c.append(x, x[::-1], table, [0, 90], [0])
    q = _rand(3, 4, 4, seed=7)
    kv = [np.stack([c.values(s, table[0], 90, h, 4)[0] for h in range(2)], 1) for s in range(2)]
    want = oatt.packed_attention(q, *kv, [0, 3], [0, 90], 0.5)
    got = c.attention(q, table, [0, 3], [90], 0.5)
    assert np.allclose(got[0], want[0], rtol=1e-12) and np.allclose(got[1], want[1], rtol=1e-12)
    w = c.weights(q, table, [0, 3], [90], got[1], 0.5, 128)
    assert np.allclose(w.sum(-1), 6.0) and (w[:, :, 90:] == 0).all()    # 3 tokens, 2 query heads: each row's sum is 1


def test_evict_keeps_recent_and_largest():
    c = _cache(pages=4)
    x = np.arange(1, 71, dtype=np.float32)[:, None, None].repeat(4, 2) / 64
    c.append(x, x, np.array([[0, 1]]), [0, 70], [0])
    w = np.zeros((1, 1, 80), np.float32)
    w[0, 0, [5, 17, 69]] = 2.0, 3.0, 9.0
    w[0, 0, 8] = np.nan
    out, left, kept = c.evict(w, np.array([[0, 1]]), np.array([70]), np.array([[2, 3]]), 6, 3)
    assert left.tolist() == [6] and kept[0, 0].tolist() == [0, 5, 17, 67, 68, 69]
    assert out[0, 0, :7].tolist() == [0, 2, 3, 0, 0, 9, 0]
    got, _ = c.values(0, np.array([2, 3]), 6, 0, 4)
    assert (np.abs(got - x[kept[0, 0], 0]) <= c.ks[2, 0]).all()
