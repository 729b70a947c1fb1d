"""Masks, rows that are not finite, pages outside the pool and lengths past the
table in every attention kernel, the ones for many rows among them; all rows of
the first and the last head against a 64-bit form."""
import numpy as np
import pytest

import kv4_ref as R
from test_gpu_kv4 import F16, F32, NP, Cache, bound, dev, fill  # noqa: F401 (dev is a fixture)

pytestmark = pytest.mark.gpu

# (head dim, q heads, KV heads, rows of the longest sequence).  One to 32 rows a
# KV head: the decode kernel; more: tiles of 64, split; from a tile for every CU
# on (n rows * heads / 64 >= 256) whole tiles of 64, of 128 (head dims 128 and,
# in f16, 256) or of 256 (head dim 64, two a CU).
FEW = [(hd, 4, 1, m) for hd in (64, 128, 256) for m in (1, 7, 40)]
MANY = [(64, 32, 4, 600), (128, 32, 4, 600), (256, 16, 2, 1100), (64, 128, 4, 1100), (128, 32, 4, 1100)]


def visible(pos, n, window, sink):
    j = np.arange(n)
    see = j[None, :] <= pos[:, None]
    if window > 0:
        see &= (j[None, :] > pos[:, None] - window) | (j[None, :] < sink)
    return see


def rows_of(q, k, v, see, scale):
    """(out, largest Σ|q k| scale) of rows q [m][hd] over k, v [n][hd]; see [m][n]."""
    q, big = q.astype(np.float64), 0.0
    out = np.zeros(q.shape)
    for a in range(0, len(q), 256):
        b = slice(a, a + 256)
        s = np.where(see[b], q[b] @ k.T * scale, -np.inf)
        p = np.exp(s - np.maximum(s.max(1, keepdims=True), -1e300))
        out[b] = p @ v / np.maximum(p.sum(1, keepdims=True), 1e-300)
        big = max(big, float((np.where(see[b], np.abs(q[b]) @ np.abs(k).T, 0)).max(initial=0) * scale))
    return out, big


def batch(m):
    """Lengths and row counts: the long one, one whose rows begin before its first token, an idle one, a short one."""
    return [m + 333, 29, 200, 90], [m, min(m, 31), 0, min(m, 17)]


def check(c, held, lens, qlens, q, out, code, window, sink, nan=lambda s, pos, see, g: np.zeros(len(pos), bool)):
    """Rows that `nan` names are NaN, all others right."""
    nh, cu = q.shape[1], np.concatenate([[0], np.cumsum(qlens)])
    for s, (n, m) in enumerate(zip(lens, qlens)):
        pos = np.arange(n - m, n)
        see = visible(pos, n, window, sink)
        for h in (0, nh - 1):
            g = h // (nh // c.nkv)
            off = nan(s, pos, see, g)
            got = out[cu[s]:cu[s + 1], h].astype(np.float64)
            assert np.isnan(got[off]).all() and np.isfinite(got[~off]).all(), (s, h)
            k, v = held[s][0][:, g], held[s][1][:, g]
            want, big = rows_of(q[cu[s]:cu[s + 1], h], k, v, see, c.hd ** -0.5)
            lim = bound(code, c.hd, n, big, float(np.abs(v).max()))
            assert not (~off).any() or np.abs(got - want)[~off].max() <= lim, (s, h, np.abs(got - want)[~off].max(), lim)
    assert (out[cu[-1]:] == -777.0).all()


def queries(rng, rows, nh, hd, code):
    return (1.5 * rng.standard_normal((rows, nh, hd))).astype(NP[code])


@pytest.mark.parametrize("hd,nh,nkv,m", MANY)
@pytest.mark.parametrize("code", [F32, F16])
@pytest.mark.parametrize("window,sink", [(0, 0), (1, 0), (33, 0), (100, 5), (1, 1), (64, 300), (1000, 200)])
def test_masks_of_many_rows(dev, hd, nh, nkv, m, code, window, sink):  # noqa: F811
    rng = np.random.default_rng(hd + m + window)
    lens, qlens = batch(m)
    c = Cache(dev, lens, nkv, hd, 16)
    held = fill(c, lens, rng, code)
    q = queries(rng, sum(qlens) + 3, nh, hd, code)
    out = c.attn(q, np.concatenate([[0], np.cumsum(qlens)]), lens, code=code, window=window, sink=sink)
    check(c, held, lens, qlens, q, out, code, window, sink)


@pytest.mark.parametrize("hd,nh,nkv,m", FEW + MANY)
@pytest.mark.parametrize("code", [F32, F16])
@pytest.mark.parametrize("window,sink", [(0, 0), (60, 3)])
def test_rows_that_are_not_finite(dev, hd, nh, nkv, m, code, window, sink):  # noqa: F811
    """A NaN in K and an infinity in V: the rows that see their tokens are NaN, all others right."""
    rng = np.random.default_rng(hd + m + window)
    lens, qlens = batch(m)
    c = Cache(dev, lens, nkv, hd, 32)
    held = fill(c, lens, rng, code)
    bad = {(0, 0): (lens[0] - m // 2 - 1, True), (0, nkv - 1): (lens[0] - m // 3 - 2, False), (3, nkv - 1): (80, True)}
    for (s, g), (at, in_k) in bad.items():
        k, v = (x[at:at + 1].astype(NP[code]).astype(np.float32) for x in held[s])
        (k if in_k else v)[0, g, 11] = np.nan if in_k else np.inf
        c.append(None, k, v, c.slots(s, at, at + 1), code=code)
    gone = {}
    for (s, g), (at, _) in bad.items():
        gone.setdefault((s, g), []).append(at)
    for s in {s for s, _ in bad}:
        gk, gv = c.read(c.slots(s, 0, lens[s]))
        held[s] = np.nan_to_num(gk.astype(np.float64)), np.nan_to_num(gv.astype(np.float64))
        for g in range(nkv):
            off = np.zeros(lens[s], bool)
            off[gone.get((s, g), [])] = True
            assert np.array_equal(np.isnan(gk[:, g]).any(1), off) and np.array_equal(np.isnan(gv[:, g]).all(1), off)
    q = queries(rng, sum(qlens), nh, hd, code)
    out = c.attn(q, np.concatenate([[0], np.cumsum(qlens)]), lens, code=code, window=window, sink=sink)
    check(c, held, lens, qlens, q, out, code, window, sink,
          lambda s, pos, see, g: see[:, gone[s, g]].any(1) if (s, g) in gone else np.zeros(len(pos), bool))


@pytest.mark.parametrize("hd,nh,nkv,m", FEW + MANY)
@pytest.mark.parametrize("code", [F32, F16])
@pytest.mark.parametrize("window,sink", [(0, 0), (60, 0), (50, 20)])
def test_pages_outside_the_pool(dev, hd, nh, nkv, m, code, window, sink):  # noqa: F811
    """The rows that see a page outside the pool are NaN, all others of its sequence right: pages behind a window may be gone."""
    rng = np.random.default_rng(hd + m + window)
    lens, qlens = batch(m)
    c = Cache(dev, lens, nkv, hd, 16)
    held = fill(c, lens, rng, code)
    gone = {0: {3: -1, (lens[0] - m // 2) // 16 - 5: c.n_pages}, 3: {1: 2 ** 31 - 1}}
    for s, entries in gone.items():
        for b, e in entries.items():
            c.table[s, b] = e
    q = queries(rng, sum(qlens), nh, hd, code)
    out = c.attn(q, np.concatenate([[0], np.cumsum(qlens)]), lens, code=code, window=window, sink=sink)

    def nan(s, pos, see, g):
        off = np.zeros(len(pos), bool)
        for b in gone.get(s, {}):
            off |= see[:, 16 * b:16 * b + 16].any(1)
        return off
    check(c, held, lens, qlens, q, out, code, window, sink, nan)


@pytest.mark.parametrize("hd,nh,nkv,m", FEW + MANY)
@pytest.mark.parametrize("code", [F32, F16])
def test_lengths_past_the_table(dev, hd, nh, nkv, m, code):  # noqa: F811
    """All rows of a sequence whose length passes its table are NaN, the others right."""
    rng = np.random.default_rng(hd + m)
    lens, qlens = batch(m)
    c = Cache(dev, lens, nkv, hd, 16)
    held = fill(c, lens, rng, code)
    said = list(lens)
    said[3] = 16 * c.width + 1
    q = queries(rng, sum(qlens), nh, hd, code)
    out = c.attn(q, np.concatenate([[0], np.cumsum(qlens)]), said, code=code)
    check(c, held, lens, qlens, q, out, code, 0, 0, lambda s, pos, see, g: np.full(len(pos), s == 3))


@pytest.mark.parametrize("hd,nh,nkv,m", MANY)
def test_scores_past_fp32_of_many_rows(dev, hd, nh, nkv, m):  # noqa: F811
    """Heads whose scores pass fp32's range are NaN, the heads beside them in a tile right."""
    rng = np.random.default_rng(hd + m)
    n = m + 90
    c = Cache(dev, [n], nkv, hd, 16)
    k, v = np.ones((n, nkv, hd), np.float32), rng.standard_normal((n, nkv, hd)).astype(np.float32)
    c.append(None, k, v, c.slots(0, 0, n))
    q = rng.standard_normal((m, nh, hd)).astype(np.float32)
    q[:, 1::4], q[:, 2::4] = 3e37, -3e37
    out = c.attn(q, [0, m], [n], scale=8.0)
    assert np.isnan(out[:, 1::4]).all() and np.isnan(out[:, 2::4]).all()
    mean = (np.cumsum(R.quantize(v)[2], 0) / np.arange(1, n + 1)[:, None, None])[n - m:]
    want = np.repeat(mean, nh // nkv, 1)
    tol = (2 * (n + 16) * 2.0 ** -24 + 2.0 ** -21) * np.abs(R.quantize(v)[2]).max()
    for x in (0, 3):
        assert np.abs(out[:, x::4] - want[:, x::4]).max() <= tol
