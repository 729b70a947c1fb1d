"""How exact the 4-bit cache's attention is, at inputs whose errors can be
counted closely: scores of one product, few visible keys, closed forms in 64
bits."""
import numpy as np
import pytest

import kv4_ref as R
from test_gpu_kv4 import F16, F32, NP, Cache, bound, dev  # noqa: F401 (dev is a fixture)

pytestmark = pytest.mark.gpu

# (head dim, q heads, KV heads, rows): rows of every kernel -- decode, two row
# tiles at head dim 128, tiles of 64, whole tiles of 64, whole tiles of 128 / 256
KERNELS = [(hd, 4, 1, m) for hd in (64, 128, 256) for m in (1, 7, 40)]
KERNELS += [(64, 32, 4, 600), (128, 32, 4, 600), (256, 32, 4, 600), (64, 32, 4, 2100), (64, 128, 4, 1100), (128, 32, 4, 1100), (256, 16, 2, 1100)]


@pytest.mark.parametrize("hd,nh,nkv,m", KERNELS)
@pytest.mark.parametrize("code", [F32, F16])
def test_probabilities_keep_22_bits(dev, hd, nh, nkv, m, code):  # noqa: F811
    """Rows that see two keys with values of about +1 and -1: the output is tanh of half the scores' difference.

    A score is one exact product of q and k (11 bits each; fp32 q: two terms,
    2^-22 of at most 4 * 0.125).  Of p: the exponent's rounding 2^-21 * ln 2
    (below 16), the exponential 2^-23, two terms 2^-22, fp32 q 2^-22: 2^-19.9
    together; the output is off by at most as much, the sums' and the
    division's roundings (6 of 2^-24) and its own rounding to its type."""
    rng = np.random.default_rng(hd + m)
    n = m + 1
    c = Cache(dev, [n], nkv, hd, 16)
    k, v = np.zeros((n, nkv, hd), np.float32), np.ones((n, nkv, hd), np.float32)
    k[:, :, 5] = rng.uniform(0.5, 2, (n, nkv)) * rng.choice([-1, 1], (n, nkv))
    v[1::2] = -1
    c.append(None, k, v, c.slots(0, 0, n))
    kv, one = R.quantize(k)[2][:, :, 5], R.quantize(v)[2][0, 0, 0]  # (1 is held as 6 times 1 / 6 to 9 bits)
    q = rng.standard_normal((m, nh, hd)).astype(NP[code])
    q[:, :, 5] = rng.uniform(0.5, 2, (m, nh)).astype(NP[code])
    out = c.attn(q, [0, m], [n], code=code, scale=0.125, window=2).astype(np.float64)
    p = np.arange(1, n)
    head = np.arange(nh) // (nh // nkv)
    s = q[:, :, 5].astype(np.float64) * 0.125
    d = s * (kv[p][:, head] - kv[p - 1][:, head]) / 2
    want = (one * np.tanh(d) * np.where(p % 2, -1, 1)[:, None])[:, :, None]
    tol = 2.0 ** -19.9 + 6 * 2.0 ** -24 + np.abs(want) * (2.0 ** -24 if code == F32 else 2.0 ** -11) + (0 if code == F32 else 2.0 ** -25)
    assert (np.abs(out - want) <= tol).all(), np.abs(out - want).max()


@pytest.mark.parametrize("hd,nh,nkv,m", KERNELS)
@pytest.mark.parametrize("mag", [1e5, 1e8, 3e8, 1e9, 1e20, 1e35])
def test_large_scores_pick_the_largest(dev, hd, nh, nkv, m, mag):  # noqa: F811
    """q of any size: the key that wins by more than the scores' rounding is the output, to 2^-20; ties stay among the values.

    A score is off by at most ds = big (2^-22 + (1.1 hd + 6) 2^-24) (two-term
    q, the fp32 sums of its products, its scaling); where the second largest is
    2 ds + 20 behind, all others weigh less than n e^-20 = 2^-19 of the first."""
    rng = np.random.default_rng(hd + m)
    n = m + 330
    c = Cache(dev, [n], nkv, hd, 16)
    k, v = (rng.standard_normal((n, nkv, hd)).astype(np.float32) for _ in range(2))
    c.append(None, k, v, c.slots(0, 0, n))
    kk, vv = R.quantize(k)[2], R.quantize(v)[2]
    q = (rng.standard_normal((m, nh, hd)) * mag).astype(np.float32)
    out = c.attn(q, [0, m], [n]).astype(np.float64)
    clear = 0
    for r in np.unique(np.concatenate([[0, m - 1], rng.integers(0, m, 12)])):
        for h in (0, nh - 1):
            g, p = h // (nh // nkv), n - m + r
            x = q[r, h].astype(np.float64) * hd ** -0.5
            s, big = kk[:p + 1, g] @ x, float((np.abs(kk[:p + 1, g]) @ np.abs(x)).max())
            ds = big * (2.0 ** -22 + (1.1 * hd + 6) * 2.0 ** -24)
            top, seen = int(s.argmax()), vv[:p + 1, g]
            assert (out[r, h] >= seen.min(0) - 1e-5).all() and (out[r, h] <= seen.max(0) + 1e-5).all(), (r, h)
            if s[top] - np.delete(s, top).max() > 2 * ds + 20:
                clear += 1
                assert np.abs(out[r, h] - seen[top]).max() <= (2.0 ** -19 + 2.0 ** -20) * np.abs(seen).max(), (r, h, s[top])
    assert clear


@pytest.mark.parametrize("hd,nh,nkv,m", KERNELS)
@pytest.mark.parametrize("mag", [1, 1e8, 1e12, 1e30])
def test_equal_scores_weigh_the_same(dev, hd, nh, nkv, m, mag):  # noqa: F811
    """All keys alike: the output is the mean of the values seen, however large the scores are.

    Equal keys have equal scores bit by bit, so p is 2^6 throughout; the sums
    take a rounding of 2^-24 a key, twice, the division and two-term p 2^-21."""
    rng = np.random.default_rng(hd + m)
    n = m + 330
    c = Cache(dev, [n], nkv, hd, 16)
    k = np.tile(rng.standard_normal((1, nkv, hd)).astype(np.float32), (n, 1, 1))
    v = rng.standard_normal((n, nkv, hd)).astype(np.float32)
    c.append(None, k, v, c.slots(0, 0, n))
    vv = R.quantize(v)[2]
    q = (rng.standard_normal((m, nh, hd)) * mag).astype(np.float32)
    out = c.attn(q, [0, m], [n]).astype(np.float64)
    mean = (np.cumsum(vv, 0) / np.arange(1, n + 1)[:, None, None])[n - m:]
    want = np.repeat(mean, nh // nkv, 1)
    assert np.abs(out - want).max() <= (2 * (n + 16) * 2.0 ** -24 + 2.0 ** -21) * np.abs(vv).max()


@pytest.mark.parametrize("hd,nh,nkv,m", [k for k in KERNELS if k[3] in (1, 7, 40, 1100)])
def test_large_scores_of_f16_rows(dev, hd, nh, nkv, m):  # noqa: F811
    """f16 rows reach scores of 1e10 too: one key is 1.25 times the others and wins."""
    rng = np.random.default_rng(hd + m)
    n = m + 330
    c = Cache(dev, [n], nkv, hd, 16)
    k, v = np.full((n, nkv, hd), 4.8e4, np.float32), rng.standard_normal((n, nkv, hd)).astype(np.float16).astype(np.float32)
    win = 77
    k[win] = 6e4
    c.append(None, k, v, c.slots(0, 0, n), code=F16)
    q = np.full((m, nh, hd), 6e4, np.float16)
    q[:, 1::2] = 3e4
    out = c.attn(q, [0, m], [n], code=F16).astype(np.float64)
    want = np.repeat(R.quantize(v)[2][win], nh // nkv, 0)
    assert (np.abs(out - want) <= np.abs(want) * 2.0 ** -11 + 2.0 ** -20).all()


@pytest.mark.parametrize("hd,nh,nkv,m", KERNELS)
@pytest.mark.parametrize("far", [2.0 ** 6, 2.0 ** 10, 2.0 ** 14, 2.0 ** 17])
def test_small_q_values_beside_large_ones(dev, hd, nh, nkv, m, far):  # noqa: F811
    """As test_probabilities_keep_22_bits, with a q channel `far` times the largest other that meets K values of 0."""
    rng = np.random.default_rng(hd + m)
    n = m + 1
    c = Cache(dev, [n], nkv, hd, 16)
    k, v = np.zeros((n, nkv, hd), np.float32), np.ones((n, nkv, hd), np.float32)
    k[:, :, 5] = rng.uniform(0.5, 2, (n, nkv)) * rng.choice([-1, 1], (n, nkv))
    v[1::2] = -1
    c.append(None, k, v, c.slots(0, 0, n))
    kv, one = R.quantize(k)[2][:, :, 5], R.quantize(v)[2][0, 0, 0]
    q = rng.uniform(0.5, 2, (m, nh, hd)).astype(np.float32)
    q[:, :, 40] = rng.choice([-1, 1], (m, nh)) * far
    out = c.attn(q, [0, m], [n], scale=0.125, window=2).astype(np.float64)
    p = np.arange(1, n)
    head = np.arange(nh) // (nh // nkv)
    d = q[:, :, 5].astype(np.float64) * 0.125 * (kv[p][:, head] - kv[p - 1][:, head]) / 2
    want = (one * np.tanh(d) * np.where(p % 2, -1, 1)[:, None])[:, :, None]
    assert (np.abs(out - want) <= 2.0 ** -19.9 + 6 * 2.0 ** -24 + np.abs(want) * 2.0 ** -24).all(), np.abs(out - want).max()


@pytest.mark.parametrize("hd,nh,nkv,m", [k for k in KERNELS if k[3] in (1, 7, 40, 1100)])
def test_channels_of_opposite_size(dev, hd, nh, nkv, m):  # noqa: F811
    """Channels where q is 2^14 times smaller and K as much larger: both halves make the score."""
    rng = np.random.default_rng(hd + m)
    n = m + 100
    c = Cache(dev, [n], nkv, hd, 16)
    size = np.where(np.arange(hd) < hd // 2, 2.0 ** 7, 2.0 ** -7)
    k, v = ((rng.standard_normal((n, nkv, hd)) * x).astype(np.float32) for x in (size, 1))
    c.append(None, k, v, c.slots(0, 0, n))
    kk, vv = R.quantize(k)[2], R.quantize(v)[2]
    q = (rng.standard_normal((m, nh, hd)) / size).astype(np.float32)
    out = c.attn(q, [0, m], [n]).astype(np.float64)
    for r in np.unique(np.concatenate([[0, m - 1], rng.integers(0, m, 12)])):
        want, big = R.attention(q[r:r + 1], kk, vv, np.array([n - m + r]), hd ** -0.5, 0, 0)
        assert np.abs(out[r] - want[0]).max() <= bound(F32, hd, n, big, np.abs(vv).max()), r
