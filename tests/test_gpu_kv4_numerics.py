"""How exact the 4-bit cache's attention is, at inputs whose errors can be
counted closely: scores of one product, few visible keys, closed forms in 64
bits."""
import numpy as np
import pytest

import kv4_ref as R
from test_gpu_kv4 import F16, F32, NP, Cache, dev  # noqa: F401 (dev is a fixture)

pytestmark = pytest.mark.gpu

# (head dim, q heads, KV heads, rows): rows of every kernel -- decode, two row
# tiles at head dim 128, tiles of 64, whole tiles of 64, whole tiles of 128 / 256
KERNELS = [(hd, 4, 1, m) for hd in (64, 128, 256) for m in (1, 7, 40)]
KERNELS += [(64, 32, 4, 600), (128, 32, 4, 600), (256, 32, 4, 600), (64, 32, 4, 2100), (128, 32, 4, 1100), (256, 16, 2, 1100)]


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
