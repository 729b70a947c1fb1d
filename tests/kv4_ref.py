"""Plain 64-bit forms of the paged 4-bit KV cache's operators (numpy)."""
import numpy as np

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)
LUT = np.concatenate([GRID, -GRID])
SCALE_MAX = 10912.0


def quantize(x):
    """(codes uint8, scales float64, values float64, finite rows) of fp32 rows [..., hd]."""
    x = np.asarray(x, np.float32).astype(np.float64)
    b = x.reshape(x.shape[:-1] + (x.shape[-1] // 32, 32))
    fin = np.isfinite(x).all(-1)
    b = np.where(np.isfinite(b), b, 0.0)
    want = np.abs(b).max(-1) / 6.0
    exp = np.frexp(want)[1] - 1
    step = np.ldexp(1.0, np.maximum(exp - 8, -23))
    s = np.minimum(np.rint(want / step) * step, SCALE_MAX)
    # nearest code, ties to the even one: distances to the even codes first
    # (past the largest one it is the nearest; the distances of 1e38 would all round alike)
    d = np.abs(np.minimum(np.abs(b), 6.0 * s[..., None])[..., None] - GRID * s[..., None, None])
    order = np.array([0, 2, 4, 6, 1, 3, 5, 7])
    code = order[np.argmin(d[..., order], -1)].astype(np.uint8)
    code = np.where(s[..., None] > 0, code, 0) | (b < 0).astype(np.uint8) << 3
    val = (LUT[code] * s[..., None]).reshape(x.shape)
    return code.reshape(x.shape), s, val, fin


def rope(x, pos, axis, table, halves):
    """x [T][heads][hd] rotated, in 64 bits; pos [axes][T], table [rows][pairs][2]."""
    y = np.asarray(x).astype(np.float64).copy()
    half = len(axis)
    for i, ax in enumerate(axis):
        p = pos[ax]
        ok = (p >= 0) & (p < len(table))
        cs = np.where(ok[:, None], table[np.where(ok, p, 0), i].astype(np.float64), np.nan)
        c, s = cs[:, :1], cs[:, 1:]
        d0, d1 = (i, i + half) if halves else (2 * i, 2 * i + 1)
        a, b = y[..., d0].copy(), y[..., d1].copy()
        y[..., d0], y[..., d1] = a * c - b * s, a * s + b * c
    return y


def plan(kv_len, q_len, table, free, n_free, n_pages, ps, n_tok):
    table = table.copy()
    width = table.shape[1]
    cu, pos, slot, out = [0], np.full(n_tok, -1), np.full(n_tok, -1), []
    taken = used = refused = 0
    n_free = min(max(n_free, 0), n_pages)
    for s, (a, q) in enumerate(zip(np.maximum(kv_len, 0).tolist(), np.maximum(q_len, 0).tolist())):
        fits = a + q <= width * ps
        have = -(-a // ps)
        need = -(-(a + q) // ps) - have if fits else 0
        ok = fits and cu[-1] + q <= n_tok and (need == 0 or taken + need <= n_free)
        if ok:
            for k in range(need):
                p = free[n_free - 1 - taken - k]
                table[s, have + k] = p if 0 <= p < n_pages else -1
            for i in range(q):
                p = table[s, (a + i) // ps]
                pos[cu[-1] + i] = a + i
                slot[cu[-1] + i] = p * ps + (a + i) % ps if 0 <= p < n_pages else -1
            used += need
        else:
            refused += 1
        taken += need
        cu.append(cu[-1] + q)
        out.append(a + q if ok else int(kv_len[s]))
    beyond = max(cu[-1] - n_tok, 0)
    return np.minimum(cu, n_tok), pos, slot, table, np.array(out), n_free - used, (refused, beyond)


def release(kv_len, keep, table, free, n_free, ps):
    table, free, back, out = table.copy(), free.copy(), [], []
    for s, (a, k) in enumerate(zip(kv_len.tolist(), keep.tolist())):
        k = min(max(k, 0), a)
        for b in range(-(-k // ps), -(-a // ps)):
            back.append(table[s, b])
            table[s, b] = -1
        out.append(k)
    free[n_free:n_free + len(back)] = back[::-1]
    return table, free, np.array(out), n_free + len(back)


def attention(q, k, v, pos, scale, window, sink):
    """q [rows][nh][hd] at positions pos over k, v [len][nkv][hd] (64 bits); (out, Σ|q k| scale at most)."""
    rows, nh, hd = q.shape
    g = nh // k.shape[1] if len(k) else 1
    out, big = np.zeros(q.shape), 0.0
    j = np.arange(len(k))
    for r in range(rows):
        see = j <= pos[r]
        if window > 0:
            see &= (j > pos[r] - window) | (j < sink)
        if not see.any():
            continue
        for h in range(nh):
            kk, vv = k[see, h // g], v[see, h // g]
            s = kk @ q[r, h].astype(np.float64) * scale
            big = max(big, float((np.abs(kk) @ np.abs(q[r, h].astype(np.float64))).max() * scale))
            p = np.exp(s - s.max())
            out[r, h] = p @ vv / p.sum()
    return out, big
