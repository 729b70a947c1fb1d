"""The paged 4-bit KV cache on the GPU through the C ABI, against plain 64-bit
forms (kv4_ref.py).

Page plans and 4-bit rows are compared exactly: every rounding decision of the
quantizer is exact in both.  Attention is held to bounds counted from its
roundings (see `bound`)."""
import ctypes as ct

import numpy as np
import pytest

import kv4_ref as R
from hip_rt import Hip

pytestmark = pytest.mark.gpu

F16, F32 = 7, 9
NP = {F16: np.float16, F32: np.float32}


@pytest.fixture
def dev():
    h = Hip()
    yield h
    h.free()


def _workspace(n):
    """Counters 0, the rest anything."""
    w = np.full(n, 0xFF, np.uint8)
    w[:16384] = 0
    return w


class Cache:
    """A pool of pages, all bytes 0xFF at first (NaN scales), and block tables over shuffled pages."""

    def __init__(self, dev, lens, nkv, hd, ps, seed=0, spare=3, width=None):
        from dracohip import lib
        self.lib, self.L, self.dev = lib, lib.load(), dev
        self.nkv, self.hd, self.ps = nkv, hd, ps
        need = [-(-n // ps) for n in lens]
        self.n_pages = sum(need) + spare
        rng = np.random.default_rng(seed + 77)
        order = rng.permutation(self.n_pages).astype(np.int32)
        self.width = width or max(need + [1]) + 1
        self.table = np.full((len(lens), self.width), -1, np.int32)
        k = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[k:k + n]
            k += n
        self.free = np.full(self.n_pages, -1, np.int32)
        self.free[:self.n_pages - k] = order[k:]
        self.n_free = self.n_pages - k
        self.page_bytes = self.L.draco_kv4_page_bytes(ps, nkv, hd)
        assert self.page_bytes == nkv * ps * hd * 9 // 8
        self.pages = dev.up(np.full(self.n_pages * self.page_bytes, 0xFF, np.uint8))
        self.desc = lib.Kv4(data=self.pages, n_pages=self.n_pages, page_size=ps, n_kv=nkv, head_dim=hd)

    def slots(self, s, a, b):
        p = np.arange(a, b)
        return (self.table[s, p // self.ps] * self.ps + p % self.ps).astype(np.int32)

    def append(self, q, k, v, slot, code=F32, rot=0, pairing=0, pos=None, axis=None, table=None, q_out=None, stream=None, rc=0):
        d, T = self.dev, len(slot)
        nh = 0 if q is None else q.shape[1]
        a = self.lib.Kv4Append(code=code, n_tok=T, n_head=nh, k=d.up(k.astype(NP[code])), v=d.up(v.astype(NP[code])),
                               k_stride=self.nkv * self.hd, v_stride=self.nkv * self.hd, slot=d.up(slot.astype(np.int32)),
                               rot=rot, pairing=pairing)
        if nh:
            a.q, a.q_out, a.q_stride, a.q_out_stride = d.up(q.astype(NP[code])), q_out, nh * self.hd, nh * self.hd
        if rot:
            a.pos, a.pos_stride, a.n_axes = d.up(pos.astype(np.int32)), pos.shape[1], pos.shape[0]
            a.table, a.table_rows = d.up(table.astype(np.float32)), len(table)
            for i, x in enumerate(axis):
                a.axis[i] = x
        got = self.L.draco_kv4_append(ct.byref(self.desc), ct.byref(a), stream)
        assert got == rc, self.lib.last_error()

    def read(self, slot):
        n = len(slot)
        fill = np.full((n, self.nkv, self.hd), -777.0, np.float32)
        k, v = self.dev.up(fill), self.dev.up(fill)
        self.lib.check(self.L.draco_kv4_read(ct.byref(self.desc), self.dev.up(slot.astype(np.int32)), n, k, v, None), "read")
        return self.dev.down(k, fill.shape, np.float32), self.dev.down(v, fill.shape, np.float32)

    def attn_args(self, q, out, cu, lens, max_q=None, max_len=None, window=0, sink=0, code=F32, scale=None, n_tok=None):
        d = self.dev
        nh = q.shape[1]
        a = self.lib.Kv4Attn(code=code, n_seq=len(lens), n_tok=len(q) if n_tok is None else n_tok,
                             max_q=max_q or max(1, max(np.diff(cu), default=1)), max_len=max(lens, default=0) if max_len is None else max_len,
                             n_head=nh, window=window, sink=sink, scale=scale or self.hd ** -0.5, max_blocks=self.width,
                             q=d.up(q.astype(NP[code])), out=out, q_stride=nh * self.hd, out_stride=nh * self.hd,
                             cu_q=d.up(np.asarray(cu, np.int32)), kv_len=d.up(np.asarray(lens, np.int32)),
                             block_table=d.up(self.table))
        need = self.L.draco_kv4_attn_workspace(ct.byref(self.desc), ct.byref(a))
        if need:
            a.work, a.work_bytes = d.up(_workspace(need)), need
        return a

    def attn(self, q, cu, lens, code=F32, stream=None, **kw):
        fill = np.full(q.shape, -777.0, NP[code])
        out = self.dev.up(fill)
        a = self.attn_args(q, out, cu, lens, code=code, **kw)
        self.lib.check(self.L.draco_kv4_attn(ct.byref(self.desc), ct.byref(a), stream), "draco_kv4_attn")
        if a.work:
            assert not self.dev.down(a.work, 4096, np.int32).any()  # counters left at 0
        return self.dev.down(out, q.shape, NP[code])


def bound(code, hd, n, big, vmax):
    """Largest |error| of an attention row over n keys, by its roundings.

    A score: two-term q (2^-22 of each product), hd + hd/16 fp32 sums, the
    exponent's fma and the reference's product (2^-24 each of 1.45 * 2 big):
    |ds| <= big * (2^-22 + 1.1 hd 2^-24 + 6 2^-24); p's relative error is that
    and the exponential's 2^-23, and it enters numerator and denominator.  The
    sums of p and p v: at most n + 8 roundings of 2^-24 each, two-term p 2^-22.
    f16 rows: p rounded to f16 (2^-11 of p) and the output (2^-11)."""
    ds = big * (2.0 ** -22 + (1.1 * hd + 6) * 2.0 ** -24) + 2.0 ** -22
    e = 2 * ds + 2 * (n + 16) * 2.0 ** -24 + 2.0 ** -21
    if code == F16:
        e += 2.0 ** -11 + 2.0 ** -11
    return e * vmax


def fill(c, lens, rng, code=F32, scale=1.0):
    """Sequences' K / V rows into the pages; the values they stand for, per sequence."""
    held = []
    for s, n in enumerate(lens):
        k = rng.standard_normal((n, c.nkv, c.hd)) * np.exp(0.5 * rng.standard_normal((c.nkv, c.hd))) * scale
        v = rng.standard_normal((n, c.nkv, c.hd))
        k, v = k.astype(NP[code]).astype(np.float32), v.astype(NP[code]).astype(np.float32)
        if n:
            c.append(None, k, v, c.slots(s, 0, n), code=code)
        held.append((R.quantize(k)[2], R.quantize(v)[2]))
    return held


def check_attn(c, held, lens, qlens, nh, rng, code=F32, window=0, sink=0, pad=0, **kw):
    cu = np.concatenate([[0], np.cumsum(qlens)])
    q = (1.5 * rng.standard_normal((int(cu[-1]) + pad, nh, c.hd))).astype(NP[code])
    out = c.attn(q, cu, lens, code=code, window=window, sink=sink, **kw)
    for s, (n, m) in enumerate(zip(lens, qlens)):
        k, v = held[s]
        want, big = R.attention(q[cu[s]:cu[s + 1]], k, v, np.arange(n - m, n), c.hd ** -0.5, window, sink)
        got = out[cu[s]:cu[s + 1]].astype(np.float64)
        vmax = float(np.abs(v).max()) if n else 0.0
        err = float(np.abs(got - want).max()) if m else 0.0
        assert np.isfinite(got).all() and err <= bound(code, c.hd, n, big, vmax), (s, n, m, err, bound(code, c.hd, n, big, vmax))
    assert (out[cu[-1]:] == -777.0).all()  # rows behind the last sequence
    return out


# ---- pages ---------------------------------------------------------------------

def _plan_call(dev, kv, q, table, free, n_free, n_pages, ps, n_tok, in_place=False, stream=None):
    from dracohip import lib
    n = len(kv)
    d = dict(block_table=dev.up(table.astype(np.int32)), kv_len=dev.up(kv.astype(np.int32)), q_len=dev.up(q.astype(np.int32)),
             free_list=dev.up(free.astype(np.int32)), n_free=dev.up(np.array([n_free], np.int32)),
             cu_q=dev.up(np.full(n + 1, -9, np.int32)), pos=dev.up(np.full(n_tok, -9, np.int32)),
             slot=dev.up(np.full(n_tok, -9, np.int32)), status=dev.up(np.full(2, -9, np.int32)), work=dev.up(np.zeros(1, np.int32)))
    d["kv_len_out"] = d["kv_len"] if in_place else dev.up(np.full(max(n, 1), -9, np.int32))
    d["n_free_out"] = d["n_free"] if in_place else dev.up(np.full(1, -9, np.int32))
    a = lib.KvPlan(n_seq=n, max_blocks=table.shape[1], n_pages=n_pages, page_size=ps, n_tok=n_tok, **d)
    lib.check(lib.load().draco_kv_plan(ct.byref(a), stream), "draco_kv_plan")
    g = lambda k, m: dev.down(d[k], m, np.int32)  # noqa: E731
    assert g("work", 1)[0] == 0
    return (g("cu_q", n + 1), g("pos", n_tok), g("slot", n_tok), g("block_table", table.shape), g("kv_len_out", n),
            int(g("n_free_out", 1)[0]), tuple(g("status", 2))), d


def _pool(rng, kv, ps, width, n_pages):
    order = rng.permutation(n_pages)
    table = np.full((len(kv), width), -1, np.int32)
    k = 0
    for s, a in enumerate(kv):
        n = -(-int(max(a, 0)) // ps)
        table[s, :n] = order[k:k + n]
        k += n
    free = np.full(n_pages, -1, np.int32)
    free[:n_pages - k] = order[k:]
    return table, free, n_pages - k


PLANS = [  # sequences, page size, cached up to, new tokens up to, rows behind, pages missing
    (1, 16, 1, 2, 0, 0), (1, 16, 0, 17, 3, 0), (7, 32, 200, 2, 0, 0), (9, 16, 64, 40, 5, 2), (130, 64, 500, 2, 0, 0),
    (1023, 16, 90, 5, 0, 0), (1024, 16, 90, 3, 1, 3), (2500, 16, 40, 30, 100, 40), (3, 256, 5000, 4000, 0, 0), (40, 128, 900, 700, 77, 5),
]


@pytest.mark.parametrize("n,ps,ctx,new,pad,short", PLANS)
@pytest.mark.parametrize("in_place", [False, True])
def test_plan_and_release(dev, n, ps, ctx, new, pad, short, in_place):
    from dracohip import lib
    rng = np.random.default_rng(n * 7 + ps)
    kv, q = rng.integers(0, ctx + 1, n), rng.integers(0, new, n)
    kv[0], q[-1] = ps * (ctx // ps), new - 1  # a full last page; a sequence that surely brings tokens
    need = int(sum(-(-(a + b) // ps) - -(-a // ps) for a, b in zip(kv, q)))
    have = int(sum(-(-a // ps) for a in kv))
    n_pages = max(1, have + need - short)
    width = -(-(ctx + new) // ps) + 1
    table, free, n_free = _pool(rng, kv, ps, width, n_pages)
    n_tok = int(q.sum()) + pad
    want = R.plan(kv, q, table, free, n_free, n_pages, ps, n_tok)
    got, d = _plan_call(dev, kv, q, table, free, n_free, n_pages, ps, n_tok, in_place)
    for k, (a, b) in enumerate(zip(got, want)):
        assert np.array_equal(np.asarray(a), np.asarray(b)), k
    if short == 0:
        assert got[6] == (0, 0) and n_free - got[5] == need
    # what the plan took goes back: the list is as it was
    L = lib.load()
    after, n_after = want[4], want[5]
    back = {k: dev.up(np.asarray(v, np.int32)) for k, v in dict(
        block_table=want[3], kv_len=after, keep=np.minimum(after, kv), free_list=free, n_free=[n_after], work=[0]).items()}
    back["kv_len_out"] = back["kv_len"] if in_place else dev.up(np.zeros(n, np.int32))
    back["n_free_out"] = back["n_free"] if in_place else dev.up(np.zeros(1, np.int32))
    a = lib.KvRelease(n_seq=n, max_blocks=width, n_pages=n_pages, page_size=ps, block_table_out=back["block_table"], **back)
    lib.check(L.draco_kv_release(ct.byref(a), None), "draco_kv_release")
    wt, wf, wl, wn = R.release(after, np.minimum(after, kv), want[3], free, n_after, ps)
    assert np.array_equal(dev.down(back["block_table"], wt.shape, np.int32), wt)
    assert np.array_equal(dev.down(back["free_list"], n_pages, np.int32), wf)
    assert np.array_equal(dev.down(back["kv_len_out"], n, np.int32), wl)
    assert int(dev.down(back["n_free_out"], 1, np.int32)[0]) == wn
    assert np.array_equal(wf[:n_free], free[:n_free])


def test_plan_bad_lengths_and_pages(dev):
    """Negative lengths count as 0; what passes the table or the rows is refused; pages outside the pool give no slot."""
    ps, n_pages, width = 16, 6, 3
    kv, q = np.array([-5, 40, 0, 10, 0]), np.array([3, 20, -4, 3, 40])
    table = np.full((5, width), -1, np.int32)
    table[1], table[3, 0] = [0, 1, 2], 99
    free = np.array([4, 77, 3, -1, -1, -1])
    for n_tok in (200, 27, 24):
        want = R.plan(kv, q, table, free, 3, n_pages, ps, n_tok)
        got, _ = _plan_call(dev, kv, q, table, free, 3, n_pages, ps, n_tok)
        for k, (a, b) in enumerate(zip(got, want)):
            assert np.array_equal(np.asarray(a), np.asarray(b)), (n_tok, k, a, b)
    got, _ = _plan_call(dev, np.zeros(0), np.zeros(0), np.zeros((0, 2)), free, 3, n_pages, ps, 5)
    assert (got[2] == -1).all() and got[0][0] == 0 and got[5] == 3
    big = np.array([2 ** 31 - 1] * 3)
    want = R.plan(np.array([0, 5, 0]), big, table[:3], free, 3, n_pages, ps, 20)
    got, _ = _plan_call(dev, np.array([0, 5, 0]), big, table[:3], free, 3, n_pages, ps, 20)
    assert got[6][0] == 3 and np.array_equal(got[0], want[0]) and (got[2] == -1).all() and got[5] == 3


# ---- append ----------------------------------------------------------------------

def _edge_rows(hd, rng):
    """Rows whose blocks sit on the quantizer's borders."""
    x = rng.standard_normal((12, 1, hd)).astype(np.float32)
    x[0] = 0.0
    # every midpoint and its neighbours at scale 1 (largest value 6) and at 2^-23's own
    m = np.array([.25, .75, 1.25, 1.75, 2.5, 3.5, 5.0], np.float32)
    row = np.concatenate([[6.0], m, np.nextafter(m, 9, dtype=np.float32), np.nextafter(m, 0, dtype=np.float32), -m, [-6.0, 0, 0]])[:32]
    x[1] = np.tile(row, hd // 32)
    x[2] = x[1] * np.float32(2.0 ** -20)
    x[3] = x[1] * np.float32(257 / 512)          # scale with 9 significant bits
    x[4] = x[1] * np.float32(513 / 1024)         # scale halfway between two: to the even one
    x[5] = x[1] * np.float32(515 / 1024)
    x[6] = rng.standard_normal(hd) * 1e-30       # every scale rounds to 0
    x[7] = rng.standard_normal(hd) * 6e4         # saturates past 65472
    x[8] = np.float32(3.4028235e38)
    x[9] = rng.standard_normal(hd) * 1e-6
    x[10, 0, :32] = 0.0
    x[11, 0, 5] = np.float32(6 * 2.0 ** -24)     # scale a tie between 0 and 2^-23
    x[11, 0, :5] = x[11, 0, 6:32] = 0.0
    return x


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("code", [F32, F16])
def test_append_quantizes_exactly(dev, hd, code):
    rng = np.random.default_rng(hd)
    x = _edge_rows(hd, rng)
    if code == F16:
        with np.errstate(over="ignore"):
            x = x.astype(np.float16).astype(np.float32)
        x[~np.isfinite(x)] = 65504.0
    T = len(x)
    c = Cache(dev, [T], 1, hd, 16)
    c.append(None, x, x[::-1], c.slots(0, 0, T), code=code)
    k, v = c.read(c.slots(0, 0, T))
    want = R.quantize(x)[2]
    off = [i for i in range(T) if not np.array_equal(k[i], want[i].astype(np.float32))]
    assert not off, (off, k[off[0]], want[off[0]], x[off[0]])
    assert np.array_equal(v, want[::-1].astype(np.float32))
    # the held values are f16 numbers
    assert np.array_equal(k.astype(np.float16).astype(np.float32), k)


@pytest.mark.parametrize("hd,nh,nkv,ps,code,rot,pairing,axes", [
    (64, 15, 5, 16, F32, 64, 0, 1), (64, 4, 4, 64, F16, 16, 1, 2), (128, 32, 8, 32, F32, 128, 1, 3), (128, 6, 2, 128, F16, 128, 0, 4),
    (256, 16, 2, 16, F32, 64, 1, 3), (256, 3, 1, 256, F16, 256, 0, 1), (128, 5, 5, 16, F32, 0, 0, 1), (64, 2, 1, 16, F32, 8, 1, 1)])
@pytest.mark.parametrize("T", [1, 37])
def test_append_rotates_and_writes(dev, hd, nh, nkv, ps, code, rot, pairing, axes, T):
    rng = np.random.default_rng(hd + nh)
    c = Cache(dev, [T + ps], nkv, hd, ps)
    q, k, v = (rng.standard_normal((T, h, hd)).astype(NP[code]) for h in (nh, nkv, nkv))
    slot = c.slots(0, ps // 2, ps // 2 + T)
    if T > 1:
        slot[3] = -1                      # rows without a slot are skipped
        slot[5] = c.n_pages * ps
    rows = 300
    pos = rng.integers(0, rows, (axes, T))
    axis = [i % axes for i in range(rot // 2)]
    ang = np.arange(rows)[:, None] * (10000.0 ** (-np.arange(0, rot, 2) / max(rot, 1)))[None, :] if rot else np.zeros((rows, 0))
    table = np.stack([np.cos(ang), np.sin(ang)], -1).astype(np.float32)
    q_out = dev.up(np.full((T, nh, hd), -777.0, NP[code]))
    c.append(q, k, v, slot, code=code, rot=rot, pairing=pairing, pos=pos, axis=axis, table=table, q_out=q_out)
    real = (slot >= 0) & (slot < c.n_pages * ps)
    got = dev.down(q_out, (T, nh, hd), NP[code])
    want = R.rope(q, pos, axis, table, pairing == 1)
    assert (got[~real] == -777.0).all()
    # one rounding of the exact value (to fp32, or by way of fp32 to f16)
    tol = np.abs(want) * (2.0 ** -24 if code == F32 else 2.0 ** -11 * 1.001) + 2.0 ** -25
    assert (np.abs(got - want)[real] <= tol[real]).all()
    gk, gv = c.read(slot)
    kw = R.quantize(R.rope(k, pos, axis, table, pairing == 1).astype(np.float32))[2]
    assert np.array_equal(gk[real], kw[real].astype(np.float32))
    assert np.array_equal(gv[real], R.quantize(v)[2][real].astype(np.float32))
    assert (gk[~real] == -777.0).all() and (gv[~real] == -777.0).all()
    # no other byte of the pool was written
    pool = dev.down(c.pages, c.n_pages * c.page_bytes, np.uint8)
    written = int(real.sum()) * nkv * hd * 9 // 8
    assert (pool != 0xFF).sum() <= written and (pool == 0xFF).sum() >= pool.size - written


def test_append_strided_and_in_place(dev):
    """q, k, v as slices of one fused buffer, q rotated in place (consecutive pairs)."""
    from dracohip import lib
    rng = np.random.default_rng(4)
    T, nh, nkv, hd, ps = 21, 6, 2, 64, 16
    c = Cache(dev, [T], nkv, hd, ps)
    w = (nh + 2 * nkv) * hd + 24
    buf = rng.standard_normal((T, w)).astype(np.float32)
    p = dev.up(buf)
    pos = np.arange(100, 100 + T)[None]
    ang = np.arange(200)[:, None] * (10000.0 ** (-np.arange(0, hd, 2) / hd))[None, :]
    table = np.stack([np.cos(ang), np.sin(ang)], -1).astype(np.float32)
    a = lib.Kv4Append(code=F32, n_tok=T, n_head=nh, q=p, q_out=p, k=p + 4 * nh * hd, v=p + 4 * (nh + nkv) * hd, q_stride=w,
                      q_out_stride=w, k_stride=w, v_stride=w, slot=dev.up(c.slots(0, 0, T)), rot=hd, pairing=0, n_axes=1,
                      pos=dev.up(pos.astype(np.int32)), pos_stride=T, table=dev.up(table), table_rows=200)
    lib.check(c.L.draco_kv4_append(ct.byref(c.desc), ct.byref(a), None), "append")
    got = dev.down(p, buf.shape, np.float32)
    x = buf[:, :nh * hd].reshape(T, nh, hd)
    want = R.rope(x, pos, [0] * (hd // 2), table, False)
    assert (np.abs(got[:, :nh * hd].reshape(x.shape) - want) <= np.abs(want) * 2.0 ** -24 + 2.0 ** -40).all()
    assert np.array_equal(got[:, nh * hd:], buf[:, nh * hd:])
    gk, gv = c.read(c.slots(0, 0, T))
    k = buf[:, nh * hd:(nh + nkv) * hd].reshape(T, nkv, hd)
    v = buf[:, (nh + nkv) * hd:(nh + 2 * nkv) * hd].reshape(T, nkv, hd)
    assert np.array_equal(gk, R.quantize(R.rope(k, pos, [0] * (hd // 2), table, False).astype(np.float32))[2].astype(np.float32))
    assert np.array_equal(gv, R.quantize(v)[2].astype(np.float32))


# ---- attention ---------------------------------------------------------------------

SHAPES = [(64, 32, 8, 16), (64, 15, 5, 32), (128, 32, 4, 64), (128, 8, 8, 16), (128, 20, 1, 128), (256, 16, 2, 32), (256, 3, 1, 256)]


@pytest.mark.parametrize("hd,nh,nkv,ps", SHAPES)
@pytest.mark.parametrize("code", [F32, F16])
def test_attn_decode(dev, hd, nh, nkv, ps, code):
    """One row a sequence; lengths around units and pages, an empty sequence, one that brings nothing."""
    rng = np.random.default_rng(hd + nh + ps)
    lens = [1, 0, 15, 16, 17, 63, 64, 65, 130, 257, 40, 700]
    c = Cache(dev, lens, nkv, hd, ps)
    held = fill(c, lens, rng, code)
    qlens = [1, 0, 1, 1, 1, 1, 1, 1, 1, 1, 0, 1]
    check_attn(c, held, lens, qlens, nh, rng, code, pad=2)


@pytest.mark.parametrize("hd,nh,nkv,ps", SHAPES)
@pytest.mark.parametrize("window,sink", [(0, 0), (50, 0), (50, 4), (1, 0), (64, 70), (1, 1), (5000, 3)])
def test_attn_ragged_chunks(dev, hd, nh, nkv, ps, window, sink):
    rng = np.random.default_rng(hd + nh + window)
    lens, qlens = [5, 150, 77, 1, 200], [5, 33, 1, 1, 17]
    c = Cache(dev, lens, nkv, hd, ps)
    held = fill(c, lens, rng)
    check_attn(c, held, lens, qlens, nh, rng, window=window, sink=sink)


@pytest.mark.parametrize("hd,nh,nkv,code", [(64, 8, 2, F32), (64, 8, 2, F16), (128, 8, 4, F32), (128, 8, 1, F16), (256, 4, 2, F32), (256, 4, 1, F16)])
@pytest.mark.parametrize("window,sink", [(0, 0), (100, 2), (300, 200)])
def test_attn_prompt(dev, hd, nh, nkv, code, window, sink):
    """Whole prompts and chunks over a prefix, more rows than a block takes."""
    rng = np.random.default_rng(hd + nh + window)
    lens, qlens = [333, 500, 64], [333, 290, 64]
    c = Cache(dev, lens, nkv, hd, 32)
    held = fill(c, lens, rng, code)
    check_attn(c, held, lens, qlens, nh, rng, code, window=window, sink=sink, pad=1)


@pytest.mark.parametrize("hd,code", [(64, F32), (128, F32), (128, F16), (256, F32)])
@pytest.mark.parametrize("window,sink", [(0, 0), (4000, 10)])
def test_attn_long_splits(dev, hd, code, window, sink):
    rng = np.random.default_rng(hd)
    lens, qlens = [9001, 12], [3, 1]
    c = Cache(dev, lens, 2, hd, 64)
    held = fill(c, lens, rng, code)
    out = check_attn(c, held, lens, qlens, 4, rng, code, window=window, sink=sink, pad=3)
    # hints that are too small cost speed only; results are the same every time
    rng2 = np.random.default_rng(hd + 1)
    state = rng2.bit_generator.state
    a = check_attn(c, held, lens, qlens, 4, rng2, code, window=window, sink=sink)
    rng2.bit_generator.state = state
    assert np.array_equal(a, check_attn(c, held, lens, qlens, 4, rng2, code, window=window, sink=sink))
    check_attn(c, held, lens, qlens, 4, rng, code, window=window, sink=sink, max_q=1, max_len=1)
    assert out.shape[0] == 7


def check_sampled(c, lens, qlens, nh, rng, code, window, sink, n_sample):
    """check_attn at n_sample of the rows, the first and last of the longest sequence among them."""
    held = fill(c, lens, rng, code)
    cu = np.concatenate([[0], np.cumsum(qlens)])
    q = (1.5 * rng.standard_normal((int(cu[-1]), nh, c.hd))).astype(NP[code])
    out = c.attn(q, cu, lens, code=code, window=window, sink=sink)
    big = int(np.argmax(qlens))
    rows = np.unique(np.concatenate([[cu[big], cu[big + 1] - 1], rng.choice(int(cu[-1]), min(n_sample, int(cu[-1])), replace=False)]))
    for r in rows:
        s = int(np.searchsorted(cu, r, "right") - 1)
        n, (k, v) = lens[s], held[s]
        want, top = R.attention(q[r:r + 1], k, v, np.array([n - (cu[s + 1] - r)]), c.hd ** -0.5, window, sink)
        err = float(np.abs(out[r:r + 1].astype(np.float64) - want).max())
        lim = bound(code, c.hd, n, top, float(np.abs(v).max()))
        assert np.isfinite(out[r].astype(np.float64)).all() and err <= lim, (s, r, err, lim)
    assert np.isfinite(out.astype(np.float64)).all()


# Row counts at which an MI355X has tiles for every CU: of 256 rows at head dims
# 64 and 128 (f16), of 128 at 128 (fp32) and 256 (f16), of 64 below those.
@pytest.mark.parametrize("hd,nh,nkv,code", [(128, 60, 4, F16), (128, 32, 4, F32), (64, 128, 8, F32), (64, 128, 8, F16), (256, 16, 2, F16),
                                            (256, 16, 2, F32), (128, 16, 4, F32), (128, 20, 4, F16), (64, 32, 4, F16)])
@pytest.mark.parametrize("window,sink", [(0, 0), (150, 70)])
def test_attn_tiles_for_every_cu(dev, hd, nh, nkv, code, window, sink):
    rng = np.random.default_rng(hd + nh + window)
    lens, qlens = [901, 257, 0, 90], [790, 257, 0, 61]
    check_sampled(Cache(dev, lens, nkv, hd, 32), lens, qlens, nh, rng, code, window, sink, 24)


@pytest.mark.parametrize("hd,nh,nkv,code", [(64, 4, 2, F32), (128, 8, 2, F32), (128, 4, 1, F16), (256, 4, 2, F16)])
@pytest.mark.parametrize("most", [1, 4, 7, 30])
def test_attn_many_sequences(dev, hd, nh, nkv, code, most):
    """More sequences than a wave reads at once, some without rows or keys: decode, drafts and chunks."""
    rng = np.random.default_rng(hd + most)
    qlens = [int(x) for x in rng.integers(0, most + 1, 150)]
    qlens[70] = most
    lens = [int(m + x * (rng.random() < 0.7)) for m, x in zip(qlens, rng.integers(0, 300, 150))]
    check_sampled(Cache(dev, lens, nkv, hd, 16), lens, qlens, nh, rng, code, 40 if most == 4 else 0, 3, 60)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("code", [F32, F16])
@pytest.mark.parametrize("most", [1, 7, 15, 40])
@pytest.mark.parametrize("window,sink", [(0, 0), (33, 0), (100, 5), (1, 1), (1000, 200)])
def test_attn_masks_of_every_kernel(dev, hd, code, most, window, sink):
    """Partly masked units (ends, window starts, sinks) in each kernel: 4, 28, 60 and 160 rows a KV head."""
    rng = np.random.default_rng(hd + most + window)
    lens, qlens = [63, 321, most, 200 + most], [1, most, most, max(1, most - 1)]
    c = Cache(dev, lens, 1, hd, 16)
    check_attn(c, fill(c, lens, rng, code), lens, qlens, 4, rng, code, window=window, sink=sink)


@pytest.mark.parametrize("hd,code", [(64, F32), (128, F16)])
@pytest.mark.parametrize("n_seq", [300, 4500])
def test_attn_whole_tiles_of_many_sequences(dev, hd, code, n_seq):
    """The search for a block's sequence in one, two and three steps of 64."""
    rng = np.random.default_rng(hd + n_seq)
    qlens = [int(x) for x in rng.integers(0, 8, n_seq)]
    qlens[n_seq // 2] = 30
    lens = [m + int(x) for m, x in zip(qlens, rng.integers(0, 12, n_seq))]
    check_sampled(Cache(dev, lens, 1, hd, 16), lens, qlens, 16, rng, code, 0, 0, 80)


@pytest.mark.parametrize("hd,code", [(64, F32), (128, F32), (128, F16), (256, F32), (256, F16)])
def test_one_workspace_for_every_shape(dev, hd, code):
    """Calls of different kinds one after another over one workspace, nothing cleared between them."""
    rng = np.random.default_rng(hd)
    lens = [700, 90, 333]
    c = Cache(dev, lens, 2, hd, 16)
    held = fill(c, lens, rng, code)
    work = None
    for qlens in ([1, 1, 1], [5, 3, 0], [6, 7, 7], [20, 1, 31], [300, 90, 200], [1, 0, 1], [16, 2, 9], [6, 7, 7]):
        cu = np.concatenate([[0], np.cumsum(qlens)])
        q = (1.5 * rng.standard_normal((int(cu[-1]), 8, hd))).astype(NP[code])
        out = dev.up(np.full(q.shape, -777.0, NP[code]))
        a = c.attn_args(q, out, cu, lens, code=code)
        if work is None:
            work = a.work, a.work_bytes
        a.work, a.work_bytes = work
        c.lib.check(c.L.draco_kv4_attn(ct.byref(c.desc), ct.byref(a), None), "draco_kv4_attn")
        got = dev.down(out, q.shape, NP[code]).astype(np.float64)
        for s in range(3):
            rows = np.unique(np.clip([0, 1, 5, qlens[s] // 2, qlens[s] - 1], 0, max(qlens[s] - 1, 0)))[:qlens[s]]
            if not len(rows):
                continue
            k, v = held[s]
            want, big = R.attention(q[cu[s] + rows], k, v, lens[s] - qlens[s] + rows, hd ** -0.5, 0, 0)
            err = float(np.abs(got[cu[s] + rows] - want).max())
            assert err <= bound(code, hd, lens[s], big, float(np.abs(v).max())), (qlens, s, err)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("m", [1, 7, 90])
def test_attn_scores_past_fp32_are_nan(dev, hd, m):
    """A row whose scores pass fp32's range is NaN (never a silent 0); the rows beside it are not touched."""
    rng = np.random.default_rng(hd + m)
    n = 200
    c = Cache(dev, [n], 1, hd, 16)
    k, v = np.ones((n, 1, hd), np.float32), rng.standard_normal((n, 1, hd)).astype(np.float32)
    c.append(None, k, v, c.slots(0, 0, n))
    q = rng.standard_normal((m, 4, hd)).astype(np.float32)
    q[:, 1] = 3e37
    q[:, 2] = -3e37
    out = c.attn(q, [0, m], [n], scale=8.0)
    assert np.isnan(out[:, 1:3]).all() and np.isfinite(out[:, [0, 3]]).all()


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("m", [1, 40, 200])
def test_attn_nan_stays_with_the_rows_that_see_it(dev, hd, m):
    """A key row with NaN, a value row with infinity: only rows that see the token are NaN."""
    rng = np.random.default_rng(hd + m)
    n, bad_k, bad_v = 260, 230, 100
    c = Cache(dev, [n], 2, hd, 32)
    k, v = (rng.standard_normal((n, 2, hd)).astype(np.float32) for _ in range(2))
    k[bad_k, 0, 7] = np.nan
    v[bad_v, 1, 40] = -np.inf
    c.append(None, k, v, c.slots(0, 0, n))
    gk, gv = c.read(c.slots(0, 0, n))
    assert np.isnan(gk[bad_k, 0]).all() and np.isnan(gv[bad_k, 0]).all() and np.isfinite(gk[bad_k, 1]).all()
    q = rng.standard_normal((m, 4, hd)).astype(np.float32)
    for window, sink in ((0, 0), (20, 3)):
        out = c.attn(q, [0, m], [n], window=window, sink=sink)
        pos = np.arange(n - m, n)
        for head, bad in ((0, bad_k), (1, bad_v)):
            sees = (pos >= bad) & ((window == 0) | (pos - window < bad) | (bad < sink))
            o = out[:, 2 * head:2 * head + 2]
            assert np.isnan(o[sees]).all() and np.isfinite(o[~sees]).all()
        # the finite rows are right
        kk, vv = np.where(np.isfinite(gk), gk, 0).astype(np.float64), np.where(np.isfinite(gv), gv, 0).astype(np.float64)
        want, big = R.attention(q, kk, vv, pos, hd ** -0.5, window, sink)
        fin = np.isfinite(out)
        assert (np.abs(out - want)[fin] <= bound(F32, hd, n, big, np.abs(vv).max())).all()


@pytest.mark.parametrize("m", [1, 90])
def test_attn_bad_pages_and_lengths(dev, m):
    """A page outside the pool makes the rows that see it NaN; a length past the table, all of its sequence's."""
    rng = np.random.default_rng(9)
    lens = [200, 200, 200]
    c = Cache(dev, lens, 1, 64, 16)
    held = fill(c, lens, rng)
    c.table[0, 2] = c.n_pages + 5
    c.table[1, 0] = -1
    q = rng.standard_normal((3 * m, 2, 64)).astype(np.float32)
    cu = [0, m, 2 * m, 3 * m]
    out = c.attn(q, cu, lens)
    assert np.isnan(out[:2 * m]).all()
    want, big = R.attention(q[2 * m:], *held[2], np.arange(200 - m, 200), 64 ** -0.5, 0, 0)
    assert np.abs(out[2 * m:] - want).max() <= bound(F32, 64, 200, big, np.abs(held[2][1]).max())
    out = c.attn(q, cu, lens, window=60)  # the bad pages are out of sight
    assert np.isfinite(out[[0, m - 1, m, 2 * m - 1]][:, :, 0] if m == 1 else out[m - 1]).all()
    out = c.attn(q, cu, [200, 16 * c.width + 1, 200], window=60)
    assert np.isnan(out[m:2 * m]).all() and np.isfinite(out[2 * m:]).all()
    # more rows than the sequence holds: those before its start see nothing
    out = c.attn(q[:m], [0, m], [0, 0, 0][:1])
    assert (out == 0).all()


def test_attn_large_scores_and_values(dev):
    """Rows of very different size: q from 1e-20 to 1e8, keys up to the format's largest, one that wins by far."""
    rng = np.random.default_rng(3)
    n, hd = 150, 128
    c = Cache(dev, [n], 1, hd, 16)
    k = rng.standard_normal((n, 1, hd)).astype(np.float32)
    v = rng.standard_normal((n, 1, hd)).astype(np.float32)
    v[::7] *= 1e3
    c.append(None, k, v, c.slots(0, 0, n))
    kk, vv = (x.astype(np.float64) for x in c.read(c.slots(0, 0, n)))
    q = rng.standard_normal((6, 4, hd)).astype(np.float32) * np.array([1e-20, 1e-3, 1, 4, 20, 0], np.float32)[:, None, None]
    out = c.attn(q, [0, 6], [n])
    for i in range(6):
        want, big = R.attention(q[i:i + 1], kk, vv, np.array([n - 6 + i]), hd ** -0.5, 0, 0)
        assert np.abs(out[i] - want[0]).max() <= bound(F32, hd, n, big, np.abs(vv).max()), i


def test_pool_past_4_gib(dev):
    """Slots and pages whose byte offsets pass 32 bits."""
    from dracohip import lib
    L = lib.load()
    nkv, hd, ps = 8, 256, 256
    page = L.draco_kv4_page_bytes(ps, nkv, hd)
    n_pages = (1 << 32) // page + 40
    rng = np.random.default_rng(6)
    c = Cache(dev, [10], nkv, hd, ps)
    c.n_pages = n_pages
    c.desc = lib.Kv4(data=dev.empty(n_pages * page), n_pages=n_pages, page_size=ps, n_kv=nkv, head_dim=hd)
    lens, ids = [600], [n_pages - 1, 3, n_pages - 2]
    c.table, c.width = np.array([ids + [-1]], np.int32), 4
    held = fill(c, lens, rng)
    gk, _ = c.read(c.slots(0, 0, 600))
    assert np.array_equal(gk, held[0][0].astype(np.float32))
    check_attn(c, held, lens, [2], 16, rng)


# ---- together -----------------------------------------------------------------------

def _session(dev, hd=128, nh=8, nkv=2, ps=16, n_seq=5, steps=6):
    """Descriptors of a decode loop that keeps its state on the device, in place."""
    from dracohip import lib
    rng = np.random.default_rng(11)
    start = [0, 15, 16, 33, 250][:n_seq]
    c = Cache(dev, start, nkv, hd, ps, spare=12, width=24)
    held = fill(c, start, rng)
    rows = 400
    ang = np.arange(rows)[:, None] * (10000.0 ** (-np.arange(0, hd, 2) / hd))[None, :]
    table = np.stack([np.cos(ang), np.sin(ang)], -1).astype(np.float32)
    up = lambda v, t=np.int32: dev.up(np.asarray(v, t))  # noqa: E731
    n_tok = n_seq + 2  # rows padded
    s = dict(kv=up(start), q_len=up([1] * n_seq), bt=up(c.table), free=up(c.free), n_free=up([c.n_free]), cu=up(np.zeros(n_seq + 1)),
             pos=up(np.zeros(n_tok)), slot=up(np.zeros(n_tok)), st=up([0, 0]), work=up([0]), q=dev.empty(n_tok * nh * hd * 4),
             k=dev.empty(n_tok * nkv * hd * 4), v=dev.empty(n_tok * nkv * hd * 4), table=dev.up(table))
    s["qo"], s["out"] = (dev.up(np.full((n_tok, nh, hd), -777.0, np.float32)) for _ in range(2))
    plan = lib.KvPlan(n_seq=n_seq, max_blocks=c.width, n_pages=c.n_pages, page_size=ps, n_tok=n_tok, block_table=s["bt"], kv_len=s["kv"],
                      q_len=s["q_len"], free_list=s["free"], n_free=s["n_free"], cu_q=s["cu"], pos=s["pos"], slot=s["slot"],
                      kv_len_out=s["kv"], n_free_out=s["n_free"], status=s["st"], work=s["work"])
    app = lib.Kv4Append(code=F32, n_tok=n_tok, n_head=nh, q=s["q"], q_out=s["qo"], k=s["k"], v=s["v"], q_stride=nh * hd, q_out_stride=nh * hd,
                        k_stride=nkv * hd, v_stride=nkv * hd, slot=s["slot"], rot=hd, pairing=1, n_axes=1, pos=s["pos"], pos_stride=n_tok,
                        table=s["table"], table_rows=rows)
    att = lib.Kv4Attn(code=F32, n_seq=n_seq, n_tok=n_tok, max_q=1, max_len=300, n_head=nh, window=0, sink=0, scale=hd ** -0.5,
                      max_blocks=c.width, q=s["qo"], out=s["out"], q_stride=nh * hd, out_stride=nh * hd, cu_q=s["cu"], kv_len=s["kv"],
                      block_table=s["bt"])
    need = c.L.draco_kv4_attn_workspace(ct.byref(c.desc), ct.byref(att))
    att.work, att.work_bytes = dev.up(_workspace(max(need, 16))), need

    def call(stream):
        for f, a in ((c.L.draco_kv_plan, (ct.byref(plan),)), (c.L.draco_kv4_append, (ct.byref(c.desc), ct.byref(app))),
                     (c.L.draco_kv4_attn, (ct.byref(c.desc), ct.byref(att)))):
            rc = f(*a, stream)
            assert rc == 0, c.lib.last_error()

    data = [(rng.standard_normal((n_tok, nh, hd)).astype(np.float32), rng.standard_normal((n_tok, nkv, hd)).astype(np.float32),
             rng.standard_normal((n_tok, nkv, hd)).astype(np.float32)) for _ in range(steps)]
    # the oracle's steps
    want, kv, seqs = [], list(start), [list(h) for h in held]
    for q, k, v in data:
        outs = []
        for i in range(n_seq):
            p = np.array([kv[i]])[None]
            kr = R.quantize(R.rope(k[i:i + 1], p, [0] * (hd // 2), table, True).astype(np.float32))[2]
            qr = R.rope(q[i:i + 1], p, [0] * (hd // 2), table, True).astype(np.float32)
            seqs[i][0] = np.concatenate([seqs[i][0], kr])
            seqs[i][1] = np.concatenate([seqs[i][1], R.quantize(v[i:i + 1])[2]])
            kv[i] += 1
            o, big = R.attention(qr, seqs[i][0], seqs[i][1], np.array([kv[i] - 1]), hd ** -0.5, 0, 0)
            outs.append((o[0], bound(F32, hd, kv[i], big, np.abs(seqs[i][1]).max()) * 1.01))
        want.append(outs)

    def put(i, stream=None):
        for name, x in zip(("q", "k", "v"), data[i]):
            dev.up(x, at=s[name])

    def check(i):
        out = dev.down(s["out"], (n_tok, nh, hd), np.float32)
        for j, (o, tol) in enumerate(want[i]):
            assert np.abs(out[j] - o).max() <= tol, (i, j)
        assert (out[n_seq:] == -777.0).all()
        assert tuple(dev.down(s["st"], 2, np.int32)) == (0, 0)
        assert np.array_equal(dev.down(s["kv"], n_seq, np.int32), np.array(start) + i + 1)

    return call, put, check, s


def test_decode_loop(dev):
    call, put, check, _ = _session(dev)
    st = dev.stream()
    for i in range(6):
        put(i)
        call(st)
        dev.sync(st)
        check(i)


def test_decode_loop_captured(dev):
    """The step as a graph, replayed with eager work of another session between the replays."""
    call, put, check, _ = _session(dev)
    other, oput, ocheck, _ = _session(dev, hd=64, nkv=4, ps=32)
    st, st2 = dev.stream(), dev.stream()
    g = dev.capture(st, lambda: call(st))
    for i in range(6):
        put(i)
        oput(i)
        dev.replay(g, st)
        other(st2)
        dev.sync(st)
        dev.sync(st2)
        check(i)
        ocheck(i)


def test_two_graphs_at_once(dev):
    """Two captured sessions on two streams, each with its own workspace, in flight together."""
    a = _session(dev)
    b = _session(dev, hd=256, nh=4, nkv=1, ps=64)
    s1, s2 = dev.stream(), dev.stream()
    g1, g2 = dev.capture(s1, lambda: a[0](s1)), dev.capture(s2, lambda: b[0](s2))
    for i in range(5):
        a[1](i)
        b[1](i)
        dev.replay(g1, s1)
        dev.replay(g2, s2)
        dev.sync(s1)
        dev.sync(s2)
        a[2](i)
        b[2](i)


def test_null_stream_is_the_librarys(dev):
    call, put, check, _ = _session(dev, n_seq=3, steps=2)
    for i in range(2):
        put(i)
        call(None)
        check(i)
