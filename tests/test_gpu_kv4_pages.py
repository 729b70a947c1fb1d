"""Releases whose block tables hold entries that are no pages: the caller took
the pages behind a sliding window back and left -1."""
import ctypes as ct

import numpy as np
import pytest

import kv4_ref as R
from test_gpu_kv4 import _plan_call, _pool, dev  # noqa: F401 (dev is a fixture)

pytestmark = pytest.mark.gpu


def _release(dev, kv, keep, table, free, n_free, n_pages, ps, in_place=False):  # noqa: F811
    from dracohip import lib
    n = len(kv)
    d = {k: dev.up(np.asarray(v, np.int32)) for k, v in dict(
        block_table=table, kv_len=kv, keep=keep, free_list=free, n_free=[n_free], work=[0]).items()}
    d["block_table_out"] = d["block_table"] if in_place else dev.up(table.astype(np.int32))
    d["kv_len_out"] = d["kv_len"] if in_place else dev.up(np.full(n, -9, np.int32))
    d["n_free_out"] = d["n_free"] if in_place else dev.up(np.full(1, -9, np.int32))
    a = lib.KvRelease(n_seq=n, max_blocks=table.shape[1], n_pages=n_pages, page_size=ps, **d)
    lib.check(lib.load().draco_kv_release(ct.byref(a), None), "draco_kv_release")
    assert dev.down(d["work"], 1, np.int32)[0] == 0
    return (dev.down(d["block_table_out"], table.shape, np.int32), dev.down(d["free_list"], n_pages, np.int32),
            dev.down(d["kv_len_out"], n, np.int32), int(dev.down(d["n_free_out"], 1, np.int32)[0]))


def _want(kv, keep, table, free, n_free, n_pages, ps):
    """The release by its definition: pages of the pool only, in the reverse of their order, no more than the list holds."""
    table, back, out = table.copy(), [], []
    for s, (a, k) in enumerate(zip(kv.tolist(), keep.tolist())):
        k = min(max(k, 0), a)
        for b in range(-(-k // ps), -(-a // ps)):
            if 0 <= table[s, b] < n_pages:
                back.append(table[s, b])
            table[s, b] = -1
        out.append(k)
    full = np.concatenate([free[:n_free], back[::-1]]).astype(np.int64)[:n_pages]
    return table, full, np.array(out)


@pytest.mark.parametrize("n", [1, 5, 16, 17, 100, 257, 300, 1025, 2500])
@pytest.mark.parametrize("share", [0.02, 0.5, 1.0])
@pytest.mark.parametrize("in_place", [False, True])
def test_release_of_windowed_sessions(dev, n, share, in_place):  # noqa: F811
    """A share of the sessions has lost its front pages to the free list; their release puts no -1 there and loses no page."""
    rng = np.random.default_rng(n)
    ps, width = 16, 40
    kv = rng.integers(0, ps * width - 5, n)
    kv[0] = ps * width - 7
    have = -(-kv // ps)
    n_pages = int(have.sum()) + 7
    table, free, n_free = _pool(rng, kv, ps, width, n_pages)
    for s in range(n):
        if s == 0 or rng.random() < share:  # the pages wholly behind the window go back by the caller's hand
            first = min(int(rng.integers(0, 3)), have[s])  # (sinks' pages stay)
            last = max(first, int(have[s]) - int(rng.integers(1, 6)))
            gone = table[s, first:last].copy()
            free[n_free:n_free + len(gone)] = gone
            n_free += len(gone)
            table[s, first:last] = rng.choice([-1, n_pages, n_pages + 70], len(gone))
    keep = np.where(rng.random(n) < 0.6, 0, np.maximum(kv - rng.integers(0, 60, n), 0))
    wt, wf, wl = _want(kv, keep, table, free, n_free, n_pages, ps)
    t, f, ln, count = _release(dev, kv, keep, table, free, n_free, n_pages, ps, in_place)
    assert count == len(wf) and np.array_equal(f[:count], wf) and np.array_equal(t, wt) and np.array_equal(ln, wl)
    # every page is in one place
    held = t[(t >= 0) & (t < n_pages)]
    assert np.array_equal(np.sort(np.concatenate([f[:count], held])), np.arange(n_pages))
    # and a plan that takes all of the list gives every token a slot
    new = np.zeros(1, np.int64), np.array([count * ps])
    got, _ = _plan_call(dev, *new, np.full((1, count + 1), -1, np.int32), f, count, n_pages, ps, count * ps)
    assert got[6] == (0, 0) and (got[2] >= 0).all() and len(np.unique(got[2])) == count * ps


@pytest.mark.parametrize("n", [3, 40, 300])
def test_release_past_the_list(dev, n):  # noqa: F811
    """More pages than the list has room for (they are in it already): it ends full, and the table's entries are gone."""
    rng = np.random.default_rng(n)
    ps, width = 32, 6
    kv = rng.integers(1, ps * width, n)
    n_pages = int((-(-kv // ps)).sum()) + 2
    table, free, n_free = _pool(rng, kv, ps, width, n_pages)
    more = n_pages - 3 - n_free
    free[n_free:n_free + more] = table[table >= 0][:more]
    n_free += more
    keep = np.zeros(n, np.int64)
    wt, wf, wl = _want(kv, keep, table, free, n_free, n_pages, ps)
    t, f, ln, count = _release(dev, kv, keep, table, free, n_free, n_pages, ps)
    assert count == len(wf) == n_pages and np.array_equal(f, wf) and np.array_equal(t, wt) and np.array_equal(ln, wl)
    assert (R.release(kv, keep, table, np.full(2 * n_pages, -1), n_free, ps)[0] == t).all()
