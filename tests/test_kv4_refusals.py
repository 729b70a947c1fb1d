"""Refusals of the paged 4-bit KV cache's entry points: every bad argument is
answered -1 with a message before the device is touched (CPU only)."""
import ctypes as ct

import pytest

from dracohip import lib

L = lib.load()
P = 4096  # a non-null, aligned address that nothing reads


def cache(**kw):
    return lib.Kv4(**{**dict(data=P, n_pages=4, page_size=16, n_kv=2, head_dim=64), **kw})


def refused(rc, word):
    assert rc == -1
    assert word in lib.last_error(), lib.last_error()


def test_page_bytes():
    assert L.draco_kv4_page_bytes(16, 5, 64) == 16 * 5 * 72
    assert L.draco_kv4_page_bytes(256, 2, 256) == 256 * 2 * 288
    for ps, nkv, hd in ((8, 1, 64), (48, 1, 64), (512, 1, 64), (16, 0, 64), (16, 1, 96)):
        assert L.draco_kv4_page_bytes(ps, nkv, hd) == 0


CACHES = [(dict(data=None), "no cache"), (dict(head_dim=96), "head dim"), (dict(page_size=24), "page size"), (dict(page_size=8), "page size"),
          (dict(n_kv=0), "bad cache"), (dict(n_pages=0), "bad cache"), (dict(n_pages=1 << 28), "bad cache"), (dict(data=P + 4), "aligned")]


@pytest.mark.parametrize("kw,word", CACHES)
def test_bad_caches(kw, word):
    c = cache(**kw)
    refused(L.draco_kv4_append(ct.byref(c), ct.byref(append()), None), word)
    refused(L.draco_kv4_attn(ct.byref(c), ct.byref(attn()), None), word)
    refused(L.draco_kv4_read(ct.byref(c), P, 1, P, P, None), word)
    assert L.draco_kv4_attn_workspace(ct.byref(c), ct.byref(attn())) == 0


def append(**kw):
    axis = kw.pop("axis", [])
    a = lib.Kv4Append(**{**dict(code=9, n_tok=3, n_head=4, q=P, q_out=2 * P, k=P, v=P, q_stride=256, q_out_stride=256, k_stride=128,
                                v_stride=128, slot=P, rot=64, pairing=1, n_axes=1, pos=P, pos_stride=3, table=P, table_rows=9), **kw})
    for i, x in enumerate(axis):
        a.axis[i] = x
    return a


@pytest.mark.parametrize("kw,word", [
    (dict(code=0), "type code"), (dict(n_tok=-1), "n_tok"), (dict(n_head=3), "q heads"), (dict(n_head=-2), "q heads"),
    (dict(q=None), "q is null"), (dict(q_out=None), "q_out is null"), (dict(k=None), "k is null"), (dict(v=P + 8), "aligned"),
    (dict(k_stride=132), "aligned"), (dict(k_stride=64), "stride"), (dict(q_stride=248), "stride"), (dict(v_stride=-128), "stride"),
    (dict(slot=None), "slot"), (dict(rot=12), "rot"), (dict(rot=72), "rot"), (dict(rot=-8), "rot"), (dict(pos=None), "without"),
    (dict(table=None), "without"), (dict(table_rows=0), "without"), (dict(table=P + 4), "table"), (dict(pairing=2), "pairing"),
    (dict(n_axes=0), "axes"), (dict(n_axes=5), "axes"), (dict(n_axes=2, pos_stride=2), "axes"), (dict(axis=[0, 1]), "axis"),
    (dict(q_out=P), "q_out is q")])
def test_append_refuses(kw, word):
    refused(L.draco_kv4_append(ct.byref(cache()), ct.byref(append(**kw)), None), word)


def attn(**kw):
    return lib.Kv4Attn(**{**dict(code=9, n_seq=2, n_tok=2, max_q=1, max_len=20, n_head=4, window=0, sink=0, scale=0.125, max_blocks=3, q=P,
                                 out=2 * P, q_stride=256, out_stride=256, cu_q=P, kv_len=P, block_table=P), **kw})


@pytest.mark.parametrize("kw,word", [
    (dict(code=5), "type code"), (dict(n_seq=-1), "bad batch"), (dict(n_tok=-1), "n_tok"), (dict(max_q=0), "max_q"), (dict(max_len=-1), "max_q"),
    (dict(n_head=5), "q heads"), (dict(n_head=0), "q heads"), (dict(window=-1), "window"), (dict(sink=-1), "window"), (dict(scale=0.0), "scale"),
    (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(max_blocks=0), "bad batch"),
    (dict(max_blocks=1 << 28), "slots"), (dict(q=None), "q is null"), (dict(out=P + 8), "aligned"), (dict(q_stride=250), "aligned"),
    (dict(out_stride=128), "stride"), (dict(out=P), "out is q"), (dict(cu_q=None), "null"), (dict(kv_len=None), "null"), (dict(block_table=None), "null")])
def test_attn_refuses(kw, word):
    refused(L.draco_kv4_attn(ct.byref(cache()), ct.byref(attn(**kw)), None), word)


def test_plan_and_release_refuse():
    ok = dict(n_seq=2, max_blocks=3, n_pages=4, page_size=16, n_tok=5, block_table=P, kv_len=P, q_len=P, free_list=P, n_free=P, cu_q=P, pos=None,
              slot=P, kv_len_out=P, n_free_out=P, status=P, work=P)
    for kw, word in [(dict(n_seq=-1), "bad batch"), (dict(max_blocks=0), "bad batch"), (dict(n_pages=0), "bad batch"), (dict(page_size=17), "page size"),
                     (dict(n_pages=1 << 29), "slots"), (dict(n_tok=-3), "n_tok")] + [({k: None}, "null") for k in ok if isinstance(ok[k], int) and ok[k] == P]:
        refused(L.draco_kv_plan(ct.byref(lib.KvPlan(**{**ok, **kw})), None), word)
    rel = dict(n_seq=2, max_blocks=3, n_pages=4, page_size=16, block_table=P, block_table_out=P, kv_len=P, keep=P, free_list=P, n_free=P,
               kv_len_out=P, n_free_out=P, work=P)
    for kw, word in [(dict(n_seq=-1), "bad batch"), (dict(page_size=1), "page size")] + [({k: None}, "null") for k in rel if rel[k] == P]:
        refused(L.draco_kv_release(ct.byref(lib.KvRelease(**{**rel, **kw})), None), word)
    refused(L.draco_kv_plan(None, None), "arguments")
    refused(L.draco_kv_release(None, None), "arguments")


def test_read_refuses():
    c = cache()
    refused(L.draco_kv4_read(ct.byref(c), P, -1, P, P, None), "n -1")
    refused(L.draco_kv4_read(ct.byref(c), None, 1, P, P, None), "null")
    refused(L.draco_kv4_read(ct.byref(c), P, 1, P + 4, P, None), "aligned")
    refused(L.draco_kv4_read(None, P, 1, P, P, None), "no cache")


def test_nothing_to_do_is_no_error():
    c = cache()
    assert L.draco_kv4_append(ct.byref(c), ct.byref(append(n_tok=0)), None) == 0
    assert L.draco_kv4_read(ct.byref(c), P, 0, P, P, None) == 0
    assert L.draco_kv4_attn(ct.byref(c), ct.byref(attn(n_tok=0, n_seq=0)), None) == 0


@pytest.mark.parametrize("n,ok", [((0x7FFFFF00 // 16), True), ((0x7FFFFF00 // 16) + 1, False)])
def test_slots_stay_ints_a_step_past_the_last(n, ok):
    """2^31 - 256 slots at most: the last step of keys of a sequence may begin in them and end behind them."""
    c = cache(n_pages=n)
    rc = L.draco_kv4_read(ct.byref(c), P, 0, P, P, None)
    assert rc == (0 if ok else -1)
    rc = L.draco_kv4_attn(ct.byref(cache()), ct.byref(attn(max_blocks=n, n_tok=0)), None)
    assert rc == (0 if ok else -1)
    if not ok:
        assert "slots" in lib.last_error()


def test_more_rows_than_ints_count():
    refused(L.draco_kv_plan(ct.byref(lib.KvPlan(n_seq=0, max_blocks=1, n_pages=1, page_size=16, n_tok=(1 << 30) + 1)), None), "n_tok")
    refused(L.draco_kv4_attn(ct.byref(cache()), ct.byref(attn(n_tok=0x7FFFFFFF // 4)), None), "n_tok")


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_one_workspace_size_serves_every_batch(hd):
    c = cache(head_dim=hd)
    sizes = {L.draco_kv4_attn_workspace(ct.byref(c), ct.byref(attn(code=code, n_seq=s, n_tok=t, max_q=q, n_head=h)))
             for code in (7, 9) for s, t, q in ((0, 0, 1), (1, 1, 1), (3, 70, 50), (9, 4000, 4000)) for h in (2, 64)}
    assert len(sizes) == 1 and sizes.pop() >= 16384


@pytest.mark.parametrize("pairing,rot", [(0, 64), (0, 0), (1, 0)])
def test_append_in_place_needs_one_stride(pairing, rot):
    """q rotated in place: rows of another stride would lie over other tokens' rows."""
    kw = dict(q_out=P, pairing=pairing, rot=rot)
    refused(L.draco_kv4_append(ct.byref(cache()), ct.byref(append(q_out_stride=264, **kw)), None), "q_out is q")
    refused(L.draco_kv4_append(ct.byref(cache()), ct.byref(append(q_stride=264, **kw)), None), "q_out is q")


def test_more_threads_than_a_launch_has():
    """2^24 blocks of 256 threads are one too many."""
    c = cache()
    refused(L.draco_kv4_append(ct.byref(c), ct.byref(append(n_tok=1 << 26, pos_stride=1 << 26)), None), "more blocks")
    refused(L.draco_kv4_append(ct.byref(c), ct.byref(append(n_tok=1 << 28, n_head=0, rot=0)), None), "more blocks")
    refused(L.draco_kv4_read(ct.byref(c), P, 1 << 28, P, P, None), "more blocks")
