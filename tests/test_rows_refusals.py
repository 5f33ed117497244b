"""Misuse of the entry points around steps of several rows (caches with a scale
a page, reads, attention of many rows, norms with rotation, verification), refused
before any device call (no GPU)."""

import ctypes

import pytest

from go_whistle_amd import needle
from go_whistle_amd._lib import CQDeviceError, CQPanic, HeadsLayout, KvPaged, check, lib

P = 256  # a pointer that is never dereferenced: the checks come first
FAR = 1 << 40


def cache(**kw):
    c = KvPaged(P, P, None, None, P, 1, 2, 64, 64, 4, 16, 8)
    for k, v in kw.items():
        setattr(c, k, v)
    return ctypes.byref(c)


def read(c=None, k=P, v=P, ks=400, kr=128, vs=400, vr=128, typ=0, batch=2, t=3, rows=None, pos=P):
    check(lib().kv_read_paged_dev(c or cache(), k, ks, kr, v, vs, vr, typ, batch, t, rows, pos, None))


def attend(c=None, out=P, os=768, orow=256, q=P, typ=0, batch=2, t=3, heads=4, rows=None, pos=P, nk=64, window=0, sink=0, scale=8.0):
    check(lib().kv_attend_rows_paged_dev(c or cache(), out, os, orow, q, 768, 256, typ, batch, t, heads, rows, pos, nk, window,
                                         sink, scale, None))


def norm(qo=P, ko=P, q=FAR, k=FAR, typ=0, layout=None, batch=2, t=3, heads=4, kv_heads=2, width=64, cos=P, sin=P, positions=10,
         pos=P, rows=None):
    y = ctypes.byref(layout) if layout is not None else None
    check(lib().nd_qk_norm_rope_dev(qo, ko, q, k, typ, y, batch, t, heads, kv_heads, width, P, P, cos, sin, positions, pos, rows,
                                    None))


def verify(acc=P, tok=2 * P, lp=4 * P, target=FAR, draft=FAR, typ=0, batch=2, t=3, n=100, drafts=FAR, drafted=None, u=FAR, nxt=FAR,
           temperature=1.0):
    check(lib().nd_verify_drafts_dev(acc, tok, lp, target, 400, 100, draft, 300, 100, typ, batch, t, n, drafts, drafted, u, nxt,
                                     temperature, None))


def append(c):
    check(lib().kv_append_paged_dev(c, P, 0, 0, P, 0, 0, 0, 2, 3, None, P, 64, None, 0, None))


def attend_one(c):
    check(lib().kv_attend_paged_dev(c, P, 0, P, 0, 0, 2, 4, P, 64, 8.0, None, None, 0, None))


def evict(c):
    check(lib().kv_evict_paged_dev(c, P, 4, P, 64, 8 * P, 64, P, P, P, 2, 64, 32, 4, 4, None))


@pytest.mark.parametrize("typ", [5, 6])
@pytest.mark.parametrize("call", [append, attend_one, evict, lambda c: attend(c), lambda c: read(c)])
def test_page_scales_are_asked_for(call, typ):
    for kw in (dict(), dict(ks=P), dict(vs=P)):
        with pytest.raises(CQPanic, match="nil cache array"):
            call(cache(type=typ, **kw))


@pytest.mark.parametrize("typ", [5, 6])
def test_eviction_of_page_scales(typ):
    with pytest.raises(CQDeviceError, match="scale a page"):
        evict(cache(type=typ, ks=P, vs=P))


@pytest.mark.parametrize("call", [lambda c: attend(c), lambda c: read(c)])
@pytest.mark.parametrize("edit,err", [(dict(type=4), CQPanic), (dict(type=7), CQPanic), (dict(type=-1), CQPanic),
                                      (dict(kv_heads=0), CQPanic), (dict(qk=40), CQDeviceError), (dict(vd=272), CQDeviceError),
                                      (dict(page_rows=12), CQPanic), (dict(pool_pages=0), CQPanic), (dict(page_stride=-1), CQPanic),
                                      (dict(k=None), CQPanic), (dict(v=None), CQPanic), (dict(pages=None), CQPanic),
                                      (dict(k=P + 8), CQPanic), (dict(pool_pages=1 << 30, page_rows=4, page_stride=64), CQDeviceError)])
def test_bad_caches(call, edit, err):
    with pytest.raises(err):
        call(cache(**edit))


@pytest.mark.parametrize("call,kw", [
    (read, dict(batch=-1)), (read, dict(t=-1)), (read, dict(typ=3)), (read, dict(typ=-1)), (read, dict(k=None)), (read, dict(v=None)),
    (read, dict(pos=None)), (read, dict(k=P + 2)), (read, dict(typ=1, v=P + 1)), (read, dict(kr=127)), (read, dict(vs=100)),
    (attend, dict(batch=-1)), (attend, dict(t=-1)), (attend, dict(nk=-1)), (attend, dict(nk=65)), (attend, dict(window=-1)),
    (attend, dict(sink=-1)), (attend, dict(typ=3)), (attend, dict(heads=3)), (attend, dict(heads=0)), (attend, dict(scale=0.0)),
    (attend, dict(scale=-1.0)), (attend, dict(scale=float("nan"))), (attend, dict(scale=1e-40)), (attend, dict(out=None)),
    (attend, dict(q=None)), (attend, dict(pos=None)), (attend, dict(q=P + 2)), (attend, dict(typ=2, out=P + 1)),
    (attend, dict(os=768, orow=255)), (attend, dict(os=0, orow=0)), (attend, dict(os=768, orow=0)), (attend, dict(os=700, orow=256)), (attend, dict(os=255, orow=256, rows=P)),
    (norm, dict(batch=-1)), (norm, dict(t=-1)), (norm, dict(heads=-1)), (norm, dict(kv_heads=-1)), (norm, dict(typ=3)),
    (norm, dict(positions=-1)), (norm, dict(cos=None)), (norm, dict(sin=None)), (norm, dict(pos=None)), (norm, dict(q=None)),
    (norm, dict(k=None)), (norm, dict(qo=None)), (norm, dict(ko=None)), (norm, dict(q=FAR + 2)), (norm, dict(typ=1, k=FAR + 1)),
    (verify, dict(batch=-1)), (verify, dict(t=-1)), (verify, dict(n=0)), (verify, dict(typ=3)), (verify, dict(temperature=-1.0)),
    (verify, dict(temperature=float("nan"))), (verify, dict(temperature=float("inf"))), (verify, dict(temperature=1e-310)),
    (verify, dict(acc=None)), (verify, dict(tok=None)), (verify, dict(target=None)), (verify, dict(drafts=None)), (verify, dict(u=None)),
    (verify, dict(nxt=None)), (verify, dict(target=FAR + 2)), (verify, dict(typ=2, draft=FAR + 1)),
    (verify, dict(drafts=2 * P)), (verify, dict(drafted=P)), (verify, dict(u=4 * P + 4)), (verify, dict(nxt=2 * P + 8)),
    (verify, dict(tok=P + 4)), (verify, dict(lp=2 * P + 12)),
])
def test_misuse(call, kw):
    with pytest.raises(CQPanic):
        call(**kw)


@pytest.mark.parametrize("call,kw", [
    (read, dict(batch=1 << 20, t=64, kr=128, ks=1 << 20, vr=128, vs=1 << 20)), (norm, dict(width=40)), (norm, dict(width=272)),
    (norm, dict(width=0)), (norm, dict(batch=1 << 16, t=1 << 14, layout=None, q=1 << 60, k=1 << 61, qo=FAR, ko=1 << 59)),
    (attend, dict(batch=1 << 16, t=1 << 16, os=1 << 24)), (verify, dict(n=(1 << 30) + 1)), (verify, dict(t=(1 << 20) + 1)),
    (verify, dict(batch=1 << 24, n=1 << 20, tok=1 << 50, lp=1 << 51, drafts=1 << 52, u=1 << 53, nxt=1 << 54)),
])
def test_unsupported(call, kw):
    with pytest.raises(CQDeviceError):
        call(**kw)


@pytest.mark.parametrize("call,kw", [
    (read, dict(batch=0)), (read, dict(t=0)), (attend, dict(batch=0)), (attend, dict(t=0)), (attend, dict(nk=0)), (norm, dict(batch=0)),
    (norm, dict(t=0)), (norm, dict(heads=0, kv_heads=0)), (verify, dict(batch=0)),
])
def test_nothing_to_do(call, kw):
    call(**kw)


def spread(batch, t, places):
    """Whether rows of several arrays, (address, width, stream, row) in elements, share none, by counting."""
    seen = set()
    for at, width, stream, row in places:
        for b in range(batch):
            for i in range(t):
                x = at + b * stream + i * row
                span = set(range(x, x + width))
                if seen & span:
                    return False
                seen |= span
    return True


@pytest.mark.parametrize("t", [1, 3])
@pytest.mark.parametrize("off", [0, 64, 128, 255, 256, 320, 384, 512, 513, 640, 768])
def test_norms_onto_a_part_of_others(t, off):
    # queries of 256 and keys of 128 side by side in rows of 640; the query's output `off` from its input
    base = 1 << 20
    y = HeadsLayout(640 * t, 640, 640 * t, 640, 640 * t, 640, 128 * t, 128)
    apart = off == 0 or spread(2, t, [(base, 256, 640 * t, 640), (base + off, 256, 640 * t, 640)])
    apart = apart and (spread(2, t, [(base + 256, 128, 640 * t, 640), (base + off, 256, 640 * t, 640)]))
    call = lambda: norm(qo=4 * (base + off), ko=FAR, q=4 * base, k=4 * (base + 256), layout=y, t=t, pos=P if not apart else None)  # noqa: E731
    # the nil positions are the next check
    if apart:
        with pytest.raises(CQPanic, match="without positions"):
            call()
    else:
        with pytest.raises(CQPanic, match="onto a part"):
            call()


def test_wrappers_refuse_host_tensors_and_shapes():
    import torch

    q = torch.zeros(2, 3, 4, 64)
    for args in ((q, q, q, q), (None, None, None, None), (q, None, None, None), (q[0], None, q[0], None)):
        with pytest.raises(CQPanic):
            needle.qk_norm_rope_dev(*args)
    x, d = torch.zeros(2, 4, 10), torch.zeros(2, 3, dtype=torch.int32)
    for target, drafts in ((x, d), (x[0], d), (x, d[0])):
        with pytest.raises(CQPanic):
            needle.verify_drafts_dev(d[:, 0], x[..., 0], target, drafts)
    k = torch.zeros(4, 16, 2, 64, dtype=torch.int8)
    with pytest.raises(CQPanic):
        needle.PagedKV(k, k, torch.zeros(2, 2, dtype=torch.int32), torch.zeros(4, 2), torch.zeros(4, 2))
