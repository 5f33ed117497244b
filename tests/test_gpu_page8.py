"""8-bit paged caches with one scale a page and head: the append's codes and
scales in exact steps, the read-back of caches of any type, and the attention of
one token over them (bounds in tests/serve_ref.py, tests/page8_ref.py)."""

import math

import numpy as np
import pytest

from go_whistle_amd import needle
from go_whistle_amd._lib import CQDeviceError
from page8_ref import CACHES, FLOATS, append_pages, cache_rows, gen, i32, make_cache, widened
from serve_ref import attend64, host

pytestmark = pytest.mark.gpu

CODES = ["i8p", "e4m3"]


def stream_state(c, b):
    """A stream's codes' values [rows, heads, width] and scales [pages, heads], of keys and values."""
    import torch

    pg = c.pages[b].long()
    return [(widened(x[pg].flatten(0, 1)), host(s[pg]).astype(np.float32)) for x, s in ((c.k, c.ks), (c.v, c.vs))]


def same_state(c, b, want, upto, R):
    """Codes up to row `upto` and the scales of their pages; a NaN code is NaN."""
    for (got_x, got_s), (x, s) in zip(stream_state(c, b), want):
        pages = -(-upto // R)
        assert np.array_equal(got_s[:pages], s[:pages]), b
        assert np.array_equal(got_x[:upto], x[:upto], equal_nan=True), b


def append_and_check(c, name, k, v, pos, rows, cap, upto):
    import torch

    R, B, t = c.k.shape[1], *k.shape[:2]
    want = [stream_state(c, b) for b in range(B)]
    c.append_dev(k, v, i32(pos), rows=None if rows is None else i32(rows), cap=cap)
    torch.cuda.synchronize()
    for b in range(B):
        n = t if rows is None else rows[b]
        n = n if 0 <= n <= t else 0
        lo, hi = max(pos[b], 0), min(pos[b] + n, cap)
        for x, (state, scales) in zip((k, v), want[b]):
            if hi > lo:
                append_pages(state, scales, host(x[b])[lo - pos[b]:hi - pos[b]].astype(np.float32), lo, hi - lo, R, name)
        same_state(c, b, want[b], max(hi, 0) if hi > lo else upto, R)


@pytest.mark.parametrize("io", FLOATS)
@pytest.mark.parametrize("name", CODES)
@pytest.mark.parametrize("Hk,qk,vd,R", [(8, 64, 64, 16), (2, 48, 64, 1), (3, 128, 16, 8), (1, 256, 240, 64), (5, 80, 96, 2),
                                        (2, 16, 32, 256)])
@pytest.mark.parametrize("t", [1, 2, 7, 40, 300])
def test_append(name, io, Hk, qk, vd, R, t):
    import torch

    B, cap = 5, 400
    g = gen(t * R + Hk)
    c = make_cache(g, name, B, -(-cap // R), R, Hk, qk, vd, 3)
    size = torch.exp(torch.randn(B, t, 1, 1, generator=g, device="cuda"))
    mk = lambda w: (size * torch.randn(B, t, Hk, w, generator=g, device="cuda")).to(getattr(torch, io))  # noqa: E731
    pos = [0, 5, R, cap - t, max(0, cap - t - 3)]
    append_and_check(c, name, mk(qk), mk(vd), pos, None, cap, 0)
    append_and_check(c, name, mk(qk), mk(vd), pos, [t, 0, max(1, t - 1), 1, t + 1], cap, 0)


@pytest.mark.parametrize("name", CODES)
def test_append_token_by_token(name):
    # rows that grow, shrink and are zero: the scale of a begun page never falls, a new page's begins anew
    import torch

    B, R, Hk, w = 3, 8, 2, 32
    g = gen(7)
    c = make_cache(g, name, B, 5, R, Hk, w, w)
    size = [0.0, 1e-3, 1e3, 1.0, 0.0, 1e4, 1.0, 1.0, 0.5, 2.0, 4.0, 8.0, 1e-30, 3.0]
    for i, z in enumerate(size):
        mk = lambda: z * torch.randn(B, 1, Hk, w, generator=g, device="cuda")  # noqa: E731
        append_and_check(c, name, mk(), mk(), [i, i + 5, i + 7], None, 40, 0)
    # drafts taken back: the rows before stay, the next ones go over the refused ones
    mk = lambda t: torch.randn(B, t, Hk, w, generator=g, device="cuda")  # noqa: E731
    append_and_check(c, name, mk(5), mk(5), [14, 19, 21], None, 40, 0)
    append_and_check(c, name, mk(2), mk(2), [16, 20, 22], None, 40, 0)


@pytest.mark.parametrize("name", CODES)
def test_append_values_that_are_not_finite_and_subnormal(name):
    import torch

    g = gen(9)
    c = make_cache(g, name, 2, 2, 16, 2, 32, 32)
    x = torch.randn(2, 16, 2, 32, generator=g, device="cuda")
    x[0, 3, 0, 5], x[0, 4, 0, 6], x[0, 5, 1, 7], x[1, 0, 0, 0] = math.inf, -math.inf, math.nan, math.nan
    x[1, :, 1] = 0
    x[1, 2, 1, 3], x[1, 3, 1, 4] = 1e-44, -3e-39
    append_and_check(c, name, x, x.flip(1).contiguous(), [0, 0], None, 32, 0)
    append_and_check(c, name, x[:, :3], x[:, 5:8], [16, 14], None, 32, 0)


def test_append_leaves_the_rest():
    # bad pages, positions outside the cache, padded slots; the accumulated weights
    import torch

    g = gen(11)
    c = make_cache(g, "i8p", 6, 4, 16, 2, 64, 64, 4)
    c.pages[0, 0], c.pages[1, 1] = -1, 10 ** 6
    x = torch.randn(6, 20, 2, 64, generator=g, device="cuda")
    before = [t.clone() for t in (c.k, c.v, c.ks, c.vs)]
    acc = torch.full((6, 2, 64), 5.0, device="cuda")
    pos, rows = [3, 10, -4, 60, 64, 0], [20, 20, 20, 20, 3, -1]
    c.append_dev(x, x, i32(pos), rows=i32(rows), cap=64, acc=acc)
    torch.cuda.synchronize()
    touched = torch.zeros(c.k.shape[0], dtype=torch.bool, device="cuda")
    for b, p in ((0, [1]), (1, [0]), (2, [0]), (3, [3])):
        touched[c.pages[b, p].long()] = True
    for t, o in zip((c.k, c.v, c.ks, c.vs), before):
        assert torch.equal(t[~touched], o[~touched]) and not torch.equal(t[touched], o[touched])
    want = torch.full((6, 2, 64), 5.0)
    want[0, :, 16:23] = 0
    want[1, :, 10:16] = 0
    want[2, :, :16] = 0
    want[3, :, 60:] = 0
    assert torch.equal(acc.cpu(), want)


def test_append_strided_rows():
    # views of one product's rows, unaligned ones too
    import torch

    for off, io in ((0, torch.bfloat16), (1, torch.bfloat16), (3, torch.float32)):
        g = gen(off)
        whole = torch.randn(3, 9, off + 2 * 2 * 64 + 5, generator=g, device="cuda").to(io)
        k, v = (whole[..., off + z * 128:off + (z + 1) * 128].unflatten(-1, (2, 64)) for z in range(2))
        c = make_cache(g, "e4m3", 3, 4, 8, 2, 64, 64)
        append_and_check(c, "e4m3", k, v, [0, 3, 8], None, 32, 0)


def test_fork_copies_pages_with_their_scales():
    import ctypes

    import torch

    from go_whistle_amd._lib import check, lib

    g = gen(12)
    c = make_cache(g, "i8p", 2, 2, 16, 3, 32, 48, 2)
    src, dst = c.pages[0].clone(), c.pages[1].clone()
    for q, s, w in ((c.k, c.ks, 32), (c.v, c.vs, 48)):
        check(lib().kv_page_copy_dev(ctypes.c_void_p(q.data_ptr()), ctypes.c_void_p(s.data_ptr()),
                                     ctypes.c_void_p(src.data_ptr()), ctypes.c_void_p(dst.data_ptr()), 2, 1, 16 * 3 * w,
                                     16 * w, c.k.shape[0], None))
    torch.cuda.synchronize()
    for x in (c.k, c.v, c.ks, c.vs):
        assert torch.equal(x[src.long()], x[dst.long()])


@pytest.mark.parametrize("io", FLOATS)
@pytest.mark.parametrize("name", CACHES)
@pytest.mark.parametrize("Hk,qk,vd,R", [(8, 64, 64, 16), (2, 48, 64, 1), (1, 256, 240, 64), (5, 80, 16, 4)])
def test_read(name, io, Hk, qk, vd, R):
    import torch

    B, t = 5, 33
    g = gen(Hk * R)
    c = make_cache(g, name, B, -(-80 // R), R, Hk, qk, vd)
    cap = c.cap
    dt = getattr(torch, io)
    pos, rows = [0, cap - 10, 5, -3, cap], [33, 33, 0, 20, 7]
    # outputs with room behind their rows, off the 16-byte grid for one of them
    k, v = torch.full((B, t, Hk * qk + 5), 9.0, device="cuda", dtype=dt), torch.full((B, t, Hk * vd), 9.0, device="cuda", dtype=dt)
    c.read_dev(k[..., 1:1 + Hk * qk].unflatten(-1, (Hk, qk)), v.unflatten(-1, (Hk, vd)), i32(pos), rows=i32(rows))
    torch.cuda.synchronize()
    assert (k[..., 0] == 9).all() and (k[..., 1 + Hk * qk:] == 9).all()
    k, v = k[..., 1:1 + Hk * qk].unflatten(-1, (Hk, qk)), v.unflatten(-1, (Hk, vd))
    for b in range(B):
        live = [i for i in range(rows[b]) if 0 <= pos[b] + i < cap]
        rest = [i for i in range(t) if i not in live]
        assert (k[b, rest] == 9).all() and (v[b, rest] == 9).all()
        if live:
            want = cache_rows(c, b, np.array([pos[b] + i for i in live]))
            for x, y in zip((k, v), want):
                y = torch.from_numpy(y.astype(np.float32)).to(dt)  # the product in float32, then rounded once
                assert torch.equal(x[b, live].cpu(), y)


def test_read_bad_pages():
    import torch

    c = make_cache(gen(3), "e4m3", 2, 3, 16, 2, 32, 32)
    c.pages[0, 1], c.pages[1, 0] = -7, c.k.shape[0]
    k, v = torch.full((2, 48, 2, 32), 9.0, device="cuda"), torch.full((2, 48, 2, 32), 9.0, device="cuda")
    c.read_dev(k, v, i32([0, 0]))
    for x in (k, v):
        assert (x[0, 16:32] == 9).all() and (x[1, :16] == 9).all() and (x[0, :16] != 9).any() and (x[1, 16:] != 9).any()


@pytest.mark.parametrize("io", FLOATS)
@pytest.mark.parametrize("name", CODES)
@pytest.mark.parametrize("H,Hk,qk,vd,R", [(8, 2, 48, 64, 16), (4, 4, 64, 64, 1), (32, 4, 128, 128, 64), (3, 1, 256, 240, 8),
                                          (12, 1, 64, 64, 256), (5, 5, 80, 96, 2)])
@pytest.mark.parametrize("nk", [1, 17, 200, 3100])
def test_attend(name, io, H, Hk, qk, vd, R, nk):
    import torch

    B = 4
    g = gen(nk + H)
    c = make_cache(g, name, B, -(-nk // R), R, Hk, qk, vd)
    q = torch.randn(B, H, qk, generator=g, device="cuda").to(getattr(torch, io))
    out = torch.full((B, H, vd), 3.0, device="cuda", dtype=q.dtype)
    third = nk // 3
    spans = [[0, 0, 0, nk], [0, third, min(nk, third + 2), nk], [0, 0, nk - 1, nk], [0, 0, 0, 0]]
    acc = torch.zeros(B, Hk, nk, device="cuda")
    c.attend_dev(out, q, i32(spans), nk, math.sqrt(qk), acc_out=acc)
    torch.cuda.synchronize()
    ho, hq, ha = host(out).astype(np.float64), host(q), host(acc).astype(np.float64)
    for b, (l0, h0, l1, h1) in enumerate(spans):
        rows = np.concatenate([np.arange(l0, h0), np.arange(l1, h1)])
        k, v = cache_rows(c, b, rows) if len(rows) else (np.zeros((0, Hk, qk)), np.zeros((0, Hk, vd)))
        for h in range(0, H, max(1, H // 4)):
            o, bound, _, _ = attend64(hq[b, h], k[:, h // (H // Hk)], v[:, h // (H // Hk)], math.sqrt(qk), q.dtype)
            assert (np.abs(ho[b, h] - o) <= bound).all(), (b, h)
        for z in range(Hk):
            w = np.zeros(len(rows))
            tol = np.zeros(len(rows))
            for h in range(z * (H // Hk), (z + 1) * (H // Hk)):
                _, _, x, e = attend64(hq[b, h], k[:, z], v[:, z], math.sqrt(qk), q.dtype)
                w, tol = w + x, tol + e
            assert (np.abs(ha[b, z, rows] - w) <= tol + len(rows) * 2.0 ** -24 + (H // Hk) * 2.0 ** -23).all()


@pytest.mark.parametrize("name", CODES)
def test_attend_past_the_last_row(name):
    # what lies behind the spans, NaN codes and scales among it, is not seen
    import torch

    g = gen(21)
    for H, Hk in ((1, 1), (2, 1), (4, 2), (24, 2)):
        c = make_cache(g, name, 2, 4, 16, Hk, 64, 64)
        q = torch.randn(2, H, 64, generator=g, device="cuda")
        out, spans = [torch.zeros(2, H, 64, device="cuda") for _ in range(2)], i32([[0, 0, 0, 37], [0, 0, 0, 20]])
        c.attend_dev(out[0], q, spans, 64, 8.0)
        for b, n in ((0, 37), (1, 20)):
            for x in (c.k, c.v):
                pg = c.pages[b].long()
                rest = x[pg[n // 16]].float()
                rest[n % 16:] = math.nan if name == "e4m3" else -128
                x[pg[n // 16]] = rest.to(x.dtype)
            for s in (c.ks, c.vs):
                s[c.pages[b, n // 16 + 1:].long()] = math.nan
        c.attend_dev(out[1], q, spans, 64, 8.0)
        assert torch.equal(out[0], out[1]) and out[0].isfinite().all()


def test_eviction_is_refused():
    import torch

    c = make_cache(gen(1), "e4m3", 2, 4, 16, 2, 64, 64, 8)
    acc, out = torch.zeros(2, 2, 64, device="cuda"), torch.zeros(2, 2, 32, device="cuda")
    with pytest.raises(CQDeviceError, match="scale a page"):
        c.evict_dev(i32([[8, 9], [10, 11]]), acc, out, i32([60, 60]), i32([0, 0]), torch.zeros(2, 2, 32, dtype=torch.int32, device="cuda"), 64)
