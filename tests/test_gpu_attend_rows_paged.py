"""PagedKV.attend_rows_dev: causal attention of many rows over paged caches of
any type, with a window and first rows, against its float64 form (bounds in
tests/serve_ref.py and tests/page8_ref.py)."""

import math

import numpy as np
import pytest

from go_whistle_amd import needle
from page8_ref import CACHES, FLOATS, cache_rows, check_rows, gen, i32, make_cache, visible, weight_error
from serve_ref import attend64, half_ulp, host

pytestmark = pytest.mark.gpu


def run(seed, io, name, H, Hk, qk, vd, R, pos, t, rows=None, window=0, sink=0, nk_max=None, sample=4, per=None):
    import torch

    B = len(pos)
    g = gen(seed)
    per = per or max(1, -(-(max(pos) + t) // R))
    c = make_cache(g, name, B, per, R, Hk, qk, vd)
    q = torch.randn(B, t, H, qk, generator=g, device="cuda").to(getattr(torch, io))
    out = torch.full((B, t, H, vd), 3.0, device="cuda", dtype=q.dtype)
    before, scale = out.clone(), math.sqrt(qk)
    c.attend_rows_dev(out, q, i32(pos), scale, rows=None if rows is None else i32(rows), nk_max=nk_max, window=window, sink=sink)
    torch.cuda.synchronize()
    check_rows(c, name, out, before, q, pos, rows, c.cap if nk_max is None else nk_max, window, sink, scale, sample, seed)
    return c, q, out


HEADS = [(8, 2, 48, 64), (4, 4, 64, 64), (8, 2, 128, 128), (3, 1, 256, 256), (5, 5, 80, 96), (6, 2, 16, 240), (2, 1, 112, 128)]


@pytest.mark.parametrize("io", FLOATS)
@pytest.mark.parametrize("name", CACHES)
@pytest.mark.parametrize("H,Hk,qk,vd", HEADS)
@pytest.mark.parametrize("t", [1, 3, 70])
def test_heads(io, name, H, Hk, qk, vd, t):
    run(t + H, io, name, H, Hk, qk, vd, 16, [0, 130, 61], t)
    run(t + H + 1, io, name, H, Hk, qk, vd, 4, [0, 130, 61], t, window=37, sink=5)


@pytest.mark.parametrize("io,name", [("bfloat16", "bfloat16"), ("float16", "e4m3"), ("bfloat16", "i8p"), ("float32", "float32"),
                                     ("float32", "i8")])
@pytest.mark.parametrize("pos,t", [(0, 1), (1, 1), (63, 1), (64, 2), (0, 64), (0, 65), (62, 3), (31, 33), (127, 130), (500, 257),
                                   (0, 300)])
def test_lengths(io, name, pos, t):
    for R in (1, 16, 128):
        run(pos * 5 + t, io, name, 4, 2, 64, 64, R, [pos, 0], t)


@pytest.mark.parametrize("io,name", [("float16", "float16"), ("bfloat16", "e4m3"), ("float32", "bfloat16")])
@pytest.mark.parametrize("window,sink", [(1, 0), (1, 1), (2, 64), (63, 3), (64, 65), (65, 0), (100, 100), (1000, 4), (7, 1000),
                                         (200, 128), (2 ** 31 - 1, 2 ** 31 - 1)])
def test_windows(io, name, window, sink):
    run(window % 1000 + sink % 1000, io, name, 4, 2, 64, 64, 16, [0, 300, 511], 140, window=window, sink=sink)
    run(window % 1000 + sink % 1000, io, name, 4, 1, 128, 128, 64, [700], 5, window=window, sink=sink)


@pytest.mark.parametrize("io", FLOATS)
@pytest.mark.parametrize("name", ["float32", "bfloat16", "i8p"])
def test_ragged_and_padded(io, name):
    # counts of zero, below it and past t, positions outside the cache, rows that pass nk_max
    pos, rows = [0, 5, 100, -1, 250, 236, 20, 7], [64, 0, 1, 5, 20, 20, -3, 65]
    run(4, io, name, 6, 2, 48, 64, 8, pos, 64, rows=rows, nk_max=256, per=40, sample=6)
    run(5, io, name, 4, 4, 128, 128, 8, pos, 64, rows=rows, nk_max=256, per=40, window=30, sink=2, sample=6)


@pytest.mark.parametrize("io,name", [("bfloat16", "bfloat16"), ("float16", "i8p"), ("float32", "float16"), ("float32", "e4m3")])
@pytest.mark.parametrize("t", [1, 4, 16])
def test_few_rows_over_long_caches(io, name, t):
    # in parts of the keys; with a window the parts of which some are not seen
    run(t, io, name, 8, 2, 64, 64, 64, [20000, 3, 9999], t, sample=2)
    run(t, io, name, 4, 1, 128, 128, 16, [6000], t, window=3000, sink=300, sample=2)
    run(t, io, name, 4, 1, 128, 128, 16, [6000, 100], t, window=2, sink=0, sample=2)


@pytest.mark.parametrize("io,name", [("bfloat16", "bfloat16"), ("float16", "float16"), ("float16", "i8p"), ("bfloat16", "e4m3"),
                                     ("float32", "float32")])
@pytest.mark.parametrize("H,Hk,w", [(8, 8, 64), (8, 8, 48), (4, 2, 128), (4, 4, 96)])
def test_many_streams(io, name, H, Hk, w):
    # many short lists, full and narrower heads
    run(H, io, name, H, Hk, w, w, 16, [(b * 37) % 200 for b in range(48)], 150, rows=[150 - b % 9 * 16 for b in range(48)], sample=1)


@pytest.mark.parametrize("io,name", [("bfloat16", "bfloat16"), ("float16", "float16"), ("float16", "i8p"), ("bfloat16", "e4m3")])
@pytest.mark.parametrize("H,Hk,w,t", [(8, 8, 64, 150), (8, 8, 48, 150), (16, 8, 128, 100), (8, 8, 112, 130), (8, 8, 256, 100),
                                      (8, 8, 240, 70)])
def test_workgroups_of_whole_tiles(io, name, H, Hk, w, t):
    # so many lists that no workgroup takes a tile's keys in halves
    pos = [(b * 37) % 200 for b in range(64)]
    run(t, io, name, H, Hk, w, w, 16, pos, t, sample=1)
    run(w, io, name, H, Hk, w, w, 8, pos, t, rows=[t - b % 5 * 16 for b in range(64)], window=70, sink=5, sample=1)


@pytest.mark.parametrize("io,name", [("bfloat16", "bfloat16"), ("float16", "float16"), ("bfloat16", "e4m3")])
@pytest.mark.parametrize("Hk,w", [(8, 64), (8, 128), (8, 240)])
def test_whole_tiles_with_values_that_are_not_finite(io, name, Hk, w):
    # the value of row pos[b] is seen by the first 40 rows alone
    import torch

    g, t, window, B = gen(w), 150, 40, 64
    pos = [(b * 37) % 200 for b in range(B)]
    c = make_cache(g, name, B, -(-(max(pos) + t) // 16), 16, Hk, w, w)
    for b in range(B):
        poison(c, b, pos[b], math.nan, keys=False)
    q = torch.randn(B, t, Hk, w, generator=g, device="cuda").to(getattr(torch, io))
    out = torch.zeros_like(q)
    c.attend_rows_dev(out, q, i32(pos), math.sqrt(w), window=window)
    assert out[:, :window].isnan().all() and not out[:, window:].isnan().any()
    rest = out[:, window:]
    check_rows(c, name, rest, rest, q[:, window:], [p + window for p in pos], None, c.cap, window, 0, math.sqrt(w), 1, 3)


@pytest.mark.parametrize("io,name", [("bfloat16", "bfloat16"), ("float16", "i8p"), ("float32", "float32")])
@pytest.mark.parametrize("B,Hk", [(1, 1), (5, 1), (70, 1), (3, 2), (5, 3), (5, 4), (2, 8), (3, 16), (40, 4)])
def test_ragged_streams_of_any_number_of_heads(io, name, B, Hk):
    # every tile of every stream has its workgroup, in whichever order they go over the chip
    pos = [(b * 53) % 150 for b in range(B)]
    for group, t in ((1, 170), (3, 75)):
        run(B + Hk, io, name, group * Hk, Hk, 64, 64, 16, pos, t, rows=[t] + [(t * b * 7) % (t + 1) for b in range(1, B)], sample=3)


@pytest.mark.parametrize("io,name", [("bfloat16", "bfloat16"), ("float32", "float16"), ("float16", "e4m3")])
def test_strided_and_unaligned(io, name):
    import torch

    g, dt = gen(8), getattr(torch, io)
    c = make_cache(g, name, 2, 10, 16, 2, 64, 64)
    for off, pad in ((0, 8), (1, 3), (2, 6)):
        whole = torch.randn(2, 70, off + 4 * 64 + pad, generator=g, device="cuda").to(dt)
        q = whole[..., off:off + 256].unflatten(-1, (4, 64))
        room = torch.full((2, 70, off + 4 * 64 + pad), 3.0, device="cuda", dtype=dt)
        out = room[..., off:off + 256].unflatten(-1, (4, 64))
        before = out.clone()
        c.attend_rows_dev(out, q, i32([3, 80]), 8.0)
        torch.cuda.synchronize()
        assert (room[..., :off] == 3).all() and (room[..., off + 256:] == 3).all()
        check_rows(c, name, out, before, q, [3, 80], None, c.cap, 0, 0, 8.0, 5)


@pytest.mark.parametrize("io,name", [("bfloat16", "bfloat16"), ("float32", "float16"), ("float16", "e4m3")])
@pytest.mark.parametrize("t", [1, 3, 40])
def test_one_query_for_all(io, name, t):
    # a query of one stream, of one row, or of one of both, expanded: strides of 0
    import torch

    c = make_cache(gen(t), name, 3, 8, 16, 2, 64, 64)
    for shape in ((1, t), (3, 1), (1, 1)):
        q = torch.randn(*shape, 4, 64, generator=gen(2), device="cuda").to(getattr(torch, io)).expand(3, t, 4, 64)
        out, want = torch.zeros(3, t, 4, 64, device="cuda", dtype=q.dtype), torch.zeros(3, t, 4, 64, device="cuda", dtype=q.dtype)
        c.attend_rows_dev(out, q, i32([0, 30, 60]), 8.0)
        c.attend_rows_dev(want, q.contiguous(), i32([0, 30, 60]), 8.0)
        assert torch.equal(out, want) and out.count_nonzero() > 0


def test_queries_that_are_not_numbers():
    # NaN rows are NaN, and the others within the bounds of what they are without them
    import torch

    for io, name, t in (("bfloat16", "bfloat16", 200), ("float32", "float16", 6), ("float16", "e4m3", 100), ("float32", "float32", 600)):
        c = make_cache(gen(t), name, 2, 60, 16, 2, 64, 64)
        q = torch.randn(2, t, 4, 64, generator=gen(3), device="cuda").to(getattr(torch, io))
        out, bad = torch.zeros_like(q), torch.zeros_like(q)
        c.attend_rows_dev(out, q, i32([0, 90]), 8.0)
        some = q.clone()
        some[0, 3, 1, 7], some[1, t - 1, 0] = math.nan, math.nan
        c.attend_rows_dev(bad, some, i32([0, 90]), 8.0)
        assert bad[0, 3, 1].isnan().all() and bad[1, t - 1, 0].isnan().all()
        bad[0, 3, 1], bad[1, t - 1, 0] = out[0, 3, 1], out[1, t - 1, 0]
        check_rows(c, name, bad, torch.zeros_like(q), q, [0, 90], None, c.cap, 0, 0, 8.0, 30)


def poison(c, b, row, what, values=True, keys=True):
    R = c.k.shape[1]
    pg = int(c.pages[b, row // R])
    for x, on in ((c.k, keys), (c.v, values)):
        if on:
            y = x[pg].float()
            y[row % R] = what
            x[pg] = y.to(x.dtype)


@pytest.mark.parametrize("io,name", [("bfloat16", "bfloat16"), ("float16", "float16"), ("float32", "float32"),
                                     ("float32", "bfloat16"), ("bfloat16", "e4m3"), ("float16", "e4m3"), ("float32", "e4m3")])
@pytest.mark.parametrize("what", [math.nan, math.inf])
@pytest.mark.parametrize("H,Hk,w,pos,t", [(4, 2, 64, 100, 90), (2, 1, 128, 3000, 6), (3, 3, 80, 0, 130)])
def test_values_that_are_not_finite(io, name, what, H, Hk, w, pos, t):
    # a row's value is seen by the rows from it on to the window's end alone, its key makes those NaN
    import torch

    if name == "e4m3":
        what = math.nan  # the type has no infinities
    g, window = gen(t), 40
    c = make_cache(g, name, 1, -(-(pos + t + 64) // 16), 16, Hk, w, w)
    q = torch.randn(1, t, H, w, generator=g, device="cuda").to(getattr(torch, io))
    args = dict(window=window, sink=3)
    bad = pos + t // 2
    poison(c, 0, bad, what, keys=False)
    poison(c, 0, pos + t, what)  # behind the last row: seen by none
    poison(c, 0, pos + t + 5, math.nan)
    hit = np.array([bad in visible(pos + i, window, 3) for i in range(t)])
    assert hit.any() and not hit.all()
    hq = host(q).astype(np.float64)
    for nan_key in (False, True):
        if nan_key:
            poison(c, 0, bad, math.nan, values=False)
        out = torch.zeros(1, t, H, w, device="cuda", dtype=q.dtype)
        c.attend_rows_dev(out, q, i32([pos]), math.sqrt(w), **args)
        ho = host(out)[0].astype(np.float64)
        seen = ho[hit]
        assert np.isnan(seen).all() if nan_key or math.isnan(what) else (seen == np.inf).all()
        for i in np.nonzero(~hit)[0]:
            j = visible(pos + i, window, 3)
            k, v = cache_rows(c, 0, j)
            for h in range(H):
                o, bound, x, _ = attend64(hq[0, i, h], k[:, h // (H // Hk)], v[:, h // (H // Hk)], math.sqrt(w), q.dtype)
                bound = bound + (1 + half_ulp(q.dtype)) * weight_error(io, name, len(j)) * (x @ np.abs(v[:, h // (H // Hk)]))
                assert (np.abs(ho[i, h] - o) <= bound).all(), (i, h)


@pytest.mark.parametrize("io,name", [("bfloat16", "bfloat16"), ("float16", "float16"), ("float32", "float32"), ("float16", "i8p")])
def test_logits_of_any_size(io, name):
    # the largest logit's weight is 1 however large it is
    import torch

    g = gen(2)
    for size in (1e-6, 30.0, 1e4, 3e8 if io != "float16" else 6e4):
        c = make_cache(g, name, 1, 10, 16, 1, 64, 64)
        q = (torch.randn(1, 66, 2, 64, generator=g, device="cuda") * size).clamp(-6e4 if io == "float16" else -1e30, 6e4 if io == "float16" else 1e30).to(getattr(torch, io))
        out = torch.zeros(1, 66, 2, 64, device="cuda", dtype=q.dtype)
        c.attend_rows_dev(out, q, i32([70]), 8.0)
        assert out.isfinite().all()
        if size >= 1e4:  # one key has all the weight
            k, v = cache_rows(c, 0, np.arange(136))
            hq, ho = host(q).astype(np.float64), host(out).astype(np.float64)
            for i in (0, 30, 65):
                lg = k[:71 + i, 0] @ hq[0, i, 0] / 8.0
                first, second = np.sort(lg)[::-1][:2]
                if first - second > 40 + 1e-6 * abs(first) * 64:
                    want = v[np.argmax(lg), 0]
                    assert np.abs(ho[0, i, 0] - want).max() <= 2.0 ** -7 * np.abs(want).max()


def test_rows_are_the_same_alone_and_together():
    # a row of a prompt, and the same row as a draft of its own: within both bounds of the same exact values
    import torch

    c, q, out = run(6, "bfloat16", "bfloat16", 4, 2, 64, 64, 16, [40], 130)
    one = torch.zeros(1, 1, 4, 64, device="cuda", dtype=q.dtype)
    before = one.clone()
    c.attend_rows_dev(one, q[:, 77:78], i32([117]), 8.0)
    check_rows(c, "bfloat16", one, before, q[:, 77:78], [117], None, c.cap, 0, 0, 8.0, 1)
    assert (one[:, 0].float() - out[:, 77].float()).abs().max() <= 2 * 2.0 ** -8 * out.abs().max()


def test_bad_pages_read_page_0():
    import torch

    g = gen(14)
    c = make_cache(g, "float16", 2, 6, 16, 2, 64, 64)
    c.pages[0, 2], c.pages[1, 0] = -1, 10 ** 7
    q = torch.randn(2, 20, 4, 64, generator=g, device="cuda").half()
    out = torch.zeros_like(q)
    c.attend_rows_dev(out, q, i32([60, 70]), 8.0)
    check_rows(c, "float16", out, torch.zeros_like(q), q, [60, 70], None, c.cap, 0, 0, 8.0, 4)


@pytest.mark.parametrize("io,name", [("bfloat16", "bfloat16"), ("bfloat16", "e4m3"), ("float32", "e4m3")])
def test_pools_past_32_bits(io, name):
    # pages that begin past 2^32 bytes of the pool
    import torch

    from go_whistle_amd import needle as nd

    g = gen(15)
    small = make_cache(g, name, 2, 4, 64, 2, 128, 128)
    pages = (1 << 32) // (64 * 2 * 128 * small.k.element_size()) + 20
    pools = []
    for x, s in ((small.k, small.ks), (small.v, small.vs)):
        big = torch.zeros(pages, *x.shape[1:], dtype=x.dtype, device="cuda")
        big[pages - 8:] = x
        if s is not None:
            sb = torch.zeros(pages, 2, device="cuda")
            sb[pages - 8:] = s
            s = sb
        pools.append((big, s))
    c = nd.PagedKV(pools[0][0], pools[1][0], small.pages + (pages - 8), pools[0][1], pools[1][1])
    q = torch.randn(2, 9, 4, 128, generator=g, device="cuda").to(getattr(torch, io))
    out, want = torch.zeros_like(q), torch.zeros_like(q)
    c.attend_rows_dev(out, q, i32([200, 100]), 11.0)
    small.attend_rows_dev(want, q, i32([200, 100]), 11.0, nk_max=c.cap)
    assert torch.equal(out, want) and want.count_nonzero() > 0
    o1, w1 = torch.zeros(2, 4, 128, device="cuda", dtype=q.dtype), torch.zeros(2, 4, 128, device="cuda", dtype=q.dtype)
    spans = i32([[0, 0, 0, 250], [0, 3, 9, 200]])
    c.attend_dev(o1, q[:, 0].contiguous(), spans, 256, 11.0)
    small.attend_dev(w1, q[:, 0].contiguous(), spans, 256, 11.0)
    assert torch.equal(o1, w1) and w1.count_nonzero() > 0
    rows = torch.randn(2, 30, 2, 128, generator=g, device="cuda")
    back = [torch.zeros_like(rows) for _ in range(4)]
    for z, x in enumerate((c, small)):
        x.append_dev(rows, rows, i32([100, 220]))
        x.read_dev(back[2 * z], back[2 * z + 1], i32([98, 215]))
    assert torch.equal(back[0], back[2]) and torch.equal(back[1], back[3]) and back[0].count_nonzero() > 0
