"""Paged caches of any type (needle.PagedKV): appends, attention of one token
split over the cache's length with accumulated weights, and eviction by them,
each against its plain float64 form (tests/serve_ref.py, where the bounds are
derived) or bit for bit."""

import math

import numpy as np
import pytest

from go_whistle_amd import needle
from oracle import binding as orc
from serve_ref import attend64, half_ulp, host, keep_rows, make_pool, pool_rows, rows_of

pytestmark = pytest.mark.gpu

TYPES = ["float32", "float16", "bfloat16", "i8"]


def gen(seed):
    import torch

    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def tables(g, streams, per, pages):
    import torch

    return torch.randperm(pages, generator=g, device="cuda")[:streams * per].view(streams, per).int().contiguous()


def i32(x):
    import torch

    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ---- append -----------------------------------------------------------------------


def expect_append(pool, scales, x, pages, pos, counts, t, cap, page_rows, name):
    import torch

    pool, scales = pool.clone(), scales.clone() if scales is not None else None
    pages = pages.cpu().numpy()
    for b in range(x.shape[0]):
        n = t if counts is None else int(counts[b])
        if not 0 <= n <= t:
            continue
        for i in range(n):
            p = int(pos[b]) + i
            if not 0 <= p < cap:
                continue
            pg = int(pages[b, p // page_rows])
            if not 0 <= pg < pool.shape[0]:
                continue
            row = x[b, i].float()
            if name == "i8":
                q, s = orc.quantize_rows(row.cpu().numpy().ravel(), row.numel(), row.shape[-1])
                pool[pg, p % page_rows] = torch.from_numpy(q.reshape(row.shape)).cuda()
                scales[pg, p % page_rows] = torch.from_numpy(s).cuda()
            else:
                pool[pg, p % page_rows] = row.to(pool.dtype)
    return pool, scales


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("io", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("B,t,Hk,qk,vd,R,strided", [(1, 1, 1, 16, 16, 1, False), (5, 3, 2, 48, 64, 16, False),
                                                    (7, 1, 8, 64, 64, 16, False), (3, 37, 3, 80, 96, 8, True),
                                                    (2, 5, 2, 256, 144, 4, True)])
def test_append(name, io, B, t, Hk, qk, vd, R, strided):
    import torch

    g = gen(B * 100 + t)
    cap = 61
    per = -(-cap // R)
    k, v, ks, vs = make_pool(g, B * per + 2, R, Hk, qk, vd, name)
    pages = tables(g, B, per, B * per + 2)
    if B > 2:
        pages[2, 0] = -1  # a bad entry: its rows are skipped
        pages[2, -1] = B * per + 2
    dt = getattr(torch, io)
    if strided:  # rows inside wider ones, starting at an odd element
        kx = torch.randn(B, t + 2, Hk * qk + 7, generator=g, device="cuda").to(dt)[:, 1:t + 1, 3:3 + Hk * qk].unflatten(2, (Hk, qk))
        vx = torch.randn(B, t + 1, Hk * vd + 5, generator=g, device="cuda").to(dt)[:, 1:, 5:].unflatten(2, (Hk, vd))
    else:
        kx = torch.randn(B, t, Hk, qk, generator=g, device="cuda").to(dt)
        vx = torch.randn(B, t, Hk, vd, generator=g, device="cuda").to(dt)
    if t > 2:
        kx[0, 1, 0] = 0  # a zero row: scale 1
        vx[0, 2, -1, 3] = float("inf")
    pos = [0, cap - 1, 5, -1, -2 ** 31, 2 ** 31 - 1, 17][:B]
    counts = [t, t, t, 1, t + 1, -1, 0][:B] if t > 1 else None
    acc = torch.ones(B, Hk, cap + 3, device="cuda")
    want = [expect_append(p, s, x, pages, pos, counts, t, cap, R, name) for p, s, x in ((k, ks, kx), (v, vs, vx))]
    needle.PagedKV(k, v, pages, ks, vs).append_dev(kx, vx, i32(pos), rows=None if counts is None else i32(counts),
                                                   cap=cap, acc=acc)
    torch.cuda.synchronize()
    for got, gs, (w, ws) in ((k, ks, want[0]), (v, vs, want[1])):
        assert torch.equal(torch.nan_to_num(got.float()), torch.nan_to_num(w.float()))
        assert gs is None or torch.equal(torch.nan_to_num(gs), torch.nan_to_num(ws))
    a = acc.cpu().numpy()
    for b in range(B):
        n = t if counts is None else counts[b]
        live = [pos[b] + i for i in range(n if 0 <= n <= t else 0) if 0 <= pos[b] + i < cap]
        live = [p for p in live if 0 <= int(pages[b, p // R]) < B * per + 2]
        want_a = np.ones((Hk, cap + 3), np.float32)
        want_a[:, live] = 0
        assert np.array_equal(a[b], want_a), b


# ---- attention ---------------------------------------------------------------------


def check_attend(k, v, ks, vs, pages, q, spans, nk, scale, out, acc, acc_out, before_out, before_acc, R, skip=()):
    H, Hk = q.shape[1], k.shape[2]
    G = H // Hk
    hk, hv = host(k), host(v)
    hks, hvs = (host(s) if s is not None else None for s in (ks, vs))
    pg, sp, hq, ho = pages.cpu().numpy(), spans.cpu().numpy(), host(q), host(out).astype(np.float64)
    for b in range(q.shape[0]):
        if b in skip:
            assert np.array_equal(ho[b], host(before_out)[b].astype(np.float64), equal_nan=True)
            if acc_out is not None:
                assert np.array_equal(host(acc_out)[b], host(before_acc)[b])
            continue
        rows = rows_of(sp[b])
        kk, vv = pool_rows(hk, hks, pg[b], rows, R), pool_rows(hv, hvs, pg[b], rows, R)
        for h in range(Hk):
            wsum, wb = np.zeros(len(rows)), np.zeros(len(rows))
            for gi in range(G):
                o, bound, w, dw = attend64(hq[b, h * G + gi], kk[:, h], vv[:, h], scale, out.dtype)
                err = np.abs(ho[b, h * G + gi] - o)
                assert (err <= bound).all(), (b, h, gi, (err / np.maximum(bound, 1e-300)).max())
                wsum += w
                wb += dw
            if acc_out is not None:
                want = host(before_acc)[b, h].astype(np.float64)
                base = host(acc)[b, h].astype(np.float64) if acc is not None else np.zeros_like(want)
                want[rows] = base[rows] + wsum
                tol = np.zeros_like(want)
                tol[rows] = wb + 2.0 ** -23 * (np.abs(want[rows]) + G)
                assert (np.abs(host(acc_out)[b, h] - want) <= tol).all(), (b, h)


def run_attend(seed, name, io, B, H, Hk, qk, vd, R, nk, spans, with_acc, acc_null=False, bad_page=False):
    import torch

    g = gen(seed)
    per = max(1, -(-nk // R))
    k, v, ks, vs = make_pool(g, B * per + 1, R, Hk, qk, vd, name)
    pages = tables(g, B, per, B * per + 1)
    if bad_page:
        pages[0, 0], pages[0, -1] = -5, B * per + 1
    q = (torch.randn(B, H, qk, generator=g, device="cuda") * 2).to(getattr(torch, io))
    out = torch.full((B, H, vd), 7.0, device="cuda", dtype=q.dtype)
    spans = i32(spans)
    acc = acc_out = None
    if with_acc:
        acc = None if acc_null else torch.rand(B, Hk, nk + 3, generator=g, device="cuda")
        acc_out = torch.full((B, Hk, nk + 3), 3.0, device="cuda")
    b_out, b_acc = out.clone(), acc_out.clone() if with_acc else None
    scale = math.sqrt(qk)
    needle.PagedKV(k, v, pages, ks, vs).attend_dev(out, q, spans, nk, scale, acc=acc, acc_out=acc_out)
    torch.cuda.synchronize()
    sp = spans.cpu().numpy()
    ok = lambda s: (0 <= s[0] <= s[1] <= nk and 0 <= s[2] <= s[3] <= nk and  # noqa: E731
                    (s[1] <= s[2] or s[0] == s[1] or s[2] == s[3]))
    check_attend(k, v, ks, vs, pages, q, spans, nk, scale, out, acc, acc_out, b_out, b_acc, R,
                 skip=[b for b in range(B) if not ok(sp[b])])


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("io", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("H,Hk,qk,vd", [(8, 2, 48, 64), (4, 4, 16, 16), (6, 2, 128, 80), (40, 2, 64, 128), (2, 1, 256, 240)])
def test_attend_types_and_heads(name, io, H, Hk, qk, vd):
    nk = 75
    run_attend(H + qk, name, io, 4, H, Hk, qk, vd, 16, nk, [[0, 0, 0, nk], [0, 0, 0, 0], [0, 3, 40, 70], [2, 3, 3, 4]], True)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("B,H,Hk", [(1, 6, 2), (1, 10, 2), (2, 16, 1), (90, 3, 1), (140, 4, 1), (300, 4, 1)])
def test_attend_groups_without_weights(name, B, H, Hk):
    # odd groups, and as many streams as take two columns a workgroup, or sixteen
    run_attend(B + H, name, "float32", B, H, Hk, 48, 64, 16, 70, [[0, b % 5, 5, 5 + (7 * b) % 66] for b in range(B)], False)


@pytest.mark.parametrize("nk", [1, 2, 15, 16, 17, 31, 32, 33, 64, 65, 127, 128, 129, 257, 1500])
@pytest.mark.parametrize("name", ["float32", "bfloat16", "i8"])
def test_attend_lengths(nk, name):
    # one stream: split; its list ends at every place in a tile
    run_attend(nk, name, "float32", 1, 8, 2, 64, 64, 16, nk, [[0, 0, 0, nk]], True, acc_null=True)


@pytest.mark.parametrize("R", [1, 2, 4, 64, 512])
@pytest.mark.parametrize("name", ["float16", "i8"])
def test_attend_page_sizes_and_bad_pages(R, name):
    run_attend(R, name, "float32", 3, 4, 2, 48, 64, R, 203, [[0, 0, 0, 203], [0, 4, 99, 203], [7, 9, 9, 150]], True,
               bad_page=True)


def test_attend_refused_spans_leave_their_streams():
    nk = 60
    spans = [[0, 0, 0, 61], [-1, 2, 3, 4], [0, 5, 3, 20], [5, 3, 6, 9], [0, 0, 20, 10], [0, 0, 0, 60], [50, 60, 0, 10],
             [0, 60, 0, 0]]
    run_attend(5, "bfloat16", "float32", 8, 4, 2, 64, 64, 16, nk, spans, True)
    run_attend(5, "i8", "bfloat16", 8, 4, 2, 64, 64, 16, nk, spans, False)


def test_attend_many_streams_one_launch():
    # more workgroups than the chip holds: no split
    nk = 100
    g = np.random.default_rng(3)
    run_attend(9, "i8", "float32", 300, 2, 2, 64, 64, 16, nk, [[0, 0, 0, int(g.integers(0, nk + 1))] for _ in range(300)], False)


def test_attend_masked_rows_may_hold_anything():
    # infinities and NaN outside the spans, and scales of them, change nothing
    import torch

    g = gen(11)
    nk, R, B, Hk, D = 130, 16, 2, 2, 64
    per = -(-nk // R)
    for name in TYPES:
        k, v, ks, vs = make_pool(g, B * per, R, Hk, D, D, name)
        pages = torch.arange(B * per, device="cuda", dtype=torch.int32).view(B, per).contiguous()
        q = torch.randn(B, 4, D, generator=g, device="cuda")
        spans = i32([[0, 5, 37, 101], [0, 0, 64, 65]])
        out = torch.empty(B, 4, D, device="cuda")
        c = needle.PagedKV(k, v, pages, ks, vs)
        c.attend_dev(out, q, spans, nk, 8.0)
        want = out.clone()
        for b in range(B):
            live = torch.zeros(per * R, dtype=torch.bool, device="cuda")
            live[torch.from_numpy(rows_of(spans[b].tolist())).cuda()] = True
            dead = ~live.view(per, R)
            for x, s in ((k, ks), (v, vs)):
                if s is None:
                    x[b * per:(b + 1) * per][dead] = float("nan")
                else:
                    s[b * per:(b + 1) * per][dead] = float("inf")
        c.attend_dev(out, q, spans, nk, 8.0)
        torch.cuda.synchronize()
        assert torch.equal(out, want), name


def test_attend_extreme_logits():
    # a key of -inf logits alone, and logits that differ by more than float32's exponent range
    import torch

    B, R, D = 1, 16, 64
    k = torch.zeros(3, R, 1, D, device="cuda")
    v = torch.randn(3, R, 1, D, device="cuda", generator=gen(2))
    pages = i32([[0, 1, 2]])
    q = torch.zeros(B, 1, D, device="cuda")
    q[..., 0] = 1.0
    k[:, :, 0, 0] = -float("inf")
    out = torch.full((B, 1, D), 5.0, device="cuda")
    c = needle.PagedKV(k, v, pages)
    c.attend_dev(out, q, i32([[0, 0, 0, 40]]), 48, 1.0)
    torch.cuda.synchronize()
    assert (out == 0).all()  # no weight anywhere
    k[:, :, 0, 0] = -1e30
    k[1, 3, 0, 0] = 1e30
    c.attend_dev(out, q, i32([[0, 0, 0, 40]]), 48, 1.0)
    torch.cuda.synchronize()
    assert torch.equal(out[0, 0], v[1, 3, 0])
    k[2, 1, 0, 0] = float("nan")
    c.attend_dev(out, q, i32([[0, 0, 0, 40]]), 48, 1.0)
    torch.cuda.synchronize()
    assert torch.isnan(out).all()


def test_attend_long_cache_past_32_bits():
    # a pool of more than 2^32 bytes, rows at its far end
    import torch

    Hk, D, R = 8, 128, 256
    pages_n = (1 << 32) // (Hk * D * 2 * R) + 40
    k = torch.empty(pages_n, R, Hk, D, dtype=torch.bfloat16, device="cuda")
    v = torch.empty(pages_n, R, Hk, D, dtype=torch.bfloat16, device="cuda")
    g = gen(21)
    nk = 5 * R - 3
    pages = i32([[pages_n - 1, 0, pages_n - 7, pages_n - 2, 3]])
    for p in pages[0].tolist():
        k[p] = torch.randn(R, Hk, D, generator=g, device="cuda").bfloat16()
        v[p] = torch.randn(R, Hk, D, generator=g, device="cuda").bfloat16()
    q = torch.randn(1, 16, D, generator=g, device="cuda").bfloat16()
    out = torch.empty(1, 16, D, dtype=torch.bfloat16, device="cuda")
    sub = pages[0].long()
    needle.PagedKV(k, v, pages).attend_dev(out, q, i32([[0, 0, 0, nk]]), nk, math.sqrt(D))
    new = torch.randn(1, 1, Hk, D, generator=g, device="cuda").bfloat16()
    needle.PagedKV(k, v, pages).append_dev(new, new, i32([2 * R + 9]))
    torch.cuda.synchronize()
    assert torch.equal(k[pages_n - 7, 9], new[0, 0]) and torch.equal(v[pages_n - 7, 9], new[0, 0])
    ident = torch.arange(5, device="cuda", dtype=torch.int32).view(1, 5)
    k2, v2 = k[sub].contiguous(), v[sub].contiguous()
    del k, v
    # the appended row was not there yet: take the rows as they were
    want = torch.empty_like(out)
    k2[2, 9], v2[2, 9] = 0, 0
    got_sub = torch.empty_like(out)
    needle.PagedKV(k2, v2, ident).attend_dev(got_sub, q, i32([[0, 2 * R + 9, 2 * R + 10, nk]]), nk, math.sqrt(D))
    needle.PagedKV(k2, v2, ident).attend_dev(want, q, i32([[0, 2 * R + 9, 2 * R + 10, nk]]), nk, math.sqrt(D))
    assert torch.equal(got_sub, want)
    # one of 1277 keys aside, the two agree within its weight
    assert (out.float() - want.float()).abs().max() < 0.5


def test_attend_same_result_every_time_and_on_two_streams():
    import torch

    g = gen(31)
    nk, R, Hk, D = 900, 16, 2, 64
    per = -(-nk // R)
    k, v, _, _ = make_pool(g, per, R, Hk, D, D, "float16")
    c = needle.PagedKV(k, v, tables(g, 1, per, per))
    qs = [torch.randn(1, 8, D, generator=g, device="cuda") for _ in range(2)]
    spans = i32([[0, 0, 0, nk]])
    want = []
    for q in qs:
        o = torch.empty(1, 8, D, device="cuda")
        c.attend_dev(o, q, spans, nk, 8.0)
        torch.cuda.synchronize()
        want.append(o)
    outs = [[torch.empty(1, 8, D, device="cuda") for _ in range(20)] for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(20):
        for z in range(2):
            with torch.cuda.stream(streams[z]):
                c.attend_dev(outs[z][i], qs[z], spans, nk, 8.0)
    torch.cuda.synchronize()
    for z in range(2):
        assert all(torch.equal(o, want[z]) for o in outs[z])


# ---- eviction ----------------------------------------------------------------------


def run_evict(seed, name, B, Hk, qk, vd, R, nk, keep, sink, recent, lens, weights):
    import torch

    g = gen(seed)
    per, dper = max(1, -(-nk // R)), max(1, -(-keep // R))
    pages_n = B * (per + dper)
    k, v, ks, vs = make_pool(g, pages_n, R, Hk, qk, vd, name)
    perm = torch.randperm(pages_n, generator=g, device="cuda").int()
    pages, dst = perm[:B * per].view(B, per).contiguous(), perm[B * per:].view(B, dper).contiguous()
    acc = weights(g, (B, Hk, nk + 2))
    acc_out = torch.full((B, Hk, keep + 1), 9.0, device="cuda")
    kept = torch.full((B, Hk, keep), 77, dtype=torch.int32, device="cuda")
    ln, ln_out = i32(lens), torch.full((B,), -3, dtype=torch.int32, device="cuda")
    pools = [x for x in (k, v, ks, vs) if x is not None]
    before = [x.clone() for x in pools]
    needle.PagedKV(k, v, pages, ks, vs).evict_dev(dst, acc, acc_out, ln, ln_out, kept, nk, sink=sink, recent=recent)
    torch.cuda.synchronize()
    ha = acc.cpu().numpy()
    hp, hd = pages.cpu().numpy(), dst.cpu().numpy()
    want_pools = [x.clone() for x in before]
    for b in range(B):
        n = lens[b]
        if not 0 <= n <= nk:
            assert int(ln_out[b]) == -3 and (kept[b] == 77).all() and (acc_out[b] == 9).all()
            continue
        assert int(ln_out[b]) == min(n, keep)
        for h in range(Hk):
            rows = keep_rows(ha[b, h], n, keep, sink, recent)
            want = np.full(keep, -1)
            want[:len(rows)] = rows
            assert np.array_equal(kept[b, h].cpu().numpy(), want), (b, h)
            wa = np.full(keep + 1, 9.0, np.float32)
            wa[:len(rows)] = ha[b, h, rows]
            assert np.array_equal(acc_out[b, h].cpu().numpy(), wa, equal_nan=True)
            i = np.arange(len(rows))
            src = (torch.from_numpy(hp[b][rows // R].astype(np.int64)), torch.from_numpy(rows % R))
            to = (torch.from_numpy(hd[b][i // R].astype(np.int64)), torch.from_numpy(i % R))
            for x, w in zip(before, want_pools):
                w[to[0], to[1], h] = x[src[0], src[1], h]
    for got, w in zip(pools, want_pools):
        assert torch.equal(got, w)


def random_weights(g, shape):
    import torch

    return torch.rand(shape, generator=g, device="cuda")


def tied_weights(g, shape):
    import torch

    return torch.randint(0, 3, shape, generator=g, device="cuda").float() * torch.where(
        torch.rand(shape, generator=g, device="cuda") < 0.5, -1.0, 1.0)  # with -0 beside 0


def odd_weights(g, shape):
    import torch

    x = torch.randn(shape, generator=g, device="cuda")
    x[..., 1::7] = float("nan")
    x[..., 2::7] = float("inf")
    x[..., 3::7] = -float("inf")
    x[..., 4::7] = 1e-42
    return x


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("qk,vd,Hk", [(48, 64, 2), (16, 256, 1), (128, 128, 3)])
def test_evict_types(name, qk, vd, Hk):
    run_evict(qk, name, 4, Hk, qk, vd, 16, 100, 37, 3, 9, [100, 37, 0, 64], random_weights)


@pytest.mark.parametrize("weights", [random_weights, tied_weights, odd_weights])
@pytest.mark.parametrize("nk,keep,sink,recent,R", [(1, 1, 0, 0, 1), (5, 0, 0, 0, 4), (50, 1, 0, 1, 8), (50, 1, 1, 0, 8),
                                                   (300, 299, 4, 64, 16), (1025, 500, 250, 250, 64),
                                                   (2500, 1024, 0, 0, 16), (9000, 2047, 16, 100, 64)])
def test_evict_choices(weights, nk, keep, sink, recent, R):
    run_evict(nk, "float16", 5, 2, 16, 32, R, nk, keep, sink, recent, [nk, nk + 1, -1, nk // 2, max(0, nk - 1)], weights)


def test_evict_of_forked_streams_and_bad_pages():
    # two streams that share their source pages are cut apart; a source page outside the pool reads page 0, a
    # destination page outside it is skipped
    import torch

    g = gen(51)
    R, nk, keep, Hk, D = 8, 40, 16, 2, 32
    k, v, ks, vs = make_pool(g, 16, R, Hk, D, D, "i8")
    pages = i32([[1, 2, 3, 4, 5], [1, 2, 3, 4, 5], [6, -1, 99, 7, 8]])
    dst = i32([[9, 10], [11, 12], [13, 16]])
    acc = torch.rand(3, Hk, nk, generator=g, device="cuda")
    acc_out = torch.zeros(3, Hk, keep, device="cuda")
    kept = torch.zeros(3, Hk, keep, dtype=torch.int32, device="cuda")
    n = i32([40, 33, 40])
    before = [x.clone() for x in (k, v, ks, vs)]
    needle.PagedKV(k, v, pages, ks, vs).evict_dev(dst, acc, acc_out, n, n, kept, nk, sink=1, recent=2)
    torch.cuda.synchronize()
    assert n.tolist() == [16, 16, 16]
    want = [x.clone() for x in before]
    for b, length in enumerate((40, 33, 40)):
        for h in range(Hk):
            rows = keep_rows(acc[b, h].cpu().numpy(), length, keep, 1, 2)
            assert kept[b, h].tolist() == rows.tolist()
            for i, j in enumerate(rows):
                sp, dp = int(pages[b, j // R]), int(dst[b, i // R])
                sp = sp if 0 <= sp < 16 else 0
                if 0 <= dp < 16:
                    for x, w in zip(before, want):
                        w[dp, i % R, h] = x[sp, j % R, h]
    for x, w in zip((k, v, ks, vs), want):
        assert torch.equal(x, w)


def test_c_strides_of_queries_and_outputs():
    # rows of wider arrays through the C entry, at an odd element
    import torch

    from go_whistle_amd._lib import check as ok
    from go_whistle_amd._lib import lib

    g = gen(61)
    B, H, Hk, D, R, nk = 3, 4, 2, 64, 16, 50
    for dt, code in ((torch.float32, 0), (torch.bfloat16, 2)):
        k, v, _, _ = make_pool(g, B * 4, R, Hk, D, D, "float16")
        c = needle.PagedKV(k, v, tables(g, B, 4, B * 4))
        wide = torch.randn(B, H * D + 9, generator=g, device="cuda").to(dt)
        out = torch.full((B, H * D + 3), 2.0, device="cuda", dtype=dt)
        spans = i32([[0, 0, 0, nk], [0, 7, 20, 31], [0, 0, 0, 0]])
        ok(lib().kv_attend_paged_dev(c._ref, out.data_ptr() + dt.itemsize, H * D + 3, wide.data_ptr() + 5 * dt.itemsize,
                                     H * D + 9, code, B, H, spans.data_ptr(), nk, 8.0, None, None, 0,
                                     torch.cuda.current_stream().cuda_stream))
        torch.cuda.synchronize()
        q, o = wide[:, 5:5 + H * D].reshape(B, H, D), out[:, 1:1 + H * D].reshape(B, H, D)
        check_attend(k, v, None, None, c.pages, q, spans, nk, 8.0, o, None, None, o, None, R)
        assert (out[:, 0] == 2).all() and (out[:, 1 + H * D:] == 2).all()


@pytest.mark.parametrize("name", TYPES)
def test_no_keys_and_no_streams(name):
    import torch

    g = gen(71)
    k, v, ks, vs = make_pool(g, 2, 4, 1, 16, 32, name)
    q, out = torch.randn(2, 3, 16, device="cuda"), torch.full((2, 3, 32), 4.0, device="cuda")
    none = needle.PagedKV(k, v, torch.zeros(2, 0, dtype=torch.int32, device="cuda"), ks, vs)
    acc = torch.zeros(2, 1, 0, device="cuda")
    none.attend_dev(out, q, torch.zeros(2, 4, dtype=torch.int32, device="cuda"), 0, 4.0, acc_out=acc)
    none.append_dev(torch.zeros(2, 1, 1, 16, device="cuda"), torch.zeros(2, 1, 1, 32, device="cuda"), i32([0, 0]))
    torch.cuda.synchronize()
    assert (out == 0).all()
    empty = needle.PagedKV(k, v, torch.zeros(0, 1, dtype=torch.int32, device="cuda"), ks, vs)
    e = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t, device="cuda")  # noqa: E731
    i = lambda *s: e(*s, t=torch.int32)  # noqa: E731
    empty.attend_dev(e(0, 3, 32), e(0, 3, 16), i(0, 4), 4, 4.0)
    empty.append_dev(e(0, 1, 1, 16), e(0, 1, 1, 32), i(0))
    empty.evict_dev(i(0, 1), e(0, 1, 4), e(0, 1, 2), i(0), i(0), i(0, 1, 2), 4)


def test_two_graphs_replayed_on_two_streams():
    # each graph's partials in its own workspace, with eager calls of the same size beside them
    import torch

    g = gen(81)
    nk, R, Hk, D = 5000, 16, 1, 64
    per = -(-nk // R)
    k, v, _, _ = make_pool(g, per, R, Hk, D, D, "bfloat16")
    c = needle.PagedKV(k, v, tables(g, 1, per, per))
    qs = [torch.randn(1, 6, D, generator=g, device="cuda") for _ in range(3)]
    spans = i32([[0, 0, 0, nk]])
    acc = torch.rand(1, Hk, nk, generator=g, device="cuda")

    def outs():
        return torch.zeros(1, 6, D, device="cuda"), torch.zeros(1, Hk, nk, device="cuda")

    want = []
    for q in qs:
        o, a = outs()
        c.attend_dev(o, q, spans, nk, 8.0, acc=acc, acc_out=a)
        torch.cuda.synchronize()
        want.append((o, a))
    got, graphs = [outs() for _ in range(3)], []
    for z in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            c.attend_dev(got[z][0], qs[z], spans, nk, 8.0, acc=acc, acc_out=got[z][1])
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for r in range(4):
        for o, a in got:
            o.zero_(), a.zero_()
        torch.cuda.synchronize()
        for z in range(2):
            with torch.cuda.stream(streams[z]):
                graphs[z].replay()
        with torch.cuda.stream(streams[2]):
            c.attend_dev(got[2][0], qs[2], spans, nk, 8.0, acc=acc, acc_out=got[2][1])
        torch.cuda.synchronize()
        for z in range(3):
            assert torch.equal(got[z][0], want[z][0]) and torch.equal(got[z][1], want[z][1]), (r, z)


# ---- a run of them together ----------------------------------------------------------


@pytest.mark.parametrize("name", TYPES)
def test_decode_with_a_bounded_cache(name):
    # prompt, steps with accumulated weights, an eviction, steps on the cut
    # cache, captured into a graph and replayed between eager work; a second
    # stream's fork shares its pages
    import torch

    g = gen(41)
    B, H, Hk, qk, vd, R, cap, keep = 3, 4, 2, 48, 64, 16, 96, 40
    per, dper = cap // R, cap // R
    k, v, ks, vs = make_pool(g, B * (per + dper), R, Hk, qk, vd, name)
    ids = torch.arange(B * (per + dper), device="cuda", dtype=torch.int32)
    pages, dst = ids[:B * per].view(B, per).clone(), ids[B * per:].view(B, dper).clone()
    c = needle.PagedKV(k, v, pages, ks, vs)
    acc = torch.full((B, Hk, cap), 5.0, device="cuda")
    prompt = [20, 0, 64]
    n = i32(prompt)
    kx, vx = (torch.randn(B, 64, Hk, w, generator=g, device="cuda") for w in (qk, vd))
    c.append_dev(kx, vx, i32([0, 0, 0]), rows=n, acc=acc)
    sp = torch.zeros(B, 4, dtype=torch.int32, device="cuda")
    steps = 12
    kq, vq, qq = (torch.randn(steps, B, z, w, generator=g, device="cuda") for z, w in ((Hk, qk), (Hk, vd), (H, qk)))
    out = torch.zeros(B, H, vd, device="cuda")
    scale = math.sqrt(qk)

    def step(i, cache, weights):
        cache.append_dev(kq[i].unsqueeze(1), vq[i].unsqueeze(1), n, acc=weights)
        sp[:, 3] = n + 1
        before = weights.clone()
        cache.attend_dev(out, qq[i], sp, cap, scale, acc=weights, acc_out=weights)
        torch.cuda.synchronize()
        check_attend(k, v, ks, vs, cache.pages, qq[i], sp, cap, scale, out, before, weights, out, before, R)
        n.add_(1)

    for i in range(6):
        step(i, c, acc)
    kept = torch.zeros(B, Hk, keep, dtype=torch.int32, device="cuda")
    acc2 = torch.zeros(B, Hk, cap, device="cuda")
    lens = n.tolist()
    c.evict_dev(dst, acc, acc2, n, n, kept, cap, sink=2, recent=8)
    torch.cuda.synchronize()
    assert n.tolist() == [min(x, keep) for x in lens]
    for b in range(B):
        for h in range(Hk):
            rows = keep_rows(acc[b, h].cpu().numpy(), lens[b], keep, 2, 8)
            assert kept[b, h, :len(rows)].tolist() == rows.tolist()
            assert torch.equal(acc2[b, h, :len(rows)], acc[b, h, torch.from_numpy(rows).cuda()])
    cut = needle.PagedKV(k, v, dst, ks, vs)
    for i in range(6, 9):
        step(i, cut, acc2)
    # the rest of the steps from a graph, replayed between eager calls
    i_dev = torch.zeros((), dtype=torch.int64, device="cuda")
    s_out = torch.zeros_like(out)
    kb, vb, qb = kq[9].clone(), vq[9].clone(), qq[9].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cut.append_dev(kb.unsqueeze(1), vb.unsqueeze(1), n, acc=acc2)
        sp[:, 3] = n + 1
        cut.attend_dev(s_out, qb, sp, cap, scale, acc=acc2, acc_out=acc2)
        n.add_(1)
    del i_dev
    for i in range(9, steps):
        kb.copy_(kq[i]), vb.copy_(vq[i]), qb.copy_(qq[i])
        before = acc2.clone()
        lens = n.tolist()
        graph.replay()
        c.attend_dev(out, qq[0], sp, cap, scale)  # an eager call of the same workspaces' kind behind it
        torch.cuda.synchronize()
        for b in range(B):
            before[b, :, lens[b]] = 0  # the append's
        check_attend(k, v, ks, vs, dst, qq[i], sp, cap, scale, s_out, before, acc2, s_out, before, R)
    assert half_ulp(torch.float32) == 2.0 ** -24


@pytest.mark.parametrize("name", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("B,H,Hk", [(1, 2, 2), (2, 16, 1), (140, 4, 1), (3, 3, 1)])
@pytest.mark.parametrize("nk", [1, 13, 47, 300])
def test_attend_an_infinite_value_of_the_last_key(name, B, H, Hk, nk):
    # its weight is above 0, so its coordinate is the infinity; the others are as without it
    import torch

    g = gen(nk)
    R, per = 16, -(-nk // 16)
    for qk, vd in ((48, 64), (128, 128), (256, 144)):
        k, v, ks, vs = make_pool(g, B * per, R, Hk, qk, vd, name)
        pages = torch.arange(B * per, device="cuda", dtype=torch.int32).view(B, per)
        q = torch.randn(B, H, qk, generator=g, device="cuda")
        spans = i32([[0, nk, nk, nk]] * B)
        outs = []
        for x in (1.0, float("inf")):
            v.view(B, per * R, Hk, vd)[:, nk - 1, :, 5] = x
            outs.append(torch.empty(B, H, vd, device="cuda"))
            needle.PagedKV(k, v, pages).attend_dev(outs[-1], q, spans, nk, math.sqrt(qk))
        torch.cuda.synchronize()
        assert (outs[1][..., 5] == float("inf")).all()
        for o in outs:
            o[..., 5] = 0
        assert torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("nk,keep", [(1, 3), (64, 70), (63, 1), (65, 64), (1023, 100), (1024, 102), (1024, 103), (447, 0)])
def test_evict_small_lists_in_one_launch(name, nk, keep):
    # heads of 64 and 96: float32 rows of 40 pieces, 102 of them at most in one launch
    sink = min(2, keep)
    run_evict(nk, name, 3, 2, 64, 96, 16, nk, keep, sink, min(7, keep - sink), [nk, nk // 2, nk + 1], random_weights)


@pytest.mark.parametrize("name", TYPES)
def test_evict_over_the_old_lengths_is_the_same(name):
    import torch

    g = gen(61)
    B, Hk, D, R, nk, keep = 33, 3, 64, 16, 200, 60
    k, v, ks, vs = make_pool(g, B * 17, R, Hk, D, D, name)
    perm = torch.randperm(B * 17, generator=g, device="cuda").int()
    pages, dst = perm[:B * 13].view(B, 13).contiguous(), perm[B * 13:].view(B, 4).contiguous()
    acc = random_weights(g, (B, Hk, nk))
    lens = torch.randint(-1, nk + 2, (B,), generator=g, device="cuda").int()
    got = []
    for over in (False, True):
        pools = [x.clone() if x is not None else None for x in (k, v, ks, vs)]
        n = lens.clone()
        n_out = n if over else lens.clone()
        kept, out = torch.full((B, Hk, keep), 5, dtype=torch.int32, device="cuda"), torch.zeros(B, Hk, keep, device="cuda")
        c = needle.PagedKV(pools[0], pools[1], pages, pools[2], pools[3])
        c.evict_dev(dst, acc, out, n, n_out, kept, nk, sink=1, recent=5)
        torch.cuda.synchronize()
        got.append([x for x in (*pools, n_out, kept, out) if x is not None])
    assert all(torch.equal(x, y) for x, y in zip(*got))
