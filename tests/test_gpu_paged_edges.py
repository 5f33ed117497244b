"""Ends of the ranges of the paged caches' calls: no keys, infinite keys, pools
past 2^32 bytes, evictions of very long lists."""

import numpy as np
import pytest

from go_whistle_amd import needle
from oracle import binding as orc
from serve_ref import attend64, host, keep_rows, make_pool, pool_rows
from test_gpu_paged_cache import random_weights, run_evict, tied_weights

pytestmark = pytest.mark.gpu


def gen(seed):
    import torch

    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def i32(x):
    import torch

    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("group", [1, 3, 20, 40])
@pytest.mark.parametrize("name", ["float32", "bfloat16", "i8"])
def test_no_keys_with_weights(group, name):
    import torch

    k, v, ks, vs = make_pool(gen(1), 4, 16, 2, 64, 64, name)
    c = needle.PagedKV(k, v, i32([[0, 1], [2, 3]]), ks, vs)
    q = torch.randn(2, 2 * group, 64, generator=gen(2), device="cuda")
    out, acc = torch.full_like(q, 3.0), torch.full((2, 2, 5), 7.0, device="cuda")
    c.attend_dev(out, q, torch.zeros(2, 4, dtype=torch.int32, device="cuda"), 0, 8.0, acc_out=acc)
    torch.cuda.synchronize()
    assert (out == 0).all() and (acc == 7).all()


FORMS = [(1, 1, 1), (2, 2, 1), (300, 1, 1), (1, 6, 2), (3, 16, 1), (64, 16, 2), (2, 20, 1), (140, 4, 1)]


@pytest.mark.parametrize("name", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("io", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("B,H,Hk", FORMS)
@pytest.mark.parametrize("nk", [20, 500])
def test_infinite_keys_have_the_logits_of_float32(name, io, B, H, Hk, nk):
    # -inf where the query's coordinate is negative: a weight of 0, as the
    # type's largest value gives, whatever the form the sizes choose. Queries
    # whose coordinate takes one, two and three bfloat16 parts.
    import torch

    g, R, per = gen(nk + B), 16, -(-nk // 16)
    for qk, vd in ((48, 64), (128, 128), (256, 144)):
        k, v, _, _ = make_pool(g, B * per, R, Hk, qk, vd, name)
        pages = torch.arange(B * per, device="cuda", dtype=torch.int32).view(B, per)
        q = torch.randn(B, H, qk, generator=g, device="cuda")
        q[..., 3] = torch.tensor([-1.0, -1.0 - 2.0 ** -9, -1.0 - 2.0 ** -20], device="cuda")[torch.arange(H, device="cuda") % 3]
        q = q.to(getattr(torch, io))
        spans, outs = i32([[0, nk, nk, nk]] * B), []
        for x in (torch.finfo(k.dtype).max, float("inf")):
            k.view(B, per * R, Hk, qk)[:, [0, nk // 2, nk - 1], :, 3] = x
            outs.append(torch.empty(B, H, vd, device="cuda", dtype=q.dtype))
            acc = torch.empty(B, Hk, nk, device="cuda")
            needle.PagedKV(k, v, pages).attend_dev(outs[-1], q, spans, nk, 2.0, acc_out=acc)
            outs.append(acc)
        torch.cuda.synchronize()
        assert torch.isfinite(outs[0]).all() and (outs[1][..., nk // 2] == 0).all()
        assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3])


@pytest.mark.parametrize("name", ["float32", "float16", "bfloat16", "i8"])
@pytest.mark.parametrize("B,H,Hk", FORMS)
@pytest.mark.parametrize("bits", [0x7f800001, 0x7fc00000, 0xff80ffff - (1 << 32), 0x7fffffff])
def test_a_nan_in_a_query(name, B, H, Hk, bits):
    # whatever its bits, its head is NaN and the others are as without it
    import torch

    g, nk, R = gen(B), 40, 16
    k, v, ks, vs = make_pool(g, 3 * B, R, Hk, 80, 64, name)
    k[..., 17] = -1  # a query of infinity there would find no key above -inf
    c = needle.PagedKV(k, v, torch.arange(3 * B, device="cuda", dtype=torch.int32).view(B, 3), ks, vs)
    q, outs = torch.randn(B, H, 80, generator=g, device="cuda"), []
    for i in range(2):
        if i:
            q.view(torch.int32)[B - 1, H - 1, 17] = bits
        outs.append(torch.empty(B, H, 64, device="cuda"))
        c.attend_dev(outs[-1], q, i32([[0, nk, nk, nk]] * B), nk, 8.0)
    torch.cuda.synchronize()
    assert torch.isnan(outs[1][B - 1, H - 1]).all()
    outs[0][B - 1, H - 1] = outs[1][B - 1, H - 1] = 0
    assert torch.equal(outs[0], outs[1])


def test_a_table_of_more_rows_than_an_int():
    # 2^20 entries of pages of 4096 rows: by default all of them may be appended to
    import torch

    k, v, _, _ = make_pool(gen(5), 3, 4096, 1, 16, 16, "float16")
    k.zero_(), v.zero_()
    pages = torch.zeros(1, 1 << 20, dtype=torch.int32, device="cuda")
    pages[0, 1], pages[0, (1 << 19) - 1] = 2, 1
    c = needle.PagedKV(k, v, pages)
    one = torch.ones(1, 1, 1, 16, device="cuda")
    c.append_dev(one, one, i32([4099]))
    c.append_dev(2 * one, 2 * one, i32([(1 << 31) - 2]))
    torch.cuda.synchronize()
    assert (k[2, 3] == 1).all() and (v[1, 4094] == 2).all() and k.count_nonzero() == 32 and v.count_nonzero() == 32


def test_sizes_past_an_int_are_refused():
    import torch

    from go_whistle_amd._lib import CQPanic

    far = 1 << 32
    k, v, _, _ = make_pool(gen(6), 4, 16, 2, 64, 64, "float32")
    c = needle.PagedKV(k, v, i32([[0, 1]]))
    q, spans, out = torch.ones(1, 2, 64, device="cuda"), i32([[0, 0, 0, 3]]), torch.full((1, 2, 64), 3.0, device="cuda")
    for nk in (far + 5, far, -far + 5, 1 << 31):
        with pytest.raises(CQPanic):
            c.attend_dev(out, q, spans, nk, 8.0)
        with pytest.raises(CQPanic):
            c.append_dev(q.view(1, 1, 2, 64), q.view(1, 1, 2, 64), i32([0]), cap=nk)
    acc, kept = torch.zeros(1, 2, 32, device="cuda"), torch.full((1, 2, 8), 7, dtype=torch.int32, device="cuda")
    for more in (dict(sink=far), dict(recent=far + 1), dict(nk_max=far + 3), dict(sink=-far)):
        with pytest.raises(CQPanic):
            c.evict_dev(i32([[2, 3]]), acc, acc.clone(), i32([20]), i32([0]), kept, **{"nk_max": 20, **more})
    rows = torch.ones(1, 1, 2, 64, device="cuda")
    many = rows.expand(1, far + 3, 2, 64)
    with pytest.raises(CQPanic):
        needle.cross_attend_dev(out.view(1, 1, 2, 64), rows, many, many, 8.0)
    with pytest.raises(CQPanic):
        needle.cross_attend_dev(many, many, rows, rows, 8.0)
    ent = torch.full((1,), 3.0, device="cuda")
    with pytest.raises(CQPanic):
        needle.logprobs_dev(torch.empty(1, far + 8, dtype=torch.float16, device="cuda"), ent=ent)
    torch.cuda.synchronize()
    assert (out == 3).all() and (ent == 3).all() and (kept == 7).all()


@pytest.mark.parametrize("weights", [random_weights, tied_weights])
@pytest.mark.parametrize("nk,keep,sink,recent", [(32768, 8192, 4, 100), (32769, 1, 0, 0), (33000, 32999, 16, 512),
                                                 (65537, 16385, 0, 64), (70001, 60000, 1, 1)])
def test_evict_very_long_lists(nk, keep, sink, recent, weights):
    # past 32,768 rows the keys are not held in registers; beside lists of every shorter kind
    run_evict(nk, "float16", 5, 1, 16, 32, 16, nk, keep, sink, recent, [nk, nk - 1, 900, nk // 3, nk + 1], weights)


# ---- arrays past 2^32 bytes --------------------------------------------------------


def far_pool(g, name, Hk, qk, vd, R):
    """Pools whose last pages lie past 2^32 bytes (int8: elements too) of the
    narrower array, with 24 pages there, at the start and in between filled."""
    import torch

    size = {"float32": 4, "i8": 1}.get(name, 2)
    pages = (1 << 32) // (Hk * min(qk, vd) * size * R) + 40
    dt = torch.int8 if name == "i8" else getattr(torch, name)
    k, v = (torch.zeros(pages, R, Hk, w, dtype=dt, device="cuda") for w in (qk, vd))
    ks = vs = None
    if name == "i8":
        ks, vs = (torch.zeros(pages, R, Hk, device="cuda") for _ in range(2))
    used = [0, 1, 2, 3, pages // 2, pages // 2 + 1, pages // 3, pages // 4] + list(range(pages - 16, pages))
    at = torch.tensor(used, device="cuda")
    for x, y in zip((k, v, ks, vs), make_pool(g, len(used), R, Hk, qk, vd, name)):
        if x is not None:
            x[at] = y
    return k, v, ks, vs, used


@pytest.mark.parametrize("name", ["float32", "float16", "bfloat16", "i8"])
@pytest.mark.parametrize("H,B", [(8, 1), (8, 2), (48, 2)])
def test_attend_pools_past_32_bits(name, H, B):
    import torch

    g, Hk, qk, vd, R = gen(41), 8, 128, 144, 64
    k, v, ks, vs, used = far_pool(g, name, Hk, qk, vd, R)
    order = np.random.default_rng(B).permutation(len(used))[:8 * B].reshape(B, 8)
    pages = np.array(used)[order]
    nk = 8 * R - 5
    q, out = torch.randn(B, H, qk, generator=g, device="cuda"), torch.empty(B, H, vd, device="cuda")
    acc = torch.empty(B, Hk, nk, device="cuda")
    needle.PagedKV(k, v, i32(pages.tolist()), ks, vs).attend_dev(out, q, i32([[3, 40, 41, nk]] * B), nk, 8.0, acc_out=acc)
    torch.cuda.synchronize()
    near = torch.tensor(used, device="cuda")
    hk, hv, hks, hvs = (None if x is None else host(x[near]) for x in (k, v, ks, vs))
    rows = np.concatenate([np.arange(3, 40), np.arange(41, nk)])
    ho, ha, hq, group = host(out), host(acc), host(q), H // Hk
    for b in range(B):
        kk, vv = pool_rows(hk, hks, order[b], rows, R), pool_rows(hv, hvs, order[b], rows, R)
        for h in range(Hk):
            want, slack = np.zeros(len(rows)), np.zeros(len(rows))
            for i in range(group):
                o, bound, w, wb = attend64(hq[b, h * group + i], kk[:, h], vv[:, h], 8.0, torch.float32)
                assert (np.abs(ho[b, h * group + i] - o) <= bound).all(), (b, h, i)
                want, slack = want + w, slack + wb
            assert (np.abs(ha[b, h, rows] - want) <= slack + group * 2.0 ** -24 * want).all(), (b, h)


@pytest.mark.parametrize("name", ["float32", "float16", "bfloat16", "i8"])
def test_append_and_evict_past_32_bits(name):
    import torch

    g, Hk, qk, vd, R = gen(43), 8, 128, 144, 64
    k, v, ks, vs, used = far_pool(g, name, Hk, qk, vd, R)
    src, dst = i32([used[-4:], [used[5], used[1], used[-5], used[0]]]), i32([used[-8:-5], [used[3], used[-9], used[4]]])
    c = needle.PagedKV(k, v, src, ks, vs)
    # rows appended at the end of the first stream and inside the second, far apart themselves
    wide = torch.zeros((1 << 31) + 9000, dtype=torch.float16, device="cuda")
    new = [wide.as_strided((2, 1, Hk, w), ((1 << 31) + 16, Hk * w, w, 1)) for w in (qk, vd)]
    wide[:2048], wide[1 << 31:] = torch.randn(2048, generator=g, device="cuda"), torch.randn(9000, generator=g, device="cuda")
    c.append_dev(new[0], new[1], i32([4 * R - 1, 2 * R + 5]))
    torch.cuda.synchronize()
    for b, at in ((0, (used[-1], R - 1)), (1, (used[-5], 5))):
        for x, s, y in ((k, ks, new[0]), (v, vs, new[1])):
            row = y[b, 0].float()
            if name == "i8":
                codes, scales = orc.quantize_rows(row.cpu().numpy().ravel(), row.numel(), row.shape[-1])
                assert torch.equal(x[at].cpu(), torch.from_numpy(codes.reshape(row.shape)))
                assert torch.equal(s[at].cpu(), torch.from_numpy(scales))
            else:
                assert torch.equal(x[at], row.to(x.dtype))
    # both streams cut to 150 rows, into pages at either end
    nk, keep = 4 * R, 150
    acc = torch.rand(2, Hk, nk, generator=g, device="cuda")
    out, kept = torch.empty(2, Hk, keep, device="cuda"), torch.empty(2, Hk, keep, dtype=torch.int32, device="cuda")
    ln = i32([nk, nk - 3])
    before = [None if x is None else x[src.long()].clone() for x in (k, v, ks, vs)]  # [2, 4, R, Hk, ...]
    c.evict_dev(dst, acc, out, ln, ln, kept, nk, sink=4, recent=30)
    torch.cuda.synchronize()
    assert ln.tolist() == [keep, keep]
    ha = acc.cpu().numpy()
    for b in range(2):
        for h in range(Hk):
            rows = torch.from_numpy(keep_rows(ha[b, h], nk - 3 * b, keep, 4, 30)).cuda()
            assert torch.equal(kept[b, h].long(), rows) and torch.equal(out[b, h], acc[b, h, rows])
            for x, y in zip((k, v, ks, vs), before):
                if x is not None:
                    got = x[dst[b].long()].flatten(0, 1)[:keep, h]
                    assert torch.equal(got, y[b].flatten(0, 1)[rows, h]), (b, h)


@pytest.mark.parametrize("name", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("t", [1, 3, 130])
def test_cross_attention_past_32_bits(name, t):
    # rows of a memory, memories, streams of queries and outputs: each far apart
    import torch

    g, dt, F, Hk, H, D, B = gen(t), getattr(torch, name), 40, 2, 4, 64, 60
    row, size = 1 << 26, 1 << 31  # elements
    buf = torch.zeros(size + 41 * row, dtype=dt, device="cuda")
    k, v = (buf[off:].as_strided((2, F, Hk, D), (size + 1024, row, D, 1)) for off in (0, 4096))
    near = [torch.randn(2, F, Hk, D, generator=g, device="cuda").to(dt) for _ in range(2)]
    k.copy_(near[0]), v.copy_(near[1])
    q = buf[8192:].as_strided((B, t, H, D), (row, H * D, D, 1))
    q.copy_(torch.randn(q.shape, generator=g, device="cuda"))
    out = buf[1 << 20:].as_strided((B, t, H, D), (row, H * D, D, 1))
    index = i32([b % 2 for b in range(B)])
    needle.cross_attend_dev(out, q, k, v, 8.0, index=index)
    torch.cuda.synchronize()
    ho, hq, hk, hv = (host(x) for x in (out, q, *near))
    for b in (0, 1, 31, 32, 33, B - 2, B - 1):
        for i in {0, t // 2, t - 1}:
            for h in range(H):
                o, bound, w, _ = attend64(hq[b, i, h], hk[b % 2, :, h // 2], hv[b % 2, :, h // 2], 8.0, dt,
                                          None if name == "float32" else dt)
                assert (np.abs(ho[b, i, h] - o) <= bound).all(), (b, i, h)


@pytest.mark.parametrize("name", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n", [1000, 60001])
def test_log_probabilities_past_32_bits(name, n):
    import torch

    g, dt, far = gen(n), getattr(torch, name), (1 << 31) + 3
    logits = torch.zeros(2 * far + n, dtype=dt, device="cuda").as_strided((3, n), (far, 1))
    near = torch.randn(3, n, generator=g, device="cuda").to(dt)
    logits.copy_(near)
    tokens = i32([5, n - 1, 0])
    outs = []
    for x in (logits, near):
        lp, ent, tl = torch.empty(3, device="cuda"), torch.empty(3, device="cuda"), torch.empty(3, 4, device="cuda")
        top = torch.empty(3, 4, dtype=torch.int32, device="cuda")
        needle.logprobs_dev(x, tokens, lp, ent, top, tl)
        outs.append((lp, ent, top, tl))
    torch.cuda.synchronize()
    want = torch.log_softmax(near.double(), -1)
    best = near.double().sort(dim=-1, descending=True, stable=True).indices[:, :4]
    assert torch.equal(outs[0][2].long(), best)
    # float32 sums of n terms: n u of the sum, a few roundings of logits up to 5 and a logarithm of 7 to 12
    slack = (n + 64) * 2.0 ** -24
    assert (outs[0][0].double() - want.gather(1, tokens.long().view(3, 1)).view(3)).abs().max() <= slack
    assert (outs[0][3].double() - want.gather(1, best)).abs().max() <= slack
    assert (outs[0][1].double() + (want.exp() * want).sum(-1)).abs().max() <= 16 * slack


def test_the_tensors_of_a_cache_stay():
    # the calls hold their addresses: another table or pool is another PagedKV, not an attribute
    import torch

    k, v, ks, vs = make_pool(gen(8), 4, 16, 2, 64, 64, "i8")
    c = needle.PagedKV(k, v, i32([[0, 1]]), ks, vs)
    assert c.k is k and c.v is v and c.ks is ks and c.vs is vs
    for name in ("k", "v", "ks", "vs", "pages"):
        with pytest.raises(AttributeError):
            setattr(c, name, torch.zeros_like(getattr(c, name)))
    q, outs = torch.randn(1, 2, 64, generator=gen(9), device="cuda"), []
    for change in (None, lambda: c.pages.copy_(i32([[3, 2]]))):  # an entry that changes is seen
        if change:
            change()
        outs.append(torch.empty_like(q))
        c.attend_dev(outs[-1], q, i32([[0, 0, 0, 20]]), 20, 8.0)
    other = torch.empty_like(q)
    needle.PagedKV(k, v, i32([[3, 2]]), ks, vs).attend_dev(other, q, i32([[0, 0, 0, 20]]), 20, 8.0)
    torch.cuda.synchronize()
    assert torch.equal(outs[1], other) and not torch.equal(outs[0], other)
