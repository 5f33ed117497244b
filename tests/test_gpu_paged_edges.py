"""Ends of the ranges of the paged caches' calls: no keys, infinite keys, pools
past 2^32 bytes, evictions of very long lists."""

import numpy as np
import pytest

from go_whistle_amd import needle
from serve_ref import attend64, host, keep_rows, make_pool, pool_rows

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
