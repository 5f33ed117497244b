"""Attention over values near float32's largest, with logits that rise by less
than what a running maximum may lag behind them: the outputs, means of finite values,
are finite and within their bounds (tests/serve_ref.py, tests/page8_ref.py)."""

import math

import numpy as np
import pytest

from go_whistle_amd import needle
from page8_ref import MOST, cache_rows, check_rows, gen, i32
from serve_ref import attend64, host

pytestmark = pytest.mark.gpu

BIG = 3e36  # 2^7.9 of it is past float32's largest, 15 are not


def lifted(n, far=100, every=97):
    """Logits of n keys in units of log2: 0, and 7.9 at some keys behind the first tiles."""
    j = np.arange(n)
    return np.where((j >= far) & (j % every == 3), 7.9, 0.0)


def large_cache(g, name, streams, n, R, Hk, qk, vd):
    """A paged cache whose keys' logits are lifted(n) for queries of ones and the scale
    log2(e) / 16 (a key's first 16 values are its logit / 256), values of either sign near BIG."""
    import torch

    per = -(-n // R)
    lg = torch.zeros(streams, per * R, device="cuda")
    lg[:, :n] = torch.tensor(lifted(n), device="cuda")
    k = torch.zeros(streams * per, R, Hk, qk, device="cuda")
    k[..., :16] = (lg / 256).view(-1, R, 1, 1)
    v = BIG * (0.5 + 0.5 * torch.rand(streams * per, R, Hk, vd, generator=g, device="cuda"))
    sign = torch.where(torch.rand(v.shape, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    v[..., :vd // 2] *= sign[0, 0, 0, :vd // 2]  # of one sign for all keys, and of either
    v[..., vd // 2:] *= sign[..., vd // 2:]
    table = torch.randperm(streams * per, generator=g, device="cuda")
    back = torch.empty_like(table)
    back[table] = torch.arange(len(table), device="cuda")
    k, v = k[back], v[back]
    pages = table.view(streams, per).int().contiguous()
    if name == "i8":  # a scale a row
        ks, vs = (torch.full((streams * per, R, Hk), top / 127, device="cuda") for top in (7.9 / 256, BIG))
        return needle.PagedKV((k / ks[..., None]).round().to(torch.int8), (v / vs[..., None]).round().to(torch.int8), pages, ks, vs)
    if name in MOST:
        ks, vs = (torch.full((streams * per, Hk), top / MOST[name], device="cuda") for top in (7.9 / 256, BIG))
        k, v = k / ks[:, None, :, None], v / vs[:, None, :, None]
        k, v = (x.round().to(torch.int8) if name == "i8p" else x.to(torch.float8_e4m3fn) for x in (k, v))
        return needle.PagedKV(k, v, pages, ks, vs)
    return needle.PagedKV(k.to(getattr(torch, name)), v.to(getattr(torch, name)), pages)


SCALE = math.log2(math.e) / 16


@pytest.mark.parametrize("io,name", [("bfloat16", "bfloat16"), ("float32", "float32"), ("float32", "bfloat16"), ("bfloat16", "i8p"),
                                     ("bfloat16", "e4m3"), ("float32", "i8p"), ("float32", "e4m3"), ("bfloat16", "float32"),
                                     ("bfloat16", "i8"), ("float32", "i8")])
@pytest.mark.parametrize("B,t,pos,H,Hk,w", [
    (1, 4, 1000, 8, 2, 64),       # parts of the keys
    (64, 3, 600, 8, 8, 64),       # many lists
    (4, 6, 1500, 16, 4, 128),
    (2, 1, 900, 64, 2, 64),       # one row of many heads
    (1, 300, 700, 4, 2, 64),      # tiles, their keys in halves or in parts
    (64, 150, 400, 8, 8, 64),     # whole tiles
    (16, 200, 300, 8, 4, 240),
])
def test_many_rows(io, name, B, t, pos, H, Hk, w):
    import torch

    g = gen(t)
    c = large_cache(g, name, B, pos + t, 16, Hk, w, w)
    q = torch.ones(B, t, H, w, device="cuda", dtype=getattr(torch, io))
    out = torch.zeros_like(q)
    c.attend_rows_dev(out, q, i32([pos] * B), SCALE)
    assert out.isfinite().all()
    check_rows(c, name, out, out, q, [pos] * B, None, c.cap, 0, 0, SCALE, 2)


@pytest.mark.parametrize("io", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["i8p", "e4m3", "i8", "bfloat16", "float32"])
@pytest.mark.parametrize("B,n,H,Hk,w", [(1, 3000, 8, 1, 64), (64, 900, 16, 2, 128), (4, 2000, 64, 2, 64), (3, 700, 3, 1, 256)])
@pytest.mark.parametrize("weights", [False, True])
def test_one_token(io, name, B, n, H, Hk, w, weights):
    import torch

    c = large_cache(gen(n), name, B, n, 16, Hk, w, w)
    q = torch.ones(B, H, w, device="cuda", dtype=getattr(torch, io))
    out = torch.zeros_like(q)
    acc = torch.zeros(B, Hk, c.cap, device="cuda")
    c.attend_dev(out, q, i32([[0, 0, 0, n]] * B), c.cap, SCALE, acc_out=acc if weights else None)
    assert out.isfinite().all()
    for b in (0, B - 1):
        k, v = cache_rows(c, b, np.arange(n))
        for h in (0, H - 1):
            g = h // (H // Hk)
            o, bound, x, xb = attend64(host(q[b, h]), k[:, g], v[:, g], SCALE, q.dtype)
            assert (np.abs(host(out[b, h]) - o) <= bound).all(), (b, h)
            if weights:  # every head of a group has the same
                assert (np.abs(host(acc[b, g, :n]) - H // Hk * x) <= H // Hk * (xb + 2.0 ** -22)).all()
