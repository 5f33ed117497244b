"""needle.qk_norm_rope_dev on rows whose streams lie between each other, and on
streams padded by part of a row, against its float64 form."""

import numpy as np
import pytest

from go_whistle_amd import needle
from page8_ref import gen, i32
from test_gpu_norm_rope import compare, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("io", ["float32", "bfloat16"])
@pytest.mark.parametrize("pad", [0, 3, 16])
@pytest.mark.parametrize("order", ["rows of streams", "padded streams"])
@pytest.mark.parametrize("counts", [False, True])
def test_packed_products_of_any_order_in_place(io, pad, order, counts):
    import torch

    B, t, width, g, dt = 5, 33, (4 + 2 + 2) * 64, gen(pad + 1), getattr(torch, io)
    if order == "rows of streams":
        room = torch.randn(t * B * width + pad, generator=g, device="cuda").to(dt)
        strides = (width, B * width)
    else:
        room = torch.randn(B * (t * width + pad + 24), generator=g, device="cuda").to(dt)
        strides = (t * width + pad + 24, width)
    old = room.clone()

    def heads(x, first, n):
        return x.as_strided((B, t, n, 64), (*strides, 64, 1), first)

    q, k = heads(room, 0, 4), heads(room, 256, 2)
    qg, kg = torch.rand(64, generator=g, device="cuda"), torch.rand(64, generator=g, device="cuda")
    cos, sin = tables(g, 64, 64)
    pos, rows = [0, 5, 31, 2, 9], [33, 0, 1, 20, -4] if counts else None
    needle.qk_norm_rope_dev(q, k, q, k, qg, kg, (cos, sin), i32(pos), rows=i32(rows) if counts else None)
    compare(q, heads(old, 0, 4), heads(old, 0, 4), qg, cos, sin, pos, rows)
    compare(k, heads(old, 256, 2), heads(old, 256, 2), kg, cos, sin, pos, rows)
    # nothing else is written
    for x in (room, old):
        heads(x, 0, 4).zero_()
        heads(x, 256, 2).zero_()
    assert torch.equal(room, old)


@pytest.mark.parametrize("io,name", [("bfloat16", "bfloat16"), ("float32", "float16"), ("float16", "e4m3")])
@pytest.mark.parametrize("t", [1, 5, 70])
@pytest.mark.parametrize("counts", [False, True])
def test_attention_beside_its_queries(io, name, t, counts):
    # queries and outputs side by side in rows of streams, and one after the other
    import torch

    from page8_ref import check_rows, make_cache

    B, g, dt = 3, gen(t), getattr(torch, io)
    c = make_cache(g, name, B, 10, 16, 2, 64, 64)
    room = torch.randn(t, B, 512 + 40, generator=g, device="cuda").to(dt)
    q, out = (room[..., x:x + 256].unflatten(-1, (4, 64)).transpose(0, 1) for x in (0, 264))
    rows, pos = [t, 0, t - 1] if counts else None, [3, 80, 31]
    before, rest, asked = out.clone(), room.clone(), q.clone()
    c.attend_rows_dev(out, q, i32(pos), 8.0, rows=i32(rows) if counts else None)
    check_rows(c, name, out, before, asked, pos, rows, c.cap, 0, 0, 8.0, 5)
    room[..., 264:520] = rest[..., 264:520]
    assert torch.equal(room, rest)


@pytest.mark.parametrize("name", ["float16", "i8", "e4m3"])
@pytest.mark.parametrize("counts", [False, True])
def test_keys_and_values_read_beside_each_other(name, counts):
    import torch

    from page8_ref import cache_rows, make_cache
    from serve_ref import host

    B, t, g = 3, 20, gen(4)
    c = make_cache(g, name, B, 5, 8, 2, 48, 64)
    room = torch.full((t, B, 2 * (48 + 64) + 3), 7.0, device="cuda")
    k, v = room[..., :96].unflatten(-1, (2, 48)).transpose(0, 1), room[..., 97:225].unflatten(-1, (2, 64)).transpose(0, 1)
    pos, rows = [0, 3, 17], [t, 0, 5] if counts else [t] * 3
    c.read_dev(k, v, i32(pos), rows=i32(rows) if counts else None)
    for b in range(B):
        wk, wv = cache_rows(c, b, np.arange(pos[b], pos[b] + rows[b]))
        # one product of float32
        assert (abs(host(k[b, :rows[b]]) - wk) <= 2.0 ** -24 * abs(wk)).all() and (abs(host(v[b, :rows[b]]) - wv) <= 2.0 ** -24 * abs(wv)).all()
        assert (k[b, rows[b]:] == 7).all() and (v[b, rows[b]:] == 7).all()
    assert (room[..., 96:97] == 7).all() and (room[..., 225:] == 7).all()
