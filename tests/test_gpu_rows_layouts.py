"""needle.qk_norm_rope_dev on rows whose streams lie between each other, and on
streams padded by part of a row, against its float64 form."""

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
