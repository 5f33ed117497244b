"""needle.qk_norm_rope_dev against its float64 form (bound in tests/page8_ref.py)
and, in float32, against the separate norm and rotation."""

import ctypes

import numpy as np
import pytest

from go_whistle_amd import needle
from go_whistle_amd._lib import check, lib
from page8_ref import FLOATS, gen, i32, norm_rope64
from serve_ref import half_ulp, host

pytestmark = pytest.mark.gpu


def tables(g, positions, width):
    import torch

    a = torch.rand(positions, width // 2, generator=g, device="cuda") * 6.28
    return a.cos().contiguous(), a.sin().contiguous()


def compare(out, before, x, gain, cos, sin, pos, rows):
    """Every row of [streams, t, heads, width] against float64; rows behind the count as they were."""
    import torch

    B, t, H, w = x.shape
    ho, hb, hx = (host(y).astype(np.float64) for y in (out, before, x))
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 2.0 ** -140
    for b in range(B):
        n = t if rows is None else rows[b]
        n = n if 0 <= n <= t else 0
        assert np.array_equal(ho[b, n:], hb[b, n:]), b
        if not n:
            continue
        p = (0 if pos is None else pos[b]) + np.arange(n)
        if cos is None:
            c, s, turn = np.ones((n, w // 2)), np.zeros((n, w // 2)), np.zeros(n, bool)
        else:
            turn = (p >= 0) & (p < cos.shape[0])
            at = np.clip(p, 0, cos.shape[0] - 1)
            c, s = host(cos)[at].astype(np.float64), host(sin)[at].astype(np.float64)
        y, bound = norm_rope64(hx[b, :n], None if gain is None else host(gain), c[:, None], s[:, None], turn[:, None, None])
        bound = bound + half_ulp(x.dtype) * (np.abs(y) + bound) + tiny
        assert (np.abs(ho[b, :n] - y) <= bound).all(), b


@pytest.mark.parametrize("io", FLOATS)
@pytest.mark.parametrize("H,Hk,w", [(8, 8, 64), (8, 2, 48), (16, 4, 128), (3, 1, 256), (1, 0, 16), (0, 2, 32), (5, 5, 80), (2, 3, 240),
                                    (7, 1, 96)])
@pytest.mark.parametrize("B,t", [(1, 1), (256, 1), (3, 70)])
def test_norm_and_rotation(io, H, Hk, w, B, t):
    import torch

    g, dt = gen(w + t), getattr(torch, io)
    q, k = (torch.randn(B, t, n, w, generator=g, device="cuda").to(dt) * 3 if n else None for n in (H, Hk))
    qg, kg = (1 + 0.3 * torch.randn(w, generator=g, device="cuda") for _ in range(2))
    cos, sin = tables(g, 90, w)
    pos = [(b * 7) % 95 - 2 for b in range(B)]  # some outside the tables
    for gains, rope in (((qg, kg), (cos, sin)), ((qg, None), (cos, sin)), ((None, kg), None), ((None, None), (cos, sin))):
        outs = [None if x is None else torch.full_like(x, 5.0) for x in (q, k)]
        before = [None if x is None else x.clone() for x in outs]
        needle.qk_norm_rope_dev(outs[0], outs[1], q, k, gains[0], gains[1], rope, i32(pos))
        for x, y, z, gain in zip((q, k), outs, before, gains):
            if x is not None:
                compare(y, z, x, gain, *(rope or (None, None)), pos, None)


@pytest.mark.parametrize("io", FLOATS)
def test_packed_in_place_and_ragged(io):
    import torch

    g, dt = gen(5), getattr(torch, io)
    rows, pos = [33, 0, 1, -4, 34, 20], [0, 5, 63, 0, 9, 31]
    for off, pad in ((0, 0), (1, 2), (8, 8)):
        whole = torch.randn(6, 33, off + (4 + 2 + 2) * 64 + pad, generator=g, device="cuda").to(dt)
        q, k = whole[..., off:off + 256].unflatten(-1, (4, 64)), whole[..., off + 256:off + 384].unflatten(-1, (2, 64))
        old = whole.clone()
        qg, kg = torch.rand(64, generator=g, device="cuda"), torch.rand(64, generator=g, device="cuda")
        cos, sin = tables(g, 64, 64)
        needle.qk_norm_rope_dev(q, k, q, k, qg, kg, (cos, sin), i32(pos), rows=i32(rows))
        oq, ok = old[..., off:off + 256].unflatten(-1, (4, 64)), old[..., off + 256:off + 384].unflatten(-1, (2, 64))
        compare(q, oq, oq, qg, cos, sin, pos, rows)
        compare(k, ok, ok, kg, cos, sin, pos, rows)
        assert torch.equal(whole[..., off + 384:], old[..., off + 384:]) and torch.equal(whole[..., :off], old[..., :off])


def test_float32_is_the_separate_norm_and_rotation():
    # the same arithmetic but for the order of an exact sum's float64 additions
    import torch

    g = gen(6)
    vp = lambda x: ctypes.c_void_p(x.data_ptr())  # noqa: E731
    for w in (16, 64, 128):
        x = torch.randn(40, 3, 2, w, generator=g, device="cuda")
        gain = torch.rand(w, generator=g, device="cuda")
        cos, sin = tables(g, 50, w)
        pos = i32([b % 48 for b in range(40)])
        out, want = torch.zeros_like(x), torch.zeros_like(x)
        needle.qk_norm_rope_dev(out, None, x, None, gain, None, (cos, sin), pos)
        check(lib().nd_zcrmsnorm_dev(vp(want), vp(x), vp(gain), 40 * 3 * 2, w, None))
        each = (pos[:, None] + torch.arange(3, device="cuda", dtype=torch.int32)).contiguous()
        check(lib().nd_rope_dev(vp(want), 40 * 3, 2, w, vp(cos), vp(sin), 50, vp(each), 1, None))
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_values_at_the_ends_of_the_types():
    import torch

    gain = torch.ones(64, device="cuda")
    for dt, big in ((torch.float32, 1e18), (torch.bfloat16, 1e18), (torch.float16, 6e4)):
        x = torch.zeros(1, 4, 1, 64, device="cuda", dtype=dt)
        x[0, 1] = big
        x[0, 2, 0, 3] = float("nan")
        x[0, 3, 0, 0] = 1e-7
        out = torch.full_like(x, 2.0)
        needle.qk_norm_rope_dev(out, None, x, None, gain)
        assert (out[0, 0] == 0).all() and ((out[0, 1].float() - 1).abs() <= 2 * half_ulp(dt)).all()
        assert out[0, 2].isnan().all() and out[0, 3].isfinite().all()


def test_one_row_for_all():
    # expanded inputs: strides of 0
    import torch

    g = gen(9)
    gain, (cos, sin) = torch.rand(64, generator=g, device="cuda"), tables(g, 40, 64)
    for shape in ((1, 5), (3, 1), (1, 1)):
        x = torch.randn(*shape, 2, 64, generator=g, device="cuda").expand(3, 5, 2, 64)
        out, want = torch.zeros(3, 5, 2, 64, device="cuda"), torch.zeros(3, 5, 2, 64, device="cuda")
        needle.qk_norm_rope_dev(out, None, x, None, gain, None, (cos, sin), i32([0, 7, 30]))
        needle.qk_norm_rope_dev(want, None, x.contiguous(), None, gain, None, (cos, sin), i32([0, 7, 30]))
        assert torch.equal(out, want) and out.count_nonzero() > 0
