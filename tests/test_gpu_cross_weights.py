"""nd_cross_attend_dev's softmax weights in 16-bit types, and the numbers they
meet: logits of any size, infinite values.

A weight enters the second product in two parts: off by 2^-16 of it in
bfloat16 (a truncation to 8 bits leaves at most 2^-7, of which rounding to the
nearest of 8 bits loses 2^-9) and by 2^-22 in float16 (2^-11 twice), where
the least subnormal's half step 2^-25 is 2^-32 of a largest weight of 2^7 at
least. Everything else is the float32 arithmetic that tests/serve_ref.py
bounds."""

import math

import numpy as np
import pytest

from go_whistle_amd import needle
from serve_ref import attend64, half_ulp, host

pytestmark = pytest.mark.gpu

HALVES = ["float16", "bfloat16"]
PARTS = {"float16": 2.0 ** -22, "bfloat16": 2.0 ** -16}


def gen(seed):
    import torch

    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


@pytest.mark.parametrize("name", HALVES)
@pytest.mark.parametrize("H,Hk,qk,vd", [(2, 2, 64, 64), (4, 1, 48, 64), (2, 2, 128, 128), (3, 1, 112, 80), (2, 1, 256, 240)])
@pytest.mark.parametrize("t,F", [(2, 33), (3, 700), (70, 130), (300, 65)])
def test_weights_hold_more_than_their_type(name, H, Hk, qk, vd, t, F):
    import torch

    g, dt, B = gen(t + F + qk), getattr(torch, name), 2
    q, k, v = (torch.randn(*s, generator=g, device="cuda").to(dt) for s in ((B, t, H, qk), (B, F, Hk, qk), (B, F, Hk, vd)))
    out = torch.empty(B, t, H, vd, device="cuda", dtype=dt)
    needle.cross_attend_dev(out, q, k, v, math.sqrt(qk))
    torch.cuda.synchronize()
    ho, hq, hk, hv = (host(x).astype(np.float64) for x in (out, q, k, v))
    pick = np.random.default_rng(t)
    for b in range(B):
        for i in sorted({0, t - 1, *pick.integers(0, t, 6).tolist()}):
            for h in range(H):
                vals = hv[b, :, h // (H // Hk)]
                o, bound, w, _ = attend64(hq[b, i, h], hk[b, :, h // (H // Hk)], vals, math.sqrt(qk), dt)
                part = PARTS[name] * (w @ np.abs(vals)) + (2.0 ** -32 * np.abs(vals).sum(0) if name == "float16" else 0)
                err = np.abs(ho[b, i, h] - o)
                assert (err <= bound + part * (1 + half_ulp(dt))).all(), (b, i, h, (err / (bound + part)).max())


@pytest.mark.parametrize("name", ["float32"] + HALVES)
@pytest.mark.parametrize("qk,vd", [(64, 64), (48, 64), (128, 80), (256, 256)])
@pytest.mark.parametrize("B,t", [(1, 1), (2, 2), (2, 140), (70, 33)])
def test_infinite_values_of_equal_weights(name, qk, vd, B, t):
    # weights of exactly 1 before the sum: one part holds them, the second is 0
    import torch

    g, dt, F, H = gen(qk + t), getattr(torch, name), 100, 2
    q = torch.zeros(B, t, H, qk, device="cuda", dtype=dt)
    k, v = (torch.randn(B, F, H, w, generator=g, device="cuda").to(dt) for w in (qk, vd))
    v[:, 3, :, 5], v[:, 77, :, 9] = float("inf"), -float("inf")
    v[:, 20, :, 11], v[:, 90, :, 11] = float("inf"), -float("inf")
    v[:, 50, :, 13] = float("nan")
    out = torch.empty(B, t, H, vd, device="cuda", dtype=dt)
    needle.cross_attend_dev(out, q, k, v, 8.0)
    clean = v.clone()
    clean[~torch.isfinite(v)] = 0
    want = torch.empty_like(out)
    needle.cross_attend_dev(want, q, k, clean, 8.0)
    torch.cuda.synchronize()
    assert (out[..., 5] == float("inf")).all() and (out[..., 9] == -float("inf")).all()
    assert torch.isnan(out[..., 11]).all() and torch.isnan(out[..., 13]).all()
    rest = [d for d in range(vd) if d not in (5, 9, 11, 13)]
    assert torch.equal(out[..., rest], want[..., rest])


@pytest.mark.parametrize("name", HALVES)
@pytest.mark.parametrize("qk,vd", [(64, 64), (112, 80), (256, 256)])
def test_a_row_of_nan_leaves_the_others_as_they_are(name, qk, vd):
    import torch

    g, dt, B, t, F, H = gen(qk), getattr(torch, name), 2, 200, 150, 2
    q, k, v = (torch.randn(*s, generator=g, device="cuda").to(dt) for s in ((B, t, H, qk), (B, F, H, qk), (B, F, H, vd)))
    outs = []
    for x in (0.5, float("nan")):
        q[1, 77, 0, 3] = x
        outs.append(torch.empty(B, t, H, vd, device="cuda", dtype=dt))
        needle.cross_attend_dev(outs[-1], q, k, v, 8.0)
    torch.cuda.synchronize()
    assert torch.isnan(outs[1][1, 77, 0]).all() and torch.isfinite(outs[0]).all()
    # a raised maximum is the wavefront's: its other rows may be rounded otherwise
    outs[0][1, 77, 0] = outs[1][1, 77, 0] = 0
    o = outs[0].float()
    assert (outs[1].float() - o).abs().max() <= 2 * half_ulp(dt) * o.abs().max()
