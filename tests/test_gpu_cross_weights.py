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
@pytest.mark.parametrize("B,t,F", [(1, 1, 100), (2, 2, 100), (2, 140, 100), (70, 33, 100), (2, 2, 300), (70, 3, 300), (1, 9, 3000)])
def test_infinite_values_of_equal_weights(name, qk, vd, B, t, F):
    # weights of exactly 1 before the sum: one part holds them, the second is 0
    import torch

    g, dt, H = gen(qk + t), getattr(torch, name), 2
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


@pytest.mark.parametrize("name", ["float32"] + HALVES)
@pytest.mark.parametrize("scale", [1.0, 8.0, math.sqrt(48)])
@pytest.mark.parametrize("B,t,F", [(1, 1, 100), (2, 2, 100), (2, 2, 700), (2, 80, 100), (70, 33, 65), (2, 400, 70)])
def test_far_logits(name, scale, B, t, F):
    # dots past 2^28 (float16: 64 products of 30000 and about as much, exact in
    # float32) or about +-1e30: the frame of the largest logit is the answer,
    # of two equal ones their mean, also from far below 0
    import torch

    dt, D = getattr(torch, name), 64
    q = torch.full((B, t, 1, D), 30000.0 if name == "float16" else 1e15, device="cuda", dtype=dt)
    v = torch.randn(B, F, 1, D, generator=gen(F), device="cuda").to(dt)
    base = torch.arange(F, device="cuda").view(1, F, 1, 1).expand(B, F, 1, D)
    for low, step, high in ((20000.0, 16.0, 30000.0), (-30000.0, 16.0, -16.0), (-30000.0, 0.0, 0.0)):
        k = (low + step * (base * 7 % 11)) * (1.0 if name == "float16" else 1e9)
        k[:, F // 2] = high * (1.0 if name == "float16" else 1e9)
        k = k.to(dt)
        out = torch.full((B, t, 1, D), 5.0, device="cuda", dtype=dt)
        needle.cross_attend_dev(out, q, k, v, scale)
        torch.cuda.synchronize()
        assert torch.equal(out, v[:, F // 2:F // 2 + 1].expand_as(out)), low
        k[:, F - 1] = k[:, F // 2]
        needle.cross_attend_dev(out, q, k, v, scale)
        torch.cuda.synchronize()
        want = ((v[:, F // 2].double() + v[:, F - 1].double()) / 2).to(dt)
        assert torch.equal(out, want.unsqueeze(1).expand_as(out)), low


@pytest.mark.parametrize("name", ["float32"] + HALVES)
@pytest.mark.parametrize("size", [2.0 ** 10, 2.0 ** 19, 2.0 ** 20, 2.0 ** 21, 2.0 ** 24, 2.0 ** 27])
def test_outputs_stay_between_the_values(name, size):
    # logits of each size, of rows side by side in a wavefront that differ in it
    import torch

    g, dt, B, t, F, D = gen(3), getattr(torch, name), 4, 130, 200, 64
    q, k, v = (torch.randn(B, n, 2, D, generator=g, device="cuda").to(dt) for n in (t, F, F))
    q[:, ::3] *= 2.0 ** 12
    q[:, 1::3] = 0
    out = torch.empty_like(q)
    needle.cross_attend_dev(out, q, k, v, 2.0 ** 15 / size)
    torch.cuda.synchronize()
    lo, hi = v.float().amin(1, keepdim=True), v.float().amax(1, keepdim=True)
    slack = 2 * half_ulp(dt) * v.float().abs().max()
    assert (out.float() >= lo - slack).all() and (out.float() <= hi + slack).all()
    mean = v.double().mean(1, keepdim=True)
    assert (out[:, 1::3].double() - mean).abs().max() <= 2 * half_ulp(dt) * mean.abs().max() + F * 2.0 ** -24


@pytest.mark.parametrize("name", HALVES)
@pytest.mark.parametrize("B,t,H,Hk,qk,vd,F", [(1, 8, 4, 4, 64, 64, 256), (2, 1, 8, 1, 48, 64, 300), (3, 4, 4, 2, 16, 16, 511),
                                              (40, 3, 4, 4, 64, 48, 290), (70, 16, 2, 2, 32, 64, 257), (70, 2, 16, 2, 64, 64, 700),
                                              (33, 5, 12, 4, 64, 64, 1030)])
def test_few_rows_of_narrow_heads(name, B, t, H, Hk, qk, vd, F):
    # lists taken whole by the split form: its weights are float32. Ragged rows
    # and memories, shared and missing ones, rows inside wider ones.
    import torch

    g, dt = gen(B + F), getattr(torch, name)
    M = max(1, B // 2)
    q = torch.randn(B, t, H * qk + 8, generator=g, device="cuda").to(dt)[..., 5:5 + H * qk].unflatten(2, (H, qk))
    k, v = (torch.randn(M, Hk, F, w, generator=g, device="cuda").to(dt).transpose(1, 2) for w in (qk, vd))
    wide = torch.full((B, t, H * vd + 3), 7.0, device="cuda", dtype=dt)
    out = wide[..., 1:1 + H * vd].unflatten(2, (H, vd))
    q_len = [(b * 5) % (t + 2) - (b == 4) for b in range(B)]
    q_len[0] = t
    k_len = [F - (m * 37) % (F + 1) for m in range(M)]
    index = [(b * 3) % (M + (B > 8)) for b in range(B)]
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    needle.cross_attend_dev(out, q, k, v, math.sqrt(qk), q_len=dev(q_len), k_len=dev(k_len), index=dev(index))
    torch.cuda.synchronize()
    assert (wide[..., 0] == 7).all() and (wide[..., 1 + H * vd:] == 7).all()
    ho, hq, hk, hv = (host(x).astype(np.float64) for x in (out, q, k, v))
    pick = np.random.default_rng(t)
    for b in range(B):
        n, m = min(max(q_len[b], 0), t), index[b]
        n = n if m < M else 0
        assert (ho[b, n:] == 7).all(), b
        for i in {0, n - 1} if n else ():
            for h in pick.integers(0, H, 3).tolist():
                o, bound, _, _ = attend64(hq[b, i, h], hk[m, :k_len[m], h // (H // Hk)], hv[m, :k_len[m], h // (H // Hk)],
                                          math.sqrt(qk), dt)
                assert (np.abs(ho[b, i, h] - o) <= bound).all(), (b, i, h)
