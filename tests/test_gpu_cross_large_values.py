"""needle.cross_attend_dev over values near float32's largest, with logits that
rise by less than what a running maximum may lag behind them: outputs are
finite and within their bounds (tests/serve_ref.py)."""

import pytest

from go_whistle_amd import needle
from page8_ref import gen
from test_gpu_cross_attend import check
from test_gpu_large_values import BIG, SCALE, lifted

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["bfloat16", "float32"])
@pytest.mark.parametrize("B,t,F,H,Hk,w", [
    (1, 1, 1500, 8, 8, 64),
    (2, 5, 1500, 8, 8, 64),
    (1, 300, 1500, 4, 2, 64),
    (64, 448, 300, 8, 8, 64),
    (32, 130, 700, 4, 4, 128),
    (30, 200, 500, 6, 3, 240),
    (64, 200, 260, 8, 8, 48),
])
def test_cross_attention(name, B, t, F, H, Hk, w):
    import torch

    g, dt = gen(t), getattr(torch, name)
    k = torch.zeros(B, F, Hk, w, device="cuda")
    k[..., :16] = torch.tensor(lifted(F), device="cuda").float()[None, :, None, None] / 256
    v = BIG * (0.5 + 0.5 * torch.rand(B, F, Hk, w, generator=g, device="cuda"))
    sign = torch.where(torch.rand(v.shape, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    v[..., :w // 2] *= sign[0, 0, 0, :w // 2]  # of one sign for all frames, and of either
    v[..., w // 2:] *= sign[..., w // 2:]
    k, v = k.to(dt), v.to(dt)
    q = torch.ones(B, t, H, w, device="cuda", dtype=dt)
    out = torch.zeros_like(q)
    needle.cross_attend_dev(out, q, k, v, SCALE)
    assert out.isfinite().all()
    some = [0, B - 1]
    check(out[some], out[some], q[some], k[some], v[some], SCALE, None, None, None, sample=3)
    # an infinite value is one still
    v[0, F // 2, 0, 3] = float("inf")
    needle.cross_attend_dev(out, q, k, v, SCALE)
    assert (out[0, :, :H // Hk, 3] == float("inf")).all() and out[0, :, :H // Hk, 4:].isfinite().all()
