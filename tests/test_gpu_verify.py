"""needle.verify_drafts_dev against its float64 form (tests/page8_ref.py). The
counts and tokens are equal: both compare in float64, and a random number would have
to lie within 1e-13 of a border to tell them apart."""

import numpy as np
import pytest

from go_whistle_amd import needle
from page8_ref import FLOATS, gen, i32, verify64
from serve_ref import host

pytestmark = pytest.mark.gpu


def verify(target, drafts, draft, u, u_next, drafted, temperature, lp=True):
    import torch

    B, t = drafts.shape
    accepted, tokens = i32([9] * B), torch.full((B, t + 1), 77, dtype=torch.int32, device="cuda")
    out = torch.full((B, t + 1), 7.0, device="cuda") if lp else None
    needle.verify_drafts_dev(accepted, tokens, target, drafts, draft=draft, u=u, u_next=u_next,
                             drafted=None if drafted is None else i32(drafted), temperature=temperature, lp=out)
    torch.cuda.synchronize()
    ht, hd = host(target), None if draft is None or temperature == 0 else host(draft)
    hu, hn = (None if x is None else host(x) for x in (u, u_next))
    for b in range(B):
        a, tok, l = verify64(ht[b], host(drafts)[b], None if hd is None else hd[b], None if hu is None else hu[b],
                             None if hn is None else hn[b], t if drafted is None else drafted[b], temperature)
        assert int(accepted[b]) == a, b
        assert tokens[b].tolist() == tok.tolist(), b
        if lp:
            # float64 but for the last rounding
            got = host(out[b]).astype(np.float64)
            assert (np.isneginf(got) == np.isneginf(l)).all()
            fin = np.isfinite(l)
            assert (np.abs(got[fin] - l[fin]) <= 2.0 ** -24 * np.abs(l[fin]) + 1e-12).all(), b
    return accepted, tokens


def inputs(seed, io, B, t, n, near=0.8):
    import torch

    g, dt = gen(seed), getattr(torch, io)
    x = 3 * torch.randn(B, t + 1, n, generator=g, device="cuda")
    y = x[:, :t] + near * torch.randn(B, t, n, generator=g, device="cuda")
    off = torch.rand(n, generator=g, device="cuda") < 0.05
    off[n // 2] = False
    x, y = x.masked_fill(off, -np.inf).to(dt), y.masked_fill(off, -np.inf).to(dt)
    w = torch.softmax(y.double(), -1).cumsum(-1)
    d = (w <= torch.rand(B, t, 1, generator=g, device="cuda", dtype=torch.float64) * w[..., -1:]).sum(-1).clamp(max=n - 1).int()
    return x, y, d, torch.rand(B, t, generator=g, device="cuda"), torch.rand(B, generator=g, device="cuda")


@pytest.mark.parametrize("io", FLOATS)
@pytest.mark.parametrize("temperature", [0.0, 0.3, 1.0, 2.5])
@pytest.mark.parametrize("given", [True, False])
@pytest.mark.parametrize("B,t,n", [(1, 4, 8199), (40, 3, 33), (7, 16, 300), (3, 1, 4096), (5, 2, 4097), (2, 0, 100), (3, 5, 2),
                                   (2, 2, 1), (4, 3, 16384), (1, 2, 70001)])
def test_verify(io, temperature, given, B, t, n):
    x, y, d, u, nxt = inputs(B + t + n, io, B, t, n)
    verify(x, d, y if given else None, u, nxt, None, temperature)
    verify(x, d, y if given else None, u, nxt, [(b * 5) % (t + 3) - 1 for b in range(B)], temperature, lp=B % 2 == 0)


@pytest.mark.parametrize("io", FLOATS)
def test_strided_logits(io):
    import torch

    x, y, d, u, nxt = inputs(3, io, 5, 4, 1000)
    for pad, off in ((24, 0), (3, 1)):
        wide = torch.zeros(5, 5, 1000 + pad, dtype=x.dtype, device="cuda")
        wide[..., off:off + 1000] = x
        drow = torch.zeros(4, 5, 1000 + pad, dtype=x.dtype, device="cuda")  # rows before streams
        drow[..., off:off + 1000] = y.transpose(0, 1)
        verify(wide[..., off:off + 1000], d, drow[..., off:off + 1000].transpose(0, 1), u, nxt, None, 1.0)


def test_one_row_for_all():
    # expanded logits: strides of 0
    x, y, d, u, nxt = inputs(9, "float32", 4, 3, 1500)
    verify(x[:1].expand(4, 4, 1500), d, y[:1].expand(4, 3, 1500), u, nxt, None, 1.0)
    verify(x[:, :1].expand(4, 4, 1500), d, y[:, :1].expand(4, 3, 1500), u, nxt, None, 1.0)
    verify(x[:1, :1].expand(4, 4, 1500), d, None, u, nxt, [3, 0, 1, 2], 1.0)


def test_random_numbers_at_the_ends():
    import torch

    x, y, d, u, nxt = inputs(4, "float32", 6, 3, 5000)
    below = float(np.nextafter(np.float32(1), np.float32(0)))
    for uu in (0.0, below):
        for nn in (0.0, below, 1.0):
            verify(x, d, y, torch.full_like(u, uu), torch.full_like(nxt, nn), None, 0.8)
            verify(x, d, None, torch.full_like(u, uu), torch.full_like(nxt, nn), None, 0.8)


def test_equal_models_keep_all():
    # p = q: u < 1 keeps every draft, whatever the residual
    import torch

    x, _, d, u, nxt = inputs(5, "bfloat16", 9, 6, 2000, near=0.0)
    a, _ = verify(x, d, x[:, :6].contiguous(), u, nxt, None, 1.0)
    assert (a == 6).all()
    a, _ = verify(x, d, x[:, :6].contiguous(), torch.ones_like(u), nxt, None, 1.0)  # 1 * q < p is false; no residual: p
    assert (a == 0).all()


@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_rows_without_probabilities_and_bad_drafts(temperature):
    import torch

    x, y, d, u, nxt = inputs(6, "float32", 8, 3, 9000)
    u = u * 0.01
    x[0, 0, 5], x[1, 1, 6], x[2, 3] = np.nan, np.inf, -np.inf
    d[2] = d[2].clamp(min=0)
    y[3, 1, 7], y[4, 0] = np.nan, -np.inf
    d[5, 1], d[6, 0], d[7, 2] = -1, 9000, 2 ** 31 - 1
    verify(x, d, y, u, nxt, None, temperature)
    verify(x, d, None, u, nxt, None, temperature)


def test_greedy_takes_the_first_of_equals():
    import torch

    x = torch.zeros(2, 3, 10000, device="cuda")
    x[0, 0, 4321], x[0, 0, 9876], x[0, 1, 4100], x[0, 1, 4090] = 2.0, 2.0, 1.0, 1.0
    d = i32([[4321, 4090], [0, 1]])
    a, tok = verify(x, d, None, None, None, None, 0.0)
    assert a.tolist() == [2, 1] and tok.tolist() == [[4321, 4090, 0], [0, 0, -1]]


@pytest.mark.parametrize("temperature", [0.0, 1.0])
@pytest.mark.parametrize("n", [40, 20000])
def test_many_drafts(temperature, n):
    # more than a workgroup keeps the statistics of, nearly all of them kept
    import torch

    x, y, d, u, nxt = inputs(8, "float32", 2, 150, n, near=1e-3)
    d = x[:, :150].argmax(-1).int()
    d[1, 100] = (d[1, 100] + 1) % n
    u = u * 0.5
    a, _ = verify(x, d, y, u, nxt, None, temperature)
    assert a.max() > 64


def test_far_logits():
    # differences past float64's exponents, and a temperature that makes them so
    import torch

    x = torch.full((1, 2, 300), -3e38, device="cuda")
    x[0, :, 17] = 3e38
    d = i32([[17]])
    half = torch.full((1, 1), 0.5, device="cuda")
    for T in (1e-30, 1.0, 1e30):
        verify(x, d, None, half, half[0], None, T)
        verify(x, d, x[:, :1].contiguous(), half, half[0], None, T)
