"""needle.verify_drafts_dev of vocabularies in many parts, call after call in one
workspace: no call sees sums that an earlier one left."""

import numpy as np
import pytest

from go_whistle_amd import needle
from page8_ref import i32, verify64
from serve_ref import host
from test_gpu_verify import inputs

pytestmark = pytest.mark.gpu


def outputs(B, t):
    import torch

    return i32([9] * B), torch.full((B, t + 1), 77, dtype=torch.int32, device="cuda"), torch.zeros(B, t + 1, device="cuda")


def right(got, args, temperature, streams):
    x, y, d, u, nxt = (host(z) for z in args)
    for b in streams:
        a, tok, lp = verify64(x[b], d[b], y[b], u[b], nxt[b], d.shape[1], temperature)
        assert int(got[0][b]) == a and got[1][b].tolist() == tok.tolist(), b
        fin = np.isfinite(lp)
        assert (np.abs(host(got[2][b])[fin] - lp[fin]) <= 2.0 ** -24 * np.abs(lp[fin]) + 1e-12).all(), b


def test_calls_of_other_sizes_in_one_workspace():
    import torch

    shapes = [(64, 2, 16384), (3, 1, 70001), (64, 2, 16384), (1, 4, 8199), (200, 1, 5000), (40, 3, 33), (3, 1, 70001)]
    calls = [(inputs(i, "float32", *s), outputs(*s[:2])) for i, s in enumerate(shapes)]
    for (x, y, d, u, nxt), got in calls:  # one behind the other, without a wait
        needle.verify_drafts_dev(got[0], got[1], x, d, draft=y, u=u, u_next=nxt, temperature=0.7, lp=got[2])
    torch.cuda.synchronize()
    for (args, got), (B, _, _) in zip(calls, shapes):
        right(got, args, 0.7, {0, B // 2, B - 1})


def test_replays_with_other_logits():
    import torch

    B, t, n = 16, 2, 16384
    sets = [inputs(40 + i, "float32", B, t, n) for i in range(5)]
    x, y, d, u, nxt = (z.clone() for z in sets[0])
    got, eager = outputs(B, t), outputs(B, t)
    call = lambda o: needle.verify_drafts_dev(o[0], o[1], x, d, draft=y, u=u, u_next=nxt, temperature=1.0, lp=o[2])  # noqa: E731
    call(got)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(got)
    for args in sets:
        for z, w in zip((x, y, d, u, nxt), args):
            z.copy_(w)
        g.replay()
        call(eager)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, eager))
        right(got, args, 1.0, (0, 7, B - 1))
