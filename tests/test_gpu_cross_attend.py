"""needle.cross_attend_dev: float cross-attention to memories of other
lengths against its float64 form (bounds in tests/serve_ref.py)."""

import math

import numpy as np
import pytest

from go_whistle_amd import needle
from serve_ref import attend64, host

pytestmark = pytest.mark.gpu


def gen(seed):
    import torch

    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def i32(x):
    import torch

    return torch.tensor(x, dtype=torch.int32, device="cuda")


def check(out, before, q, k, v, scale, q_len, k_len, index, sample=None, seed=0):
    """Every output row, or `sample` of them, against float64; rows behind the last as they were."""
    import torch

    B, t, H, qk = q.shape
    M, F, Hk, vd = v.shape
    G = H // Hk
    ho, hb, hq, hk, hv = host(out).astype(np.float64), host(before).astype(np.float64), host(q), host(k), host(v)
    p_type = None if q.dtype == torch.float32 else q.dtype
    pick = np.random.default_rng(seed)
    for b in range(B):
        n = t if q_len is None else min(max(int(q_len[b]), 0), t)
        m = b if index is None else int(index[b])
        if not 0 <= m < M:
            n = 0
        assert np.array_equal(ho[b, n:], hb[b, n:]), b
        f = F if k_len is None or n == 0 else min(max(int(k_len[m]), 0), F)
        rows = range(n) if sample is None or n <= sample else sorted({0, n - 1, *pick.integers(0, n, sample).tolist()})
        for i in rows:
            for h in range(H) if sample is None else pick.integers(0, H, 2).tolist():
                o, bound, _, _ = attend64(hq[b, i, h], hk[m, :f, h // G], hv[m, :f, h // G], scale, q.dtype, p_type)
                err = np.abs(ho[b, i, h] - o)
                assert (err <= bound).all(), (b, i, h, (err / np.maximum(bound, 1e-300)).max())


def run(seed, name, B, t, M, F, H, Hk, qk, vd, q_len=None, k_len=None, index=None, sample=None):
    import torch

    g = gen(seed)
    dt = getattr(torch, name)
    mk = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dt)  # noqa: E731
    q, k, v = mk(B, t, H, qk), mk(M, F, Hk, qk), mk(M, F, Hk, vd)
    out = torch.full((B, t, H, vd), 3.0, device="cuda", dtype=dt)
    before, scale = out.clone(), math.sqrt(qk)
    dev = lambda x: None if x is None else i32(x)  # noqa: E731
    needle.cross_attend_dev(out, q, k, v, scale, q_len=dev(q_len), k_len=dev(k_len), index=dev(index))
    torch.cuda.synchronize()
    check(out, before, q, k, v, scale, q_len, k_len, index, sample, seed)


FLOATS = ["float32", "float16", "bfloat16"]


@pytest.mark.parametrize("name", FLOATS)
@pytest.mark.parametrize("H,Hk,qk,vd", [(8, 2, 48, 64), (4, 4, 16, 16), (6, 2, 128, 80), (3, 1, 256, 240), (2, 2, 80, 128),
                                        (5, 5, 112, 48)])
@pytest.mark.parametrize("t", [1, 3, 70])
def test_heads(name, H, Hk, qk, vd, t):
    run(t + H, name, 3, t, 3, 90, H, Hk, qk, vd, sample=None if t < 70 else 12)


@pytest.mark.parametrize("name", FLOATS)
@pytest.mark.parametrize("t,F", [(1, 1), (2, 15), (16, 16), (17, 33), (31, 64), (32, 65), (64, 127), (65, 128), (127, 31),
                                 (129, 257), (300, 375), (448, 63)])
def test_lengths(name, t, F):
    run(t * 7 + F, name, 2, t, 2, F, 4, 2, 64, 64, sample=14)


@pytest.mark.parametrize("name", FLOATS)
@pytest.mark.parametrize("t", [2, 130])
def test_ragged_shared_and_empty(name, t):
    # unequal query and memory lengths, empty ones, out-of-range ones (clamped),
    # beams that share a memory, indices outside the memories
    q_len = [t, 0, 1, t + 5, -3, t - 1, t, t]
    k_len = [200, 0, 1, 250, 77]
    index = [0, 1, 2, 3, 4, 0, -1, 5]
    run(t, name, 8, t, 5, 201, 6, 2, 48, 64, q_len, k_len, index, sample=10)
    run(t + 1, name, 8, t, 5, 201, 4, 4, 128, 128, q_len, k_len, [1, 1, 1, 3, 3, 3, 4, 2], sample=10)


@pytest.mark.parametrize("name", FLOATS)
@pytest.mark.parametrize("H,Hk,qk,vd,F", [(8, 4, 64, 64, 300), (8, 8, 48, 64, 130), (4, 4, 128, 128, 97),
                                          (4, 4, 112, 80, 200), (4, 2, 256, 256, 65), (4, 2, 144, 240, 33)])
def test_many_rows_of_many_streams(name, H, Hk, qk, vd, F):
    # enough columns for the float32 matrix form at every width, full and narrower than it
    run(H * qk, name, 40, 130, 40, F, H, Hk, qk, vd, [130 - (b % 7) * 20 for b in range(40)],
        [F - (m % 5) * (F // 6) for m in range(40)], None, sample=3)


@pytest.mark.parametrize("name", FLOATS)
@pytest.mark.parametrize("B", [64, 65])
def test_many_workgroups_of_unequal_memories(name, B):
    # more workgroups than one round: streams of long memories first (to 64 streams), equal lengths among them
    lens = [int(x) for x in np.random.default_rng(B).integers(0, 120, 20)]
    lens[3] = lens[7] = lens[11] = 119
    index = [(7 * b) % 22 - 1 for b in range(B)]  # one past either end too
    run(B, name, B, 150, 20, 120, 8, 4, 64, 64, [150 - b for b in range(B)], lens, index, sample=3)


@pytest.mark.parametrize("name", FLOATS)
def test_memories_fewer_than_streams_without_an_index(name):
    run(5, name, 3, 4, 2, 20, 2, 1, 32, 32)


@pytest.mark.parametrize("name", FLOATS)
@pytest.mark.parametrize("t", [1, 5, 90])
def test_no_frames_no_memories_and_the_dense_layout(name, t):
    import torch

    from go_whistle_amd._lib import check as ok
    from go_whistle_amd._lib import lib

    g = gen(29)
    dt = getattr(torch, name)
    B, F, H, Hk, D = 3, 40, 4, 2, 64
    mk = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dt)  # noqa: E731
    q = mk(B, t, H, D)
    out = torch.full_like(q, 5.0)
    needle.cross_attend_dev(out, q, mk(B, 0, Hk, D), mk(B, 0, Hk, D), 8.0)
    torch.cuda.synchronize()
    assert (out == 0).all()
    out.fill_(5.0)
    needle.cross_attend_dev(out, q, mk(0, F, Hk, D), mk(0, F, Hk, D), 8.0, index=i32([0, 0, 0]))
    torch.cuda.synchronize()
    assert (out == 5).all()
    needle.cross_attend_dev(out[:0], q[:0], mk(2, F, Hk, D), mk(2, F, Hk, D), 8.0)
    needle.cross_attend_dev(out[:, :0], q[:, :0], mk(3, F, Hk, D), mk(3, F, Hk, D), 8.0)
    k, v, want = mk(B, F, Hk, D), mk(B, F, Hk, D), torch.empty_like(q)
    needle.cross_attend_dev(want, q, k, v, 8.0)
    ok(lib().nd_cross_attend_dev(out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                 FLOATS.index(name), None, B, t, H, Hk, D, D, B, F, None, None, None, 8.0,
                                 torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("name", FLOATS)
@pytest.mark.parametrize("t", [1, 100])
def test_strides(name, t):
    # head-major memories, queries and outputs inside wider rows
    import torch

    g = gen(17)
    dt = getattr(torch, name)
    B, M, F, H, Hk, D = 2, 2, 77, 4, 2, 64
    k = torch.randn(M, Hk, F, D, generator=g, device="cuda").to(dt).transpose(1, 2)
    v = torch.randn(M, F, Hk, 2 * D, generator=g, device="cuda").to(dt)[..., D:]
    q = torch.randn(B, t + 1, H * D + 3, generator=g, device="cuda").to(dt)[:, 1:, 3:].unflatten(2, (H, D))
    wide = torch.full((B, t, H * D + 5), 2.0, device="cuda", dtype=dt)
    out = wide[:, :, 1:1 + H * D].unflatten(2, (H, D))
    needle.cross_attend_dev(out, q, k, v, 8.0)
    torch.cuda.synchronize()
    check(out, out.clone(), q, k, v, 8.0, None, None, None, sample=20)
    assert (wide[:, :, 0] == 2).all() and (wide[:, :, 1 + H * D:] == 2).all()


@pytest.mark.parametrize("name", FLOATS)
@pytest.mark.parametrize("t,B", [(1, 2), (80, 2), (80, 60)])
def test_frames_behind_the_last_may_hold_anything(name, t, B):
    import torch

    g = gen(19)
    dt = getattr(torch, name)
    F, H, Hk, D = 150, 4, 2, 64
    q, k, v = (torch.randn(*s, generator=g, device="cuda").to(dt) for s in ((B, t, H, D), (B, F, Hk, D), (B, F, Hk, D)))
    k_len = i32([101, 0] + [150] * (B - 2))
    outs = []
    for fill in (0.0, float("nan"), float("inf")):
        k[0, 101:], v[0, 101:], k[1], v[1] = fill, fill, fill, fill
        out = torch.full((B, t, H, D), 4.0, device="cuda", dtype=dt)
        needle.cross_attend_dev(out, q, k, v, 8.0, k_len=k_len)
        torch.cuda.synchronize()
        outs.append(out)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    assert (outs[0][1] == 0).all() and torch.isfinite(outs[0]).all()


@pytest.mark.parametrize("name", FLOATS)
@pytest.mark.parametrize("t,B", [(1, 1), (80, 1), (80, 200)])
def test_extreme_logits(name, t, B):
    import torch

    dt = getattr(torch, name)
    q = torch.zeros(B, t, 1, 64, device="cuda", dtype=dt)
    q[..., 0] = 1
    k = torch.zeros(B, 100, 1, 64, device="cuda", dtype=dt)
    v = torch.randn(B, 100, 1, 64, generator=gen(3), device="cuda").to(dt)
    out = torch.empty(B, t, 1, 64, device="cuda", dtype=dt)
    k[..., 0] = -float("inf")
    needle.cross_attend_dev(out, q, k, v, 1.0)
    torch.cuda.synchronize()
    assert (out == 0).all()
    k[..., 0] = -30000
    k[:, 57, 0, 0] = 30000
    needle.cross_attend_dev(out, q, k, v, 1.0)
    torch.cuda.synchronize()
    assert torch.equal(out, v[:, 57:58].expand_as(out))
    k[:, 99, 0, 0] = float("nan")
    needle.cross_attend_dev(out, q, k, v, 1.0)
    torch.cuda.synchronize()
    assert torch.isnan(out).all()


@pytest.mark.parametrize("name", ["float32", "bfloat16"])
@pytest.mark.parametrize("t", [2, 200])
def test_graph_replays(name, t):
    import torch

    g = gen(23)
    B, F, H, D = 2, 700, 4, 64
    dt = getattr(torch, name)
    q, k, v = (torch.randn(B, n, H, D, generator=g, device="cuda").to(dt) for n in (t, F, F))
    k_len = i32([F, 333])
    out, other = torch.empty_like(q), torch.empty_like(q)
    needle.cross_attend_dev(other, q, k, v, 8.0, k_len=k_len)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        needle.cross_attend_dev(out, q, k, v, 8.0, k_len=k_len)
    for r in range(3):
        q.copy_(torch.randn(q.shape, generator=g, device="cuda").to(dt))
        out.zero_()
        graph.replay()
        needle.cross_attend_dev(other, q, k, v, 8.0, k_len=k_len)
        torch.cuda.synchronize()
        assert torch.equal(out, other), r


@pytest.mark.parametrize("name", FLOATS)
@pytest.mark.parametrize("B,t,F", [(1, 1, 5), (2, 1, 300), (2, 3, 77), (2, 40, 33), (2, 80, 150), (60, 80, 150), (1, 90, 65)])
@pytest.mark.parametrize("D,W", [(64, 64), (48, 64), (128, 80), (256, 256)])
def test_an_infinite_value_of_the_last_frame(name, B, t, F, D, W):
    # the last frame's weight is above 0, so its coordinate is the infinity; the others are as without it
    import torch

    g = gen(31)
    dt = getattr(torch, name)
    q, k, v = (torch.randn(*s, generator=g, device="cuda").to(dt) for s in ((B, t, 4, D), (B, F, 2, D), (B, F, 2, W)))
    outs = []
    for x in (1.0, float("inf")):
        v[:, F - 1, :, 7] = x
        outs.append(torch.empty(B, t, 4, W, device="cuda", dtype=dt))
        needle.cross_attend_dev(outs[-1], q, k, v, math.sqrt(D))
    torch.cuda.synchronize()
    assert (outs[1][..., 7] == float("inf")).all()
    for o in outs:
        o[..., 7] = 0
    assert torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("name", FLOATS)
@pytest.mark.parametrize("B,t", [(1, 2), (16, 400)])
def test_many_small_weights_beside_a_large_one(name, B, t):
    # 20,000 frames of weight e^-17.375 = 2.85e-8, below half of float16's
    # least subnormal, beside one of 1: 5.7e-4 of the sum. The bound of
    # serve_ref, and where weights are rounded to float16, whose subnormals'
    # half step 2^-25 is 2^-32 of a largest weight of 2^7, that much of every
    # |v| = 1: 4.7e-6.
    import torch

    dt = getattr(torch, name)
    F = 20001
    q = torch.ones(B, t, 8, 64, device="cuda", dtype=dt)
    k = torch.full((1, F, 8, 64), -17.375 / 64, device="cuda", dtype=dt)  # 17.375 / 64 = 139 / 512
    v = torch.ones(1, F, 8, 64, device="cuda", dtype=dt)
    k[:, 0] = 0
    v[:, 0] = 0
    out = torch.empty_like(q)
    needle.cross_attend_dev(out, q, k, v, 1.0, index=i32([0] * B))
    torch.cuda.synchronize()
    kq, vq = host(k)[0, :, 0], host(v)[0, :, 0]
    o, bound, _, _ = attend64(host(q)[0, 0, 0], kq, vq, 1.0, dt, None if name == "float32" else dt)
    err = np.abs(host(out).astype(np.float64) - o)
    if name == "float16":
        bound = bound + F * 2.0 ** -32
    assert (err <= bound).all(), (err / bound).max()
