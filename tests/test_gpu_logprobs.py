"""needle.logprobs_dev: log probabilities of given tokens, entropy and the top
alternatives against float64.

Bounds, u = 2^-24: x - m is off by u |x - m|, e^(x - m) by that and 2^-21
(the exponent function) relatively, the sum l by that of its terms weighed
by them and its own n u, the logarithm by u log l: so a log probability by
u (2 D + n + 4) + 2^-20 + 2 u |lp| with D the largest |x - m| whose term is
above 0 (at most 104). The entropy is a mean of x - m with those weights
beside log l: twice that times (1 + D)."""

import math

import numpy as np
import pytest

from go_whistle_amd import needle
from serve_ref import U, host

pytestmark = pytest.mark.gpu

FLOATS = ["float32", "float16", "bfloat16"]


def gen(seed):
    import torch

    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def run(x, tok, top):
    import torch

    rows = x.shape[0]
    lp, ent = (torch.full((rows,), 9.0, device="cuda") for _ in range(2))
    ti = torch.full((rows, top), -7, dtype=torch.int32, device="cuda")
    tl = torch.full((rows, top), 9.0, device="cuda")
    needle.logprobs_dev(x, tokens=tok, lp=lp, ent=ent, top=ti, top_lp=tl)
    torch.cuda.synchronize()
    return lp, ent, ti, tl


def check(x, tok, top):
    lp, ent, ti, tl = (host(z) for z in run(x, tok, top))
    h, tk = host(x).astype(np.float64), tok.cpu().numpy()
    n = x.shape[1]
    for r in range(x.shape[0]):
        m = h[r].max()
        with np.errstate(invalid="ignore", over="ignore"):
            e = np.exp(h[r] - m)
        want = (h[r] - m) - math.log(e.sum())  # m + log would lose the log where m is the type's lowest value
        d = min(104.0, float((m - h[r][np.isfinite(h[r])]).max()))
        tol = U * (2 * d + n + 4) + 2.0 ** -20

        def close(got, w):
            if w == -np.inf:
                return got == -np.inf
            return abs(got - w) <= tol + 2 * U * abs(w)

        if tk[r] < 0:
            assert lp[r] == 0
        elif tk[r] >= n:
            assert np.isnan(lp[r])
        else:
            assert close(lp[r], want[tk[r]]), r
        p = np.exp(want)
        went = -(p[p > 0] * want[p > 0]).sum()
        assert abs(ent[r] - went) <= 2 * tol * (1 + d), (r, ent[r], went)
        order = np.lexsort((np.arange(n), -h[r]))[:top]
        assert np.array_equal(ti[r], order), r
        assert all(close(tl[r, q], want[order[q]]) for q in range(top)), r


@pytest.mark.parametrize("name", FLOATS)
@pytest.mark.parametrize("n", [1, 2, 7, 63, 64, 65, 511, 512, 513, 1000, 8199, 16383, 16384, 16385, 50001])
def test_sizes(name, n):
    import torch

    g = gen(n)
    x = (4 * torch.randn(5, n, generator=g, device="cuda")).to(getattr(torch, name))
    tok = torch.tensor([0, n - 1, -1, n, n // 2], dtype=torch.int32, device="cuda")
    check(x, tok, min(n, 10))


@pytest.mark.parametrize("top", [0, 1, 2, 31, 32, 33, 64])
@pytest.mark.parametrize("n", [64, 777, 20000, 140000])
def test_tops(top, n):
    import torch

    g = gen(top)
    x = torch.randn(3, n, generator=g, device="cuda")
    check(x, torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda"), top)


@pytest.mark.parametrize("n", [100, 4096, 16384, 33000])
def test_ties_take_the_lowest_index(n):
    import torch

    g = gen(n)
    tok = torch.zeros(6, dtype=torch.int32, device="cuda")
    x = torch.randint(0, 3, (6, n), generator=g, device="cuda").float()
    x[1] = 0.0  # all equal
    x[2] = torch.where(torch.rand(n, generator=g, device="cuda") < 0.5, 0.0, -0.0)  # -0 is 0
    x[3] = -torch.arange(n, device="cuda").float() / n  # in order
    x[4] = torch.arange(n, device="cuda").float() / n  # against it
    check(x, tok, 33)
    check(x.bfloat16(), tok, 20)


def test_suppressed_tokens_and_lowest_values():
    import torch

    x = torch.randn(4, 9000, generator=gen(1), device="cuda")
    x[0, ::2] = -float("inf")
    x[1, 5:] = -float("inf")  # fewer live ones than alternatives
    x[2, 1:] = torch.finfo(torch.float32).min
    x[3, :] = torch.finfo(torch.float32).min  # all equal and lowest
    tok = torch.tensor([0, 4, 0, 17], dtype=torch.int32, device="cuda")
    check(x[1:2], tok[1:2], 12)
    check(x[[0, 3]].contiguous(), tok[[0, 3]], 12)
    lp, ent, ti, tl = run(x[2:3], tok[2:3], 3)
    assert lp.item() == 0 and ent.item() == 0 and ti[0].tolist() == [0, 1, 2]


@pytest.mark.parametrize("n", [40, 16384, 40000])
def test_rows_of_infinities_and_nan(n):
    import torch

    x = torch.randn(5, n, generator=gen(n), device="cuda")
    x[0] = -float("inf")
    x[1, n // 2] = float("nan")
    x[2, 3] = float("inf")
    x[3] = float("nan")
    x[4, 1:] = -float("inf")
    tok = torch.tensor([1, 1, 3, 0, 0], dtype=torch.int32, device="cuda")
    lp, ent, ti, tl = run(x, tok, 4)
    assert lp[0] == -float("inf") and ent[0] == 0 and ti[0].tolist() == [0, 1, 2, 3] and (tl[0] == -float("inf")).all()
    for r in (1, 2, 3):
        assert torch.isnan(lp[r]) and torch.isnan(ent[r]) and torch.isnan(tl[r]).all(), r
    h = torch.where(torch.isnan(x), -float("inf"), x).cpu().numpy()
    for r in range(5):
        assert ti[r].tolist() == np.lexsort((np.arange(n), -h[r]))[:4].tolist(), r
    assert lp[4] == 0 and ent[4] == 0


@pytest.mark.parametrize("name", FLOATS)
def test_row_strides_and_odd_starts(name):
    import torch

    big = torch.randn(7, 9001, generator=gen(3), device="cuda").to(getattr(torch, name))
    tok = torch.tensor([0, 5, 2000, 70, 8190, 1, 2], dtype=torch.int32, device="cuda")
    check(big[:, 3:8202], tok, 5)
    check(big[::2, 1:500], tok[::2].contiguous(), 5)


def test_parts_on_their_own():
    # each output alone, and rows wider than one workgroup's part from two streams at once
    import torch

    x = torch.randn(40, 70000, generator=gen(9), device="cuda")
    tok = torch.arange(40, dtype=torch.int32, device="cuda")
    lp, ent, ti, tl = run(x, tok, 6)
    for z in range(3):
        a = torch.zeros(40, device="cuda")
        i, b = torch.zeros(40, 6, dtype=torch.int32, device="cuda"), torch.zeros(40, 6, device="cuda")
        if z == 0:
            needle.logprobs_dev(x, tokens=tok, lp=a)
            assert torch.equal(a, lp)
        elif z == 1:
            needle.logprobs_dev(x, ent=a)
            assert torch.equal(a, ent)
        else:
            needle.logprobs_dev(x, top=i, top_lp=b)
            assert torch.equal(i, ti) and torch.equal(b, tl)
    streams = [torch.cuda.Stream() for _ in range(2)]
    xs = [x, x.flip(0).contiguous()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for s in range(2):
            with torch.cuda.stream(streams[s]):
                e = torch.empty(40, device="cuda")
                needle.logprobs_dev(xs[s], ent=e)
                got[s].append(e)
    torch.cuda.synchronize()
    assert all(torch.equal(e, ent) for e in got[0]) and all(torch.equal(e, ent.flip(0)) for e in got[1])


def test_graph_replays():
    import torch

    g = gen(13)
    x = torch.randn(3, 50000, generator=g, device="cuda")
    tok = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")
    lp, ent = torch.zeros(3, device="cuda"), torch.zeros(3, device="cuda")
    top, tl = torch.zeros(3, 8, dtype=torch.int32, device="cuda"), torch.zeros(3, 8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        needle.logprobs_dev(x, tokens=tok, lp=lp, ent=ent, top=top, top_lp=tl)
    for _ in range(3):
        x.normal_(generator=g)
        graph.replay()
        want = run(x, tok, 8)
        assert all(torch.equal(a, b) for a, b in zip((lp, ent, top, tl), want))


@pytest.mark.parametrize("name", FLOATS)
@pytest.mark.parametrize("n", [2040, 2041, 2048, 2049, 4097, 6145, 8185, 10241, 12289, 14337, 32760, 32761, 32768, 32769])
def test_wavefronts_of_a_row(name, n):
    # sizes either side of what one more wavefront holds, in rows that start on a 16-byte boundary and in others
    import torch

    g = gen(n)
    wide = (3 * torch.randn(4, n + 8 - n % 8 + 8, generator=g, device="cuda")).to(getattr(torch, name))
    tok = torch.tensor([n - 1, 0, n // 3, 7], dtype=torch.int32, device="cuda")
    check(wide[:, :n], tok, 3)
    check(wide[:, 1:n + 1], tok, 33)
    check(wide.view(-1)[7:7 + n].view(1, n), tok[:1], 64)


@pytest.mark.parametrize("name", FLOATS)
@pytest.mark.parametrize("n,top", [(600, 64), (2000, 7), (3000, 64), (20000, 5)])
def test_equal_logits_of_short_rows(name, n, top):
    # more of them than are ranked at once
    import torch

    x = torch.full((3, n), -2.5, device="cuda", dtype=getattr(torch, name))
    x[1, n // 2:] = 1.0
    x[2, n - 1] = 4.0
    check(x, torch.tensor([0, n - 1, n], dtype=torch.int32, device="cuda"), top)
