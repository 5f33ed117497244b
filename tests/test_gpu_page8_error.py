"""How far the rows of 8-bit pages with one scale a page and head are from the
rows that were appended: half a step for each scale that their page has had since.

A value x takes the code of float32(x / s), and a code c under a new scale s' that
of float32(float32(c s) / s'). With u = 2^-24 the quotients are off by u and 2 u
of themselves, at most L 2 u <= 2^-14 code values (L = 448), and the code by half a step: 1/2
in int8; in e4m3 2^-4 of the quotient, at least half the subnormal step, 2^-10. So
the row's error grows by s (1/2 + 2^-14) in int8, and in e4m3 by s (max(2^-4 |y|,
2^-10) + 2^-14) with y the quotient, at most (|x| + its error before) / s (1 + 2 u)."""

import numpy as np
import pytest

from page8_ref import cache_rows, gen, i32, make_cache
from serve_ref import host

pytestmark = pytest.mark.gpu

R, HK, W = 16, 2, 32


def grown(error, x, s, name):
    """The bound of rows x [n, heads, width] after one more rounding under the scales s [heads]."""
    s = s.astype(np.float64)[None, :, None]
    if name == "i8p":
        return error + s * (0.5 + 2.0 ** -14)
    return error + np.maximum(2.0 ** -4 * (np.abs(x) + error) * (1 + 2.0 ** -23), s * 2.0 ** -10) + s * 2.0 ** -14


SIZES = {
    "rising a little": 1.004 ** np.arange(R),      # every row has the page rounded anew, each time to one side
    "rising": 1.3 ** np.arange(R),
    "falling": 1.3 ** -np.arange(R),               # one rounding each
    "any": np.exp(np.random.default_rng(3).normal(size=R)),
    "one large": np.where(np.arange(R) == 9, 300.0, 1.0),
}


@pytest.mark.parametrize("name", ["i8p", "e4m3"])
@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("at_once", [1, 3, R])
def test_rows_are_near_what_was_appended(name, sizes, at_once):
    import torch

    g = gen(at_once)
    c = make_cache(g, name, 1, 2, R, HK, W, W)
    x = torch.rand(1, R, HK, W, generator=g, device="cuda") * 2 - 1
    x[..., 0] = 1.0  # every row's largest: its size
    x *= torch.tensor(SIZES[sizes], device="cuda").float()[None, :, None, None]
    hx, hy = host(x[0]).astype(np.float64), -host(x[0]).astype(np.float64)
    error = [np.zeros_like(hx), np.zeros_like(hx)]
    before, roundings, pg = None, 0, int(c.pages[0, 0])
    for first in range(0, R, at_once):
        n = min(at_once, R - first)
        rows = x[:, first:first + n].contiguous()
        c.append_dev(rows, -rows, i32([first]))
        scales = [host(s[pg]) for s in (c.ks, c.vs)]
        for z, y in enumerate((hx, hy)):
            upto = first + n
            again = grown(error[z][:first], y[:first], scales[z], name)
            if before is not None:  # heads whose scale stood still are as they were
                again = np.where((scales[z] != before[z])[None, :, None], again, error[z][:first])
            error[z][:first] = again
            error[z][first:upto] = grown(error[z][first:upto], y[first:upto], scales[z], name)
        roundings += before is not None and (scales[0] != before[0]).any()
        before = scales
        for got, y, e in zip(cache_rows(c, 0, np.arange(first + n)), (hx, hy), error):
            assert (np.abs(got - y[:first + n]) <= e[:first + n]).all(), first
    if at_once == 1:
        assert roundings == {"falling": 0, "one large": 1}.get(sizes, roundings) and (roundings == R - 1 or "rising" not in sizes)
