"""Ends of the ranges of the paged caches' calls: no keys, infinite keys, pools
past 2^32 bytes, evictions of very long lists."""

import numpy as np
import pytest

from go_whistle_amd import needle
from serve_ref import attend64, host, keep_rows, make_pool, pool_rows

pytestmark = pytest.mark.gpu


def gen(seed):
    import torch

    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def i32(x):
    import torch

    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("group", [1, 3, 20, 40])
@pytest.mark.parametrize("name", ["float32", "bfloat16", "i8"])
def test_no_keys_with_weights(group, name):
    import torch

    k, v, ks, vs = make_pool(gen(1), 4, 16, 2, 64, 64, name)
    c = needle.PagedKV(k, v, i32([[0, 1], [2, 3]]), ks, vs)
    q = torch.randn(2, 2 * group, 64, generator=gen(2), device="cuda")
    out, acc = torch.full_like(q, 3.0), torch.full((2, 2, 5), 7.0, device="cuda")
    c.attend_dev(out, q, torch.zeros(2, 4, dtype=torch.int32, device="cuda"), 0, 8.0, acc_out=acc)
    torch.cuda.synchronize()
    assert (out == 0).all() and (acc == 7).all()
