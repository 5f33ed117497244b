"""Plain float64 forms of the serving operators (paged caches, attention over
them, eviction, cross-attention, log probabilities) and the error bounds of
their float32 arithmetic, for the tests.

Bounds, with u = 2^-24 and round(t) = finfo(t).eps / 2 the largest relative
error of one rounding to t:
  a logit is a dot of qk products and a few scalings of it, so it is off by
  at most (qk + 6) u sum |q k| / scale, and its distance to the maximum by u
  times its size more; the weight 2^x is off by twice that (numerator and
  sum) plus 2^-21 for the exponent function; the sums of n terms add n u
  each; so an output is off by at most
      sum w |v| (4 (qk + 8) u A + 8 u L + 2 n u + 2^-20)
  with A the largest sum |q k| / scale and L the largest |logit|, plus its
  own rounding to the output's type. Kernels that round the weights to a
  16-bit type p before the second product add round(p) of sum w |v|."""

import numpy as np

U = 2.0 ** -24


def half_ulp(dtype):
    import torch

    return torch.finfo(dtype).eps / 2


def attend64(q, k, v, scale, dtype, p_type=None):
    """One query head: out, its bound, the weights and theirs."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    vd, n = v.shape[1], k.shape[0]
    if n == 0:
        z = np.zeros(vd)
        return z, z, np.zeros(0), np.zeros(0)
    lg = k @ q / scale
    w = np.exp(lg - lg.max())
    w /= w.sum()
    a = (np.abs(k) @ np.abs(q)).max() / abs(scale)
    rel = 4 * (q.size + 8) * U * a + 8 * U * np.abs(lg).max() + 2 * n * U + 2.0 ** -20
    o, mag = w @ v, w @ np.abs(v)
    b = mag * (rel + (half_ulp(p_type) if p_type is not None else 0.0))
    import torch

    # the smallest subnormal step of the output's type, for results near 0
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    return o, b + half_ulp(dtype) * (np.abs(o) + b) + tiny, w, w * rel


def rows_of(spans):
    lo0, hi0, lo1, hi1 = (int(x) for x in spans)
    return np.concatenate([np.arange(lo0, hi0), np.arange(lo1, hi1)]).astype(np.int64)


def pool_rows(pool, scales, pages, rows, page_rows):
    """The values of a stream's rows [n, kv_heads, width], in float64."""
    pg, at = np.asarray(pages)[rows // page_rows], rows % page_rows
    pg = np.where((pg >= 0) & (pg < pool.shape[0]), pg, 0)
    x = pool[pg, at].astype(np.float64)
    return x * scales[pg, at].astype(np.float64)[..., None] if scales is not None else x


def keep_rows(acc, n, keep, sink, recent):
    """The rows kv_evict_paged_dev keeps of one key head's n."""
    w = np.asarray(acc[:n], np.float64).copy()
    w[np.isnan(w)] = -np.inf
    held = (np.arange(n) < sink) | (np.arange(n) >= n - recent)
    # held rows first, then the larger weight (a NaN the least), then the lower row
    nan = np.isnan(np.asarray(acc[:n], np.float64))
    order = sorted(range(n), key=lambda j: (not held[j], bool(nan[j]), -w[j], j))
    return np.array(sorted(order[:keep]), np.int64)


def host(t):
    """A tensor's values as a numpy array (bfloat16 widened)."""
    import torch

    t = t.detach().cpu()
    return (t.float() if t.dtype in (torch.bfloat16, torch.float16) else t).numpy()


def make_pool(g, pages, page_rows, kv_heads, qk, vd, name):
    """Device pools of a type: (k, v, ks, vs)."""
    import torch

    out = []
    for w in (qk, vd):
        x = torch.randn(pages, page_rows, kv_heads, w, generator=g, device="cuda")
        if name == "i8":
            out.append((torch.clamp((x * 40).round(), -127, 127).to(torch.int8),
                        torch.rand(pages, page_rows, kv_heads, generator=g, device="cuda") * 0.03 + 0.01))
        else:
            out.append((x.to(getattr(torch, name)), None))
    return out[0][0], out[1][0], out[0][1], out[1][1]
