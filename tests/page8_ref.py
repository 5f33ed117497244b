"""Caches of any type for the tests of the operators around steps of several
rows, with their plain forms: 8-bit pages with one scale a page and head in
exact steps of float32 arithmetic, attention of many rows in float64.

The attention's bound is serve_ref.attend64's for float32 products. Where the
products are of 16 bits the softmax weights take part as two parts of the
values' type (float16 where the cache is of that type, else bfloat16): off by
2^-22 and 2^-16 of the weight (in float16 at least 2^-32 of the largest weight,
which the sum of n weights is n times at most), that is `extra` of sum w |v|."""

import math

import numpy as np

from serve_ref import U, attend64, half_ulp, host

MOST = {"i8p": 127.0, "e4m3": 448.0}
CACHES = ["float32", "float16", "bfloat16", "i8", "i8p", "e4m3"]
FLOATS = ["float32", "float16", "bfloat16"]


def gen(seed):
    import torch

    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def i32(x):
    import torch

    return torch.tensor(x, dtype=torch.int32, device="cuda")


def nearest(x, name):
    """The nearest value of a code type to float64 x, ties to the even one."""
    if name != "e4m3":
        return np.rint(x)
    e = np.maximum(np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -30))), -6)
    step = np.exp2(e - 3)
    return np.rint(x / step) * step


def make_cache(g, name, streams, per, page_rows, Hk, qk, vd, extra_pages=0):
    """(PagedKV, k, v): a cache of normal values on shuffled pages."""
    import torch

    from go_whistle_amd import needle

    pages = streams * per + extra_pages
    t = []
    for w in (qk, vd):
        x = torch.randn(pages, page_rows, Hk, w, generator=g, device="cuda")
        if name == "i8":
            t.append((torch.clamp((x * 40).round(), -127, 127).to(torch.int8),
                      torch.rand(pages, page_rows, Hk, generator=g, device="cuda") * 0.03 + 0.01))
        elif name in MOST:
            s = (torch.rand(pages, Hk, generator=g, device="cuda") + 0.5) * (4 / MOST[name])
            x = torch.clamp(x * (MOST[name] / 4), -MOST[name], MOST[name])
            t.append((x.round().to(torch.int8) if name == "i8p" else x.to(torch.float8_e4m3fn), s))
        else:
            t.append((x.to(getattr(torch, name)), None))
    table = torch.randperm(pages, generator=g, device="cuda")[:streams * per].view(streams, per).int().contiguous()
    return needle.PagedKV(t[0][0], t[1][0], table, t[0][1], t[1][1])


def widened(t):
    """A device tensor's values in float64 on the host."""
    import torch

    return host(t.float() if t.dtype == torch.float8_e4m3fn else t).astype(np.float64)


def cache_rows(c, b, rows):
    """Keys and values of a stream's rows, float64 [n, kv_heads, width]."""
    R = c.k.shape[1]
    pg = c.pages[b].cpu().numpy().astype(np.int64)[np.asarray(rows) // R]
    pg = np.where((pg >= 0) & (pg < c.k.shape[0]), pg, 0)
    import torch

    at, dev = torch.as_tensor(np.asarray(rows) % R, device="cuda"), torch.as_tensor(pg, device="cuda")
    out = []
    for x, s in ((c.k, c.ks), (c.v, c.vs)):
        y = widened(x[dev, at])
        if s is not None:
            y = y * host(s[dev, at] if s.dim() == 3 else s[dev]).astype(np.float64)[..., None]
        out.append(y)
    return out


def visible(p, window, sink):
    """The rows that the one at position p attends."""
    j = np.arange(p + 1)
    return j if not window else j[(j > p - window) | (j < sink)]


def weight_error(q_name, cache_name, n):
    """What the softmax weights' parts add to the bound, relative to sum w |v|."""
    if q_name == "float32" or cache_name == "float32" or (cache_name in FLOATS and cache_name != q_name):
        return 0.0
    return 2.0 ** -22 + n * 2.0 ** -32 if cache_name == "float16" else 2.0 ** -16


def check_rows(c, cache_name, out, before, q, pos, rows, nk_max, window, sink, scale, sample, seed=0):
    """Rows of every stream (`sample` of them, with their first and last) against
    float64; the others as they were."""
    B, t, H, _ = q.shape
    G = H // c.kv_heads
    ho, hb, hq = (host(x).astype(np.float64) for x in (out, before, q))
    name = str(q.dtype).split(".")[1]
    pick = np.random.default_rng(seed)
    for b in range(B):
        n = t if rows is None else int(rows[b])
        if not 0 < n <= t or pos[b] < 0 or pos[b] + n > nk_max:
            n = 0
        assert np.array_equal(ho[b, n:], hb[b, n:], equal_nan=True), b
        if not n:
            continue
        k, v = cache_rows(c, b, np.arange(pos[b] + n))
        for i in range(n) if n <= sample else sorted({0, n - 1, *pick.integers(0, n, sample).tolist()}):
            j = visible(pos[b] + i, window, sink)
            for h in range(H) if H <= 2 else sorted({0, H - 1, int(pick.integers(0, H))}):
                o, bound, w, _ = attend64(hq[b, i, h], k[j, h // G], v[j, h // G], scale, q.dtype)
                bound = bound + (1 + half_ulp(q.dtype)) * weight_error(name, cache_name, len(j)) * (w @ np.abs(v[j, h // G]))
                err = np.abs(ho[b, i, h] - o)
                assert (err <= bound).all(), (b, i, h, (err / np.maximum(bound, 1e-300)).max())


def append_pages(state, scales, x, pos, n, R, name):
    """One stream's rows x [t, heads, width] (float32 values) appended: `state`
    holds its codes' values [rows, heads, width], `scales` [pages, heads]; in place."""
    most = np.float32(MOST[name])
    at = pos
    while at < pos + n:
        first = at // R * R
        end = min(first + R, pos + n)
        y = x[at - pos:end - pos]
        size = np.where(np.isfinite(y), np.abs(y), np.float32(0))
        s = (size.max((0, 2)) / most).astype(np.float32)
        had = scales[at // R].copy() if at > first else np.zeros_like(s)
        s = np.maximum(s, had)
        div = np.where(s > 0, s, np.float32(1))

        def codes(z):
            r = (z / div[None, :, None]).astype(np.float32).astype(np.float64)
            r = np.where(np.isnan(r), 0.0 if name == "i8p" else np.nan, np.clip(r, -float(most), float(most)))
            return nearest(r, name)

        with np.errstate(all="ignore"):
            again = codes((state[first:at].astype(np.float32) * had[None, :, None]).astype(np.float32))
            state[first:at] = np.where((s != had)[None, :, None], again, state[first:at])
            state[at:end] = codes(y)
        scales[at // R] = s
        at = end


def norm_rope64(x, gain, cos, sin, turn):
    """Float64 norm of heads [.., width] and their rotation (turn: rows that are rotated), and
    the largest error of float32 arithmetic: with u = 2^-24 the quotient is off by 8 u (the sum's
    n u halved by the root, with n <= 256 in float32: n / 2 u more), a rotated value by 4 u of |a c| + |b s|."""
    x = x.astype(np.float64)
    w = x.shape[-1]
    rel = 0.0
    if gain is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6) * gain.astype(np.float64)
        rel = (8 + w / 2) * U
    mag = np.abs(x)
    a, b = x[..., :w // 2], x[..., w // 2:]
    y = np.concatenate([a * cos - b * sin, b * cos + a * sin], -1)
    ma, mb = mag[..., :w // 2], mag[..., w // 2:]
    ac, asn = np.abs(cos), np.abs(sin)
    m = np.concatenate([ma * ac + mb * asn, mb * ac + ma * asn], -1)
    y, m = np.where(turn, y, x), np.where(turn, m, mag)
    return y, m * (rel + 4 * U)


def softmax64(x, temperature):
    """p of a row of logits, or None for a row that has none."""
    x = x.astype(np.float64)
    if np.isnan(x).any() or (x == np.inf).any() or (x == -np.inf).all():
        return None
    p = np.exp((x - x.max()) / temperature)
    return p / p.sum()


def verify64(target, drafts, draft, u, u_next, count, temperature):
    """One stream: accepted, tokens [t + 1], log probabilities [t + 1]."""
    t, n = len(drafts), target.shape[1]
    T = temperature or 1.0
    count = min(max(count, 0), t)
    tokens, lp = np.full(t + 1, -1), np.zeros(t + 1)
    a = 0
    while True:
        p = softmax64(target[a], T)
        if a == count:
            break
        d = int(drafts[a])
        ok = p is not None and 0 <= d < n
        q = None
        if ok and temperature == 0:
            ok = int(np.argmax(target[a])) == d
        elif ok:
            q = None if draft is None else softmax64(draft[a], T)
            qd = 1.0 if draft is None else np.nan if q is None else q[d]
            ok = float(u[a]) * qd < p[d]
        if not ok:
            break
        tokens[a], lp[a] = d, math.log(p[d]) if p[d] > 0 else -np.inf
        a += 1
    if p is not None:
        if temperature == 0:
            token = int(np.argmax(target[a]))
        else:
            w = p.copy()
            if a < count:
                if draft is None:
                    if 0 <= drafts[a] < n:
                        w[drafts[a]] = 0
                else:
                    q = softmax64(draft[a], T)
                    w = np.maximum(p - q, 0) if q is not None else np.zeros(n)
            if not w.sum() > 0:
                w = p
            c = np.cumsum(w)
            over = np.nonzero((c > float(u_next) * c[-1]) & (w > 0))[0]
            token = int(over[0]) if len(over) else int(np.nonzero(w > 0)[0][-1])
        tokens[a] = token
        with np.errstate(divide="ignore"):
            lp[a] = np.log(p[token])
    return a, tokens, lp
