"""Timing cases of the operators around steps of several rows a stream (prompts
and drafted tokens) and of 8-bit paged caches with one scale a page and head,
through the framework's public entry points.

A case is a dict of plain values with a "kind":

  norm     norms of the query and key heads and their rotation in one pass
           (needle.qk_norm_rope_dev)
  quant    rows quantised as they are appended to an 8-bit paged cache with a
           scale for each page and key head (PagedKV.append_dev), and the pages
           that were written read back (PagedKV.read_dev)
  attend8  attention of one new token a stream over such a cache
           (PagedKV.attend_dev)
  rows     causal attention of many rows a stream over a paged cache of any
           type, with a window and first rows that stay visible
           (PagedKV.attend_rows_dev)
  verify   drafted tokens against the target's probabilities, and the log
           probabilities of the tokens that come of it (needle.verify_drafts_dev)

run(state) computes a case either by elementary torch operations (own false) or
by the framework's kernels (own true); exact(case, seed) gives the same values
in float64 from the definitions.
"""

import math

import torch

own = False

E4M3 = torch.float8_e4m3fn
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8, "e4m3": E4M3}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1, "e4m3": 1}
MOST = {"i8": 127.0, "e4m3": 448.0}  # the largest code


def listed():
    return [
        # One token of each of 256 decoding streams, float32 activations: all
        # launch latency.
        {"name": "norm_token_256", "kind": "norm", "batch": 256, "t": 1, "heads": 8, "kv_heads": 8, "width": 64,
         "type": "f32", "packed": False},
        # The prompts of 32 streams, of unequal lengths, straight out of one
        # product for queries, keys and values.
        {"name": "norm_prompt_32x448", "kind": "norm", "batch": 32, "t": 448, "heads": 16, "kv_heads": 4, "width": 128,
         "type": "bf16", "packed": True},
        # One token of each of 256 streams, most of them into a page that
        # others are in.
        {"name": "quant_token_256", "kind": "quant", "batch": 256, "t": 1, "kv_heads": 8, "qk": 64, "vd": 64,
         "io": "f32", "type": "i8", "cap": 448, "page_rows": 16},
        # The prompts of 32 streams, of unequal lengths.
        {"name": "quant_prompt_32x448", "kind": "quant", "batch": 32, "t": 448, "kv_heads": 8, "qk": 128, "vd": 128,
         "io": "bf16", "type": "e4m3", "cap": 512, "page_rows": 16},
        # 64 streams at different positions, int8 pages.
        {"name": "attend8_64_ragged", "kind": "attend8", "batch": 64, "heads": 8, "kv_heads": 2, "qk": 48, "vd": 64,
         "io": "f32", "type": "i8", "nk": 448, "page_rows": 16, "ragged": True},
        # Few streams with very long caches: half a GiB of codes.
        {"name": "attend8_long_65000", "kind": "attend8", "batch": 4, "heads": 32, "kv_heads": 8, "qk": 128, "vd": 128,
         "io": "bf16", "type": "e4m3", "nk": 65000, "page_rows": 64, "ragged": False},
        # Four drafted tokens of one stream over a short float16 cache, float32
        # queries like the decoder's activations: the smallest attention.
        {"name": "rows_draft_1x4", "kind": "rows", "batch": 1, "t": 4, "heads": 8, "kv_heads": 2, "qk": 48, "vd": 64,
         "io": "f32", "type": "f16", "nk": 200, "page_rows": 16, "window": 0, "sink": 0, "ragged": False},
        # Five drafted tokens of each of 32 streams over long e4m3 caches.
        {"name": "rows_draft_32x5", "kind": "rows", "batch": 32, "t": 5, "heads": 32, "kv_heads": 8, "qk": 128,
         "vd": 128, "io": "bf16", "type": "e4m3", "nk": 8000, "page_rows": 64, "window": 0, "sink": 0, "ragged": True},
        # Whole prompts: the largest products.
        {"name": "rows_prompt_8x2000", "kind": "rows", "batch": 8, "t": 2000, "heads": 16, "kv_heads": 4, "qk": 128,
         "vd": 128, "io": "bf16", "type": "bf16", "nk": 2000, "page_rows": 16, "window": 0, "sink": 0, "ragged": False},
        # Parts of long prompts behind what the cache holds, a window of 1024 and
        # the first rows, int8 pages, unequal lengths.
        {"name": "rows_window_4x1000", "kind": "rows", "batch": 4, "t": 1000, "heads": 16, "kv_heads": 4, "qk": 64,
         "vd": 64, "io": "f16", "type": "i8", "nk": 8000, "page_rows": 64, "window": 1024, "sink": 4, "ragged": True},
        # Four drafted tokens of one stream over the tied head's vocabulary.
        {"name": "verify_1x4", "kind": "verify", "batch": 1, "t": 4, "n": 8199, "type": "f32", "temperature": 1.0,
         "given": "logits"},
        # Eight of each of 64 streams over the benchmark's vocabulary.
        {"name": "verify_64x8", "kind": "verify", "batch": 64, "t": 8, "n": 16384, "type": "f32", "temperature": 0.7,
         "given": "logits"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


HEADS = [(8, 2, 48, 64), (8, 8, 64, 64), (8, 8, 64, 64), (16, 4, 128, 128), (32, 8, 128, 128), (6, 6, 48, 48),
         (12, 1, 64, 64), (5, 5, 80, 96)]


def draw(rng):
    kind = rng.choice(["norm", "quant", "attend8", "rows", "rows", "rows", "verify"])
    heads, kv_heads, qk, vd = rng.choice(HEADS)
    io = rng.choice(["f32", "f16", "bf16"])
    page_rows = rng.choice([1, 8, 16, 16, 64, 256])
    row = kv_heads * (qk + vd)
    if kind == "norm":
        t = 1 if rng.random() < 0.4 else _log_int(rng, 2, 2000)
        batch = _log_int(rng, 1, max(1, min(256, (30 << 20) // (t * (heads + kv_heads) * qk))))
        return {"kind": kind, "batch": batch, "t": t, "heads": heads, "kv_heads": kv_heads, "width": qk, "type": io,
                "packed": rng.random() < 0.5}
    if kind == "quant":
        t = 1 if rng.random() < 0.5 else _log_int(rng, 2, 448)
        cap = max(t, _log_int(rng, 16, 512))
        batch = _log_int(rng, 1, max(1, min(256, (14 << 20) // (max(t, page_rows) * row))))
        return {"kind": kind, "batch": batch, "t": t, "kv_heads": kv_heads, "qk": qk, "vd": vd, "io": io,
                "type": rng.choice(["i8", "e4m3"]), "cap": cap, "page_rows": page_rows}
    if kind == "attend8":
        batch = _log_int(rng, 1, 256)
        nk = _log_int(rng, 1, max(1, min(65000, (400 << 20) // (batch * row))))
        return {"kind": kind, "batch": batch, "heads": heads, "kv_heads": kv_heads, "qk": qk, "vd": vd, "io": io,
                "type": rng.choice(["i8", "e4m3"]), "nk": nk, "page_rows": page_rows, "ragged": rng.random() < 0.6}
    if kind == "rows":
        typ = rng.choice([io, io, "f16", "bf16", "f32", "i8", "e4m3"])
        t = _log_int(rng, 1, 16) if rng.random() < 0.4 else _log_int(rng, 17, 2000)
        nk = max(t, _log_int(rng, 1, 20000))
        # rows times keys: products in float32 cost more
        work = 8 * 2000 * 1000 * 16 * 128 // (8 if io == "f32" or typ == "f32" or SIZE[typ] == 2 and typ != io else 1)
        nk = max(t, min(nk, work // (t * heads * max(qk, vd)), (1 << 30) // (8 * row)))
        t = max(1, min(t, work // (nk * heads * max(qk, vd))))
        batch = _log_int(rng, 1, max(1, min(64, work // (t * nk * heads * max(qk, vd)), (1 << 30) // (8 * nk * row))))
        window = 0 if rng.random() < 0.4 else _log_int(rng, 1, 2 * nk)
        return {"kind": kind, "batch": batch, "t": t, "heads": heads, "kv_heads": kv_heads, "qk": qk, "vd": vd, "io": io,
                "type": typ, "nk": nk, "page_rows": page_rows, "window": window,
                "sink": rng.choice([0, 1, 4, 16, 100]) if window else 0, "ragged": rng.random() < 0.6}
    n = rng.choice([8199, 16384, _log_int(rng, 32, 150000)])
    t = _log_int(rng, 1, 16)
    batch = _log_int(rng, 1, max(1, min(256, 17_000_000 // (n * (2 * t + 1)))))
    return {"kind": kind, "batch": batch, "t": t, "n": n, "type": io, "temperature": rng.choice([0.0, 0.5, 0.7, 1.0, 1.3]),
            "given": rng.choice(["logits", "logits", "tokens"])}


# ---- inputs ---------------------------------------------------------------------


def _randn(g, shape, typ):
    return torch.randn(shape, generator=g, device="cuda").to(TYPES[typ])


def _zeros(shape, typ):
    return torch.zeros(shape, dtype=TYPES[typ], device="cuda")


def _lengths(g, n, most, ragged):
    """n lengths up to `most`; ragged: unequal ones, the first 0 (a padded slot) where there are several."""
    if not ragged:
        return torch.full((n,), most, dtype=torch.int32, device="cuda")
    ln = torch.randint(1, most + 1, (n,), generator=g, device="cuda", dtype=torch.int32)
    if n > 2:
        ln[0] = 0
        ln[1] = most
    return ln


def _cache_state(g, c, per):
    """A pool of pages of normal keys and values, and a shuffled page table of `per` pages a stream; 8-bit
    pools as codes with a scale for each page and key head."""
    s = {}
    pool_pages = c["batch"] * per
    for name, width in (("k", c["qk"]), ("v", c["vd"])):
        shape = (pool_pages, c["page_rows"], c["kv_heads"], width)
        x = torch.empty(shape, dtype=TYPES[c["type"]] if c["type"] in ("f16", "bf16") else torch.float32, device="cuda")
        x.normal_(generator=g)
        if c["type"] in MOST:
            s[name + "s"] = torch.empty(pool_pages, c["kv_heads"], device="cuda").uniform_(0.8, 1.6, generator=g) * (
                4 / MOST[c["type"]])
            x *= MOST[c["type"]] / 4
            x = x.round_().clamp_(-127, 127).to(torch.int8) if c["type"] == "i8" else x.clamp_(-448, 448).to(E4M3)
        s[name] = x
    perm = torch.randperm(pool_pages, generator=g, device="cuda")
    s["pages"] = perm.view(c["batch"], per).to(torch.int32).contiguous()
    return s


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": c}
    if c["kind"] == "norm":
        B, t, H, Hk, w = c["batch"], c["t"], c["heads"], c["kv_heads"], c["width"]
        if c["packed"]:  # one product's rows: queries, keys, values side by side
            x = _randn(g, (B, t, (H + 2 * Hk) * w), c["type"])
            s["q"] = x[..., :H * w].unflatten(-1, (H, w))
            s["k"] = x[..., H * w:(H + Hk) * w].unflatten(-1, (Hk, w))
        else:
            s["q"], s["k"] = _randn(g, (B, t, H, w), c["type"]), _randn(g, (B, t, Hk, w), c["type"])
        s["q_out"], s["k_out"] = _zeros((B, t, H, w), c["type"]), _zeros((B, t, Hk, w), c["type"])
        for name in ("q_gain", "k_gain"):
            s[name] = 1 + 0.2 * torch.randn(w, generator=g, device="cuda")
        positions = max(2 * t, 512)
        angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (
            -torch.arange(w // 2, device="cuda", dtype=torch.float64) / (w // 2))
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["pos"] = torch.randint(0, positions - t + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        s["n"] = _lengths(g, B, t, t > 1)
    elif c["kind"] == "quant":
        B, t, R = c["batch"], c["t"], c["page_rows"]
        s |= _cache_state(g, c, -(-c["cap"] // R))
        # rows of unequal size, as keys of different tokens are
        size = torch.exp(0.5 * torch.randn(B, t, 1, 1, generator=g, device="cuda"))
        s["k_rows"] = (size * torch.randn(B, t, c["kv_heads"], c["qk"], generator=g, device="cuda")).to(TYPES[c["io"]])
        s["v_rows"] = (size * torch.randn(B, t, c["kv_heads"], c["vd"], generator=g, device="cuda")).to(TYPES[c["io"]])
        s["n"] = _lengths(g, B, t, t > 1)
        s["pos"] = (torch.rand(B, generator=g, device="cuda") * (c["cap"] - t + 1)).to(torch.int32)
        # what is read back: from the first row of the page that the append begins in
        s["from"] = s["pos"] // R * R
        s["count"] = torch.where(s["n"] > 0, s["pos"] + s["n"] - s["from"], torch.zeros_like(s["n"]))
        s["k_back"] = _zeros((B, t + R - 1, c["kv_heads"], c["qk"]), c["io"])
        s["v_back"] = _zeros((B, t + R - 1, c["kv_heads"], c["vd"]), c["io"])
    elif c["kind"] == "attend8":
        s |= _cache_state(g, c, -(-c["nk"] // c["page_rows"]))
        s["q"] = _randn(g, (c["batch"], c["heads"], c["qk"]), c["io"])
        s["out"] = _zeros((c["batch"], c["heads"], c["vd"]), c["io"])
        s["scale"] = math.sqrt(c["qk"])
        s["spans"] = torch.zeros(c["batch"], 4, dtype=torch.int32, device="cuda")
        s["spans"][:, 3] = _lengths(g, c["batch"], c["nk"], c["ragged"])
    elif c["kind"] == "rows":
        B, t, nk = c["batch"], c["t"], c["nk"]
        s |= _cache_state(g, c, -(-nk // c["page_rows"]))
        s["q"] = _randn(g, (B, t, c["heads"], c["qk"]), c["io"])
        s["out"] = _zeros((B, t, c["heads"], c["vd"]), c["io"])
        s["scale"] = math.sqrt(c["qk"])
        s["n"] = _lengths(g, B, t, c["ragged"])
        # the rows' first position: what the cache holds before them
        held = torch.rand(B, generator=g, device="cuda") if c["ragged"] else torch.ones(B, device="cuda")
        s["pos"] = (held * (nk - t)).to(torch.int32)
    else:
        B, t, n = c["batch"], c["t"], c["n"]
        x = 3 * torch.randn(B, t + 1, n, generator=g, device="cuda")
        # the draft's model is near the target's; suppressed tokens in both
        y = x[:, :t] + 0.8 * torch.randn(B, t, n, generator=g, device="cuda")
        off = torch.rand(n, generator=g, device="cuda") < 0.05
        off[n // 2] = False
        s["target"] = x.masked_fill_(off, -math.inf).to(TYPES[c["type"]])
        draft = y.masked_fill_(off, -math.inf).to(TYPES[c["type"]])
        # what the draft's model chose: by its probabilities, or its likeliest
        if c["temperature"] > 0 and c["given"] == "logits":
            p = torch.softmax(draft.double() / c["temperature"], -1).cumsum(-1)
            u = torch.rand(B, t, 1, generator=g, device="cuda", dtype=torch.float64)
            d = (p <= u * p[..., -1:]).sum(-1).clamp_(max=n - 1)
        else:
            d = draft.float().argmax(-1)
        s["drafts"] = d.to(torch.int32)
        s["draft"] = draft if c["temperature"] > 0 and c["given"] == "logits" else None
        s["u"] = torch.rand(B, t, generator=g, device="cuda")
        s["u_next"] = torch.rand(B, generator=g, device="cuda")
        s["n"] = _lengths(g, B, t, B > 2)
        s["accepted"] = torch.zeros(B, dtype=torch.int32, device="cuda")
        s["tokens"] = torch.zeros(B, t + 1, dtype=torch.int32, device="cuda")
        s["lp"] = torch.zeros(B, t + 1, device="cuda")
    return s


# ---- the framework's kernels ------------------------------------------------------


def _needle():
    import importlib

    return importlib.import_module("go-whistle_amd").needle


def _cache(s):
    """The cache's handle, made once as a user's program makes it with its pool."""
    if "cache" not in s:
        s["cache"] = _needle().PagedKV(s["k"], s["v"], s["pages"], s.get("ks"), s.get("vs"))
    return s["cache"]


def _run_own(s):
    c = s["case"]
    if c["kind"] == "norm":
        _needle().qk_norm_rope_dev(s["q_out"], s["k_out"], s["q"], s["k"], q_gain=s["q_gain"], k_gain=s["k_gain"],
                                   rope=(s["cos"], s["sin"]), pos=s["pos"], rows=s["n"])
    elif c["kind"] == "quant":
        _cache(s).append_dev(s["k_rows"], s["v_rows"], s["pos"], rows=s["n"], cap=c["cap"])
        _cache(s).read_dev(s["k_back"], s["v_back"], s["from"], rows=s["count"])
    elif c["kind"] == "attend8":
        _cache(s).attend_dev(s["out"], s["q"], s["spans"], c["nk"], s["scale"])
    elif c["kind"] == "rows":
        _cache(s).attend_rows_dev(s["out"], s["q"], s["pos"], s["scale"], rows=s["n"], nk_max=c["nk"],
                                  window=c["window"], sink=c["sink"])
    else:
        _needle().verify_drafts_dev(s["accepted"], s["tokens"], s["target"], s["drafts"], draft=s["draft"], u=s["u"],
                                    u_next=s["u_next"], drafted=s["n"], temperature=c["temperature"], lp=s["lp"])


# ---- the plain forms ----------------------------------------------------------------


def _plain_norm(s):
    c = s["case"]
    t, half = c["t"], c["width"] // 2
    i = torch.arange(t, device="cuda")
    at = s["pos"].long()[:, None] + i
    cos, sin = s["cos"][at][:, :, None], s["sin"][at][:, :, None]
    live = (i < s["n"][:, None])[..., None, None]
    for name in ("q", "k"):
        x = s[name].float()
        x = s[name + "_gain"] * (x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6))
        a, b = x[..., :half], x[..., half:]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(s[name].dtype)
        s[name + "_out"].copy_(torch.where(live, y, s[name + "_out"]))


def _codes(x, typ):
    """The 8-bit codes of x, whose values are within the type's."""
    return torch.round(x).clamp(-127, 127).to(torch.int8) if typ == "i8" else x.clamp(-448, 448).to(E4M3)


def _plain_quant(s):
    """Page by page: the largest of the scale of the rows before and the new rows' own; every row's codes under it."""
    c, R = s["case"], s["case"]["page_rows"]
    most = MOST[c["type"]]
    dead = s["n"][:, None, None] == 0
    # a page of the table at a time, as rows [batch, pages, R]; a stream's new rows are [pos, pos + n)
    touched = -(-(c["t"] + R - 1) // R)
    page = (s["pos"] // R).long()[:, None] + torch.arange(touched, device="cuda")  # [B, P]
    row = page[..., None] * R + torch.arange(R, device="cuda")  # [B, P, R]
    i = row - s["pos"].long()[:, None, None]
    new = (i >= 0) & (i < s["n"].long()[:, None, None])
    old = (i < 0) & ~dead
    b, p = torch.nonzero(new.any(-1), as_tuple=True)
    at = s["pages"].long()[b, page[b, p]]
    new, old, i = new[b, p][..., None, None], old[b, p][..., None, None], i[b, p].clamp(0, c["t"] - 1)
    for name in ("k", "v"):
        x = s[name + "_rows"][b[:, None], i].float()  # [N, R, Hk, width]
        sc = torch.where(old.any(1), s[name + "s"][at][..., None], torch.zeros(1, device="cuda"))[:, :, 0]  # [N, Hk]
        had = sc
        top = torch.where(new, x.abs(), torch.zeros_like(x)).amax((1, 3))
        sc = torch.maximum(sc, top / most)
        div = torch.where(sc > 0, sc, torch.ones_like(sc))[:, None, :, None]
        held = s[name][at]
        again = _codes(held.float() * had[:, None, :, None] / div, c["type"])
        again = torch.where((had == sc)[:, None, :, None], held.float(), again.float())
        y = torch.where(new, _codes(x / div, c["type"]).float(), torch.where(old, again, held.float()))
        s[name][at] = y.to(TYPES[c["type"]])
        s[name + "s"][at] = sc
    # read back
    j = torch.arange(c["t"] + R - 1, device="cuda")
    b, j = torch.nonzero(j[None, :] < s["count"][:, None], as_tuple=True)
    r = s["from"].long()[b] + j
    at = s["pages"].long()[b, r // R]
    for name in ("k", "v"):
        x = s[name][at, r % R].float() * s[name + "s"][at][..., None]
        s[name + "_back"][b, j] = x.to(TYPES[c["io"]])


def _softmax_av(logits, mask, v):
    """softmax of the unmasked logits times v, 0 for rows whose mask leaves nothing."""
    logits = torch.where(mask, logits, torch.full_like(logits, -math.inf))
    m = logits.amax(-1, keepdim=True)
    p = torch.where(mask, torch.exp(logits - torch.where(m == -math.inf, torch.zeros_like(m), m)), torch.zeros_like(logits))
    d = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(d == 0, torch.ones_like(d), d)


def _cache_rows(s, name, pages):
    """The rows of those pages of a cache, [.., rows, kv_heads, width] in float32."""
    x = s[name][pages].float()
    if name + "s" in s:
        x = x * s[name + "s"][pages][..., None, :, None]
    return x.flatten(-4, -3)


def _plain_attend8(s):
    c = s["case"]
    B, nk, H, Hk = c["batch"], c["nk"], c["heads"], c["kv_heads"]
    k, v = (_cache_rows(s, name, s["pages"].long())[:, :nk] for name in ("k", "v"))
    q = s["q"].float().view(B, Hk, H // Hk, c["qk"])
    logits = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) / s["scale"]
    mask = torch.arange(nk, device="cuda") < s["spans"][:, 3:]
    o = _softmax_av(logits, mask[:, None, None, :].expand_as(logits), v.permute(0, 2, 1, 3).contiguous())
    s["out"].copy_(o.reshape(B, H, c["vd"]))


def _plain_rows(s):
    c = s["case"]
    t, nk, H, Hk = c["t"], c["nk"], c["heads"], c["kv_heads"]
    j, i = torch.arange(nk, device="cuda"), torch.arange(t, device="cuda")
    for b in range(c["batch"]):
        k, v = (_cache_rows(s, name, s["pages"][b].long())[:nk] for name in ("k", "v"))
        q = s["q"][b].float().view(t, Hk, H // Hk, c["qk"]).permute(1, 2, 0, 3).reshape(Hk, -1, c["qk"])
        logits = torch.matmul(q, k.permute(1, 2, 0).contiguous()) / s["scale"]
        at = (s["pos"][b] + i)[:, None]
        mask = j <= at
        if c["window"]:
            mask &= (j < c["sink"]) | (j > at - c["window"])
        mask = mask.repeat(H // Hk, 1).expand_as(logits)
        o = _softmax_av(logits, mask, v.permute(1, 0, 2).contiguous())
        o = o.view(Hk, H // Hk, t, c["vd"]).permute(2, 0, 1, 3).reshape(t, H, c["vd"])
        live = (i < s["n"][b])[:, None, None]
        s["out"][b] = torch.where(live, o.to(s["out"].dtype), s["out"][b])


def _plain_verify(s):
    """In float64: a running sum's next value may lie next to the random number."""
    c = s["case"]
    B, t, n = c["batch"], c["t"], c["n"]
    b, i = torch.arange(B, device="cuda"), torch.arange(t, device="cuda")
    d, drafted = s["drafts"].long(), s["n"].long()
    if c["temperature"] == 0:
        best = s["target"].float().argmax(-1)
        ok = best[:, :t] == d
    else:
        p = torch.softmax(s["target"].double() / c["temperature"], -1)
        pd = p[:, :t].gather(-1, d[..., None])[..., 0]
        if s["draft"] is None:
            qd = torch.ones_like(pd)
        else:
            q = torch.softmax(s["draft"].double() / c["temperature"], -1)
            qd = q.gather(-1, d[..., None])[..., 0]
        ok = s["u"].double() * qd < pd
    ok &= i < drafted[:, None]
    a = ok.long().cumprod(-1).sum(-1)
    if c["temperature"] == 0:
        token = best[b, a]
    else:
        w = p[b, a]
        at = a.clamp(max=t - 1)
        if s["draft"] is None:
            less = torch.zeros_like(w).scatter_(-1, d[b, at][:, None], math.inf)
        else:
            less = q[b, at]
        w = torch.where((a < drafted)[:, None], (w - less).clamp(min=0), w)
        run_ = w.cumsum(-1)
        token = (run_ <= s["u_next"].double()[:, None] * run_[:, -1:]).sum(-1)
    out = torch.where(torch.arange(t + 1, device="cuda") < a[:, None], torch.cat([d, d[:, :1]], -1), -1)
    out[b, a] = token
    s["accepted"].copy_(a)
    s["tokens"].copy_(out)
    x = s["target"].double() / (c["temperature"] or 1.0)
    lp = x.gather(-1, out.clamp(min=0)[..., None])[..., 0] - torch.logsumexp(x, -1)
    s["lp"].copy_(torch.where(out >= 0, lp, torch.zeros_like(lp)))


PLAIN = {"norm": _plain_norm, "quant": _plain_quant, "attend8": _plain_attend8, "rows": _plain_rows,
         "verify": _plain_verify}
OUTPUTS = {"norm": ("q_out", "k_out"), "quant": ("k_back", "v_back"), "attend8": ("out",), "rows": ("out",),
           "verify": ("accepted", "tokens", "lp")}


def run(state):
    kind = state["case"]["kind"]
    if own:
        _run_own(state)
    else:
        PLAIN[kind](state)
    return [state[name] for name in OUTPUTS[kind]]


# ---- what a pass cannot do without ---------------------------------------------------


def work(case):
    """Bytes read and written once, and operations; unequal lengths count with their mean."""
    c = case
    if c["kind"] == "norm":
        part = 1 if c["t"] == 1 else 0.5
        values = part * c["batch"] * c["t"] * (c["heads"] + c["kv_heads"]) * c["width"]
        return {"bytes": values * 2 * SIZE[c["type"]] + part * c["batch"] * c["t"] * c["width"] * 4, "flops": 8 * values}
    if c["kind"] == "quant":
        new = c["batch"] * (c["t"] if c["t"] == 1 else (c["t"] + 1) / 2)
        back = new + c["batch"] * (c["page_rows"] - 1) / 2
        values = c["kv_heads"] * (c["qk"] + c["vd"])
        return {"bytes": values * (new * (SIZE[c["io"]] + 1) + back * (1 + SIZE[c["io"]])), "flops": 0}
    if c["kind"] == "attend8":
        keys = c["batch"] * (c["nk"] if not c["ragged"] else (c["nk"] + 1) / 2)
        ends = c["batch"] * c["heads"] * (c["qk"] + c["vd"]) * SIZE[c["io"]]
        return {"bytes": keys * c["kv_heads"] * (c["qk"] + c["vd"] + 8 / c["page_rows"]) + ends,
                "flops": 2 * keys * c["heads"] * (c["qk"] + c["vd"])}
    if c["kind"] == "rows":
        n = (c["t"] + 1) / 2 if c["ragged"] else c["t"]
        pos = (c["nk"] - c["t"]) * (0.5 if c["ragged"] else 1)
        pairs, low = 0, 0
        for i in range(int(n)):
            at = pos + i + 1
            pairs += at if not c["window"] else min(at, c["window"] + min(c["sink"], max(0, at - c["window"])))
        if c["window"]:
            low = max(0, pos + 1 - c["window"] - c["sink"])
        keys = pos + n - low
        scales = 8 / c["page_rows"] if c["type"] in MOST else 0
        return {"bytes": c["batch"] * (keys * c["kv_heads"] * ((c["qk"] + c["vd"]) * SIZE[c["type"]] + scales) +
                                       n * c["heads"] * (c["qk"] + c["vd"]) * SIZE[c["io"]]),
                "flops": 2 * c["batch"] * pairs * c["heads"] * (c["qk"] + c["vd"])}
    rows = c["batch"] * (c["t"] + 1 + (c["t"] if c["given"] == "logits" and c["temperature"] > 0 else 0))
    return {"bytes": rows * c["n"] * SIZE[c["type"]] + 12 * c["batch"] * (c["t"] + 1), "flops": 4 * rows * c["n"]}


# ---- the definitions in float64 --------------------------------------------------------


def _exact_norm(s):
    c = s["case"]
    outs = []
    for name in ("q", "k"):
        y = s[name + "_out"].double()
        for b, (n, p) in enumerate(zip(s["n"].tolist(), s["pos"].tolist())):
            x = s[name][b, :n].double()
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * s[name + "_gain"].double()
            z = torch.complex(x[..., :c["width"] // 2], x[..., c["width"] // 2:])
            z = z * torch.complex(s["cos"][p:p + n].double(), s["sin"][p:p + n].double())[:, None]
            y[b, :n] = torch.cat([z.real, z.imag], -1)
        outs.append(y)
    return outs


def _nearest(x, typ):
    """The nearest value that the type holds, ties to the even one."""
    if typ == "i8":
        return torch.round(x)
    exponent = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -30))).clamp(min=-6)
    step = torch.exp2(exponent - 3)
    return torch.round(x / step) * step


def _exact_quant(s):
    """A page's scale is the larger of float32(max |x| / most) and, where it has rows before, theirs; a row's codes
    are those nearest to float32(x / scale), of rows that the page held x their float32 values."""
    c, R = s["case"], s["case"]["page_rows"]
    outs = []
    for name in ("k", "v"):
        back = s[name + "_back"].double()
        for b, (n, p) in enumerate(zip(s["n"].tolist(), s["pos"].tolist())):
            at = p
            while at < p + n:
                first, end = at // R * R, min(at // R * R + R, p + n)
                page = int(s["pages"][b, at // R])
                x = s[name + "_rows"][b, at - p:end - p].double()
                sc = (x.abs().amax((0, 2)) / MOST[c["type"]]).float().double()
                if at > first:
                    had = s[name + "s"][page].double()
                    sc = torch.maximum(sc, had)
                    held = (s[name][page, :at - first].double() * had[:, None]).float().double()
                    kept = (had == sc)[:, None]
                    again = _nearest((held / sc[:, None]).float().double(), c["type"]) * sc[:, None]
                    back[b, first - p // R * R:at - p // R * R] = torch.where(
                        kept, s[name][page, :at - first].double() * had[:, None], again)
                y = _nearest((x / sc[:, None]).float().double(), c["type"]) * sc[:, None]
                back[b, at - p // R * R:end - p // R * R] = y
                at = end
        outs.append(back)
    return outs


def _exact_key_rows(s, b, name, lo, hi):
    r = torch.arange(lo, hi, device="cuda")
    page, R = s["pages"].long()[b, r // s["case"]["page_rows"]], s["case"]["page_rows"]
    x = s[name][page, r % R].double()
    return x * s[name + "s"][page].double()[..., None] if name + "s" in s else x


def _exact_attend8(s):
    c = s["case"]
    G = c["heads"] // c["kv_heads"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["spans"][:, 3].tolist()):
        if not n:
            continue
        k, v = (_exact_key_rows(s, b, name, 0, n) for name in ("k", "v"))
        for h in range(c["kv_heads"]):
            w = torch.softmax(s["q"][b, h * G:(h + 1) * G].double() @ k[:, h].t().contiguous() / s["scale"], -1)
            out[b, h * G:(h + 1) * G] = w @ v[:, h].contiguous()
    return [out]


def _exact_rows(s):
    c = s["case"]
    G = c["heads"] // c["kv_heads"]
    out = s["out"].double()
    for b, (n, p) in enumerate(zip(s["n"].tolist(), s["pos"].tolist())):
        if not n:
            continue
        k, v = (_exact_key_rows(s, b, name, 0, p + n) for name in ("k", "v"))
        back = p + torch.arange(n, device="cuda")[:, None] - torch.arange(p + n, device="cuda")  # rows behind the query
        hidden = back < 0
        if c["window"]:
            hidden |= (back >= c["window"]) & (torch.arange(p + n, device="cuda") >= c["sink"])
        for h in range(c["heads"]):
            x = s["q"][b, :n, h].double() @ k[:, h // G].t().contiguous() / s["scale"]
            out[b, :n, h] = torch.softmax(x.masked_fill_(hidden, -math.inf), -1) @ v[:, h // G].contiguous()
    return [out]


def _exact_verify(s):
    """Stream by stream; the whole numbers are no computed ones, and the log probabilities go by them."""
    c = s["case"]
    T = c["temperature"] or 1.0
    lp = torch.zeros(s["lp"].shape, dtype=torch.float64, device="cuda")
    drafts, counts, u, u_next = (s[name].tolist() for name in ("drafts", "n", "u", "u_next"))
    for b, count in enumerate(counts):
        logp = torch.log_softmax(s["target"][b].double() / T, -1)
        p, tokens = logp.exp(), drafts[b][:count]
        q = None if s["draft"] is None else torch.softmax(s["draft"][b].double() / T, -1)
        at = torch.arange(count, device="cuda")
        pd = p[at, tokens].tolist()
        qd = [1.0] * count if q is None else q[at, tokens].tolist()
        best = p.argmax(-1).tolist()
        a = 0
        while a < count and (best[a] == tokens[a] if c["temperature"] == 0 else u[b][a] * qd[a] < pd[a]):
            a += 1
        w = p[a].clone()
        if a < count and q is not None:
            w = torch.relu(w - q[a])
        elif a < count:
            w[tokens[a]] = 0
        total = torch.cumsum(w, 0)
        last = best[a] if c["temperature"] == 0 else int(torch.searchsorted(total, u_next[b] * total[-1:], right=True))
        lp[b, :a + 1] = logp[torch.arange(a + 1, device="cuda"), tokens[:a] + [last]]
    return [None, None, lp]


EXACT = {"norm": _exact_norm, "quant": _exact_quant, "attend8": _exact_attend8, "rows": _exact_rows,
         "verify": _exact_verify}


def exact(case, seed):
    return EXACT[case["kind"]](prepare(case, seed))
