"""Timing cases of the float and int8 serving operators around a decode step,
through the framework's public entry points.

A case is a dict of plain values with a "kind":

  append    rows of keys and values appended to a paged cache (PagedKV.append_dev):
            one token of many streams, or whole prompts
  attend    attention of one new token a stream over a paged cache of any length,
            with the accumulated attention weights on request (PagedKV.attend_dev)
  evict     eviction from a paged cache by those weights (PagedKV.evict_dev)
  cross     attention of a step's or a prompt's rows to encoder states of other
            lengths (needle.cross_attend_dev)
  logprobs  log probabilities of given tokens, entropy and the top alternatives
            (needle.logprobs_dev)

run(state) computes a case either by elementary torch operations in float32
(own false) or by the framework's kernels (own true); exact(case, seed) gives the
same values in float64 from the definitions.
"""

import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}


def listed():
    return [
        # One token of each of 256 decoding streams into their paged caches:
        # all launch latency.
        {"name": "append_token_256", "kind": "append", "batch": 256, "t": 1, "kv_heads": 8, "qk": 64, "vd": 64,
         "io": "f32", "type": "bf16", "cap": 448, "page_rows": 16},
        # The prompts of 32 streams, of unequal lengths, appended at once.
        {"name": "append_prompt_32x448", "kind": "append", "batch": 32, "t": 448, "kv_heads": 8, "qk": 128, "vd": 128,
         "io": "f32", "type": "f16", "cap": 512, "page_rows": 16},
        # One stream's decode step over a grouped-query int8 cache (8 heads of
        # 48 over 2 key heads): the smallest attention.
        {"name": "attend_one_200", "kind": "attend", "batch": 1, "heads": 8, "kv_heads": 2, "qk": 48, "vd": 64,
         "io": "f32", "type": "i8", "nk": 200, "page_rows": 16, "spans": "full", "acc": False},
        # 256 streams at different positions of an int8 cache, their weights
        # accumulated for the eviction.
        {"name": "attend_256_ragged", "kind": "attend", "batch": 256, "heads": 8, "kv_heads": 8, "qk": 64, "vd": 64,
         "io": "f32", "type": "i8", "nk": 448, "page_rows": 16, "spans": "ragged", "acc": True},
        # Few streams with very long 16-bit caches: the work has to be split
        # over the cache's length. A pass over 1 GiB.
        {"name": "attend_long_65000", "kind": "attend", "batch": 4, "heads": 32, "kv_heads": 8, "qk": 128, "vd": 128,
         "io": "bf16", "type": "bf16", "nk": 65000, "page_rows": 64, "spans": "full", "acc": False},
        # A few streams' caches cut to a budget between two steps.
        {"name": "evict_8_to_256", "kind": "evict", "batch": 8, "kv_heads": 2, "qk": 48, "vd": 64, "type": "f16",
         "nk": 448, "keep": 256, "sink": 4, "recent": 64, "page_rows": 16},
        # Long caches cut to a quarter.
        {"name": "evict_16_to_2048", "kind": "evict", "batch": 16, "kv_heads": 8, "qk": 128, "vd": 128, "type": "bf16",
         "nk": 8192, "keep": 2048, "sink": 16, "recent": 512, "page_rows": 64},
        # The cross-attention of a decode step: 5 beams over the 375 frames
        # of their one utterance, in float32 like the decoder's activations.
        {"name": "cross_beams_5", "kind": "cross", "batch": 5, "memories": 1, "t": 1, "frames": 375, "heads": 8,
         "kv_heads": 2, "qk": 48, "vd": 64, "type": "f32", "ragged": False},
        # Teacher-forced hypotheses over the frames of 64 long clips: the
        # largest products.
        {"name": "cross_score_64x448", "kind": "cross", "batch": 64, "memories": 64, "t": 448, "frames": 1500,
         "heads": 8, "kv_heads": 8, "qk": 64, "vd": 64, "type": "bf16", "ragged": False},
        # Hypotheses and clips of unequal lengths, wide grouped-query heads.
        {"name": "cross_ragged_f16", "kind": "cross", "batch": 40, "memories": 8, "t": 333, "frames": 1500, "heads": 16,
         "kv_heads": 4, "qk": 128, "vd": 128, "type": "f16", "ragged": True},
        # A beam step's candidates over the tied head's vocabulary.
        {"name": "logprobs_beams_5", "kind": "logprobs", "rows": 5, "n": 8199, "top": 10, "type": "f32"},
        # Every position of 16 teacher-forced hypotheses over the benchmark's
        # vocabulary: one pass over 470 MB.
        {"name": "logprobs_score_7168", "kind": "logprobs", "rows": 7168, "n": 16384, "top": 5, "type": "f32"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


HEADS = [(8, 2, 48, 64), (8, 8, 64, 64), (8, 8, 64, 64), (16, 4, 128, 128), (32, 8, 128, 128), (6, 6, 48, 48),
         (12, 1, 64, 64), (5, 5, 80, 96)]


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "evict", "cross", "cross", "cross", "logprobs", "logprobs"])
    heads, kv_heads, qk, vd = rng.choice(HEADS)
    page_rows = rng.choice([1, 8, 16, 16, 64, 256])
    kv = rng.choice(["f32", "f16", "bf16", "i8"])
    row = kv_heads * (qk + vd)
    if kind == "append":
        t = 1 if rng.random() < 0.5 else _log_int(rng, 2, 448)
        cap = max(t, _log_int(rng, 16, 512))
        batch = _log_int(rng, 1, max(1, min(256, (14 << 20) // (cap * row))))
        return {"kind": kind, "batch": batch, "t": t, "kv_heads": kv_heads, "qk": qk, "vd": vd,
                "io": rng.choice(["f32", "f32", "f16", "bf16"]), "type": kv, "cap": cap, "page_rows": page_rows}
    if kind == "attend":
        batch = _log_int(rng, 1, 256)
        nk = _log_int(rng, 1, max(1, min(65000, (400 << 20) // (4 * batch * row))))
        return {"kind": kind, "batch": batch, "heads": heads, "kv_heads": kv_heads, "qk": qk, "vd": vd,
                "io": rng.choice(["f32", "f32", "f16", "bf16"]), "type": kv, "nk": nk, "page_rows": page_rows,
                "spans": rng.choice(["full", "ragged", "window"]), "acc": rng.random() < 0.4}
    if kind == "evict":
        batch = _log_int(rng, 1, 64)
        nk = _log_int(rng, 16, max(16, min(30000, (100 << 20) // (4 * batch * row))))
        keep = rng.randint(1, nk)
        sink = rng.randint(0, min(keep, 16))
        return {"kind": kind, "batch": batch, "kv_heads": kv_heads, "qk": qk, "vd": vd, "type": kv, "nk": nk,
                "keep": keep, "sink": sink, "recent": rng.randint(0, (keep - sink) // 2), "page_rows": page_rows}
    if kind == "cross":
        typ = rng.choice(["f32", "f16", "bf16"])
        t = 1 if rng.random() < 0.3 else _log_int(rng, 2, 448)
        frames = _log_int(rng, 1, 2900)
        work = 64 * 448 * 1500 * 8 * 64 // (8 if typ == "f32" else 1)
        batch = _log_int(rng, 1, max(1, min(64, work // (t * frames * heads * max(qk, vd)))))
        memories = batch if rng.random() < 0.6 else rng.randint(1, batch)
        return {"kind": kind, "batch": batch, "memories": memories, "t": t, "frames": frames, "heads": heads,
                "kv_heads": kv_heads, "qk": qk, "vd": vd, "type": typ, "ragged": rng.random() < 0.6}
    typ = rng.choice(["f32", "f32", "f16", "bf16"])
    n = rng.choice([8199, 16384, _log_int(rng, 32, 260000)])
    rows = _log_int(rng, 1, max(1, min(8192, 100_000_000 // n)))
    return {"kind": kind, "rows": rows, "n": n, "top": min(n, rng.choice([0, 1, 5, 10, 32])), "type": typ}


# ---- inputs ---------------------------------------------------------------------


def _pool(g, c, pool_pages):
    """The pages of a cache: normal keys and values, int8 ones as codes with a scale a row and head."""
    s = {}
    for name, width in (("k", c["qk"]), ("v", c["vd"])):
        shape = (pool_pages, c["page_rows"], c["kv_heads"], width)
        x = torch.empty(shape, dtype=torch.float32 if c["type"] in ("f32", "i8") else TYPES[c["type"]], device="cuda")
        x.normal_(generator=g)
        if c["type"] == "i8":
            s[name + "s"] = torch.empty(shape[:3], device="cuda").uniform_(0.01, 0.04, generator=g)
            x = (x * 40).round_().clamp_(-127, 127).to(torch.int8)
        s[name] = x
    return s


def _tables(g, batch, per, pool_pages):
    perm = torch.randperm(pool_pages, generator=g, device="cuda")
    return perm[:batch * per].view(batch, per).to(torch.int32).contiguous(), perm[batch * per:].to(torch.int32)


def _randn(g, shape, typ):
    return torch.randn(shape, generator=g, device="cuda").to(TYPES[typ])


def _lengths(g, n, most, ragged):
    """n lengths up to `most`; ragged: unequal ones, the first 0 (a padded slot) where there are several."""
    if not ragged:
        return torch.full((n,), most, dtype=torch.int32, device="cuda")
    ln = torch.randint(1, most + 1, (n,), generator=g, device="cuda", dtype=torch.int32)
    if n > 2:
        ln[0] = 0
        ln[1] = most
    return ln


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": c}
    zeros = lambda *shape, t="f32": torch.zeros(shape, dtype=TYPES[t], device="cuda")  # noqa: E731
    if c["kind"] == "append":
        B, t, R = c["batch"], c["t"], c["page_rows"]
        per = -(-c["cap"] // R)
        s |= _pool(g, c, B * per)
        s["pages"], _ = _tables(g, B, per, B * per)
        s["k_rows"] = _randn(g, (B, t, c["kv_heads"], c["qk"]), c["io"])
        s["v_rows"] = _randn(g, (B, t, c["kv_heads"], c["vd"]), c["io"])
        s["n"] = _lengths(g, B, t, t > 1)
        # where each stream's rows begin: so that they fit
        s["pos"] = (torch.rand(B, generator=g, device="cuda") * (c["cap"] - t + 1)).to(torch.int32)
    elif c["kind"] == "attend":
        B, R, nk = c["batch"], c["page_rows"], c["nk"]
        per = -(-nk // R)
        s |= _pool(g, c, B * per)
        s["pages"], _ = _tables(g, B, per, B * per)
        s["q"] = _randn(g, (B, c["heads"], c["qk"]), c["io"])
        s["out"] = zeros(B, c["heads"], c["vd"], t=c["io"])
        s["scale"] = math.sqrt(c["qk"])
        n = _lengths(g, B, nk, c["spans"] != "full")
        spans = torch.zeros(B, 4, dtype=torch.int32, device="cuda")
        spans[:, 3] = n
        if c["spans"] == "window":  # the first rows and a window of the last
            spans[:, 1] = torch.clamp(n, max=4)
            spans[:, 2] = torch.maximum(spans[:, 1], n - max(1, nk // 2))
        s["spans"] = spans
        if c["acc"]:
            s["acc"] = torch.rand(B, c["kv_heads"], nk, generator=g, device="cuda")
            s["acc_out"] = zeros(B, c["kv_heads"], nk)
    elif c["kind"] == "evict":
        B, R, nk = c["batch"], c["page_rows"], c["nk"]
        per, dper = -(-nk // R), -(-c["keep"] // R)
        s |= _pool(g, c, B * (per + dper))
        s["pages"], rest = _tables(g, B, per, B * (per + dper))
        s["dst"] = rest.view(B, dper).contiguous()
        # accumulated weights: a few heavy rows, many light ones, some never attended
        acc = torch.exp(2 * torch.randn(B, c["kv_heads"], nk, generator=g, device="cuda") - 3)
        s["acc"] = torch.where(torch.rand(acc.shape, generator=g, device="cuda") < 0.1, torch.zeros_like(acc), acc)
        s["acc_out"] = zeros(B, c["kv_heads"], c["keep"])
        s["len"] = _lengths(g, B, nk, True)
        s["len_out"] = torch.zeros(B, dtype=torch.int32, device="cuda")
        s["kept"] = torch.zeros(B, c["kv_heads"], c["keep"], dtype=torch.int32, device="cuda")
    elif c["kind"] == "cross":
        B, M = c["batch"], c["memories"]
        s["q"] = _randn(g, (B, c["t"], c["heads"], c["qk"]), c["type"])
        s["k"] = _randn(g, (M, c["frames"], c["kv_heads"], c["qk"]), c["type"])
        s["v"] = _randn(g, (M, c["frames"], c["kv_heads"], c["vd"]), c["type"])
        s["out"] = zeros(B, c["t"], c["heads"], c["vd"], t=c["type"])
        s["index"] = (torch.arange(B, device="cuda") % M).to(torch.int32)
        s["q_len"] = _lengths(g, B, c["t"], c["ragged"])
        s["k_len"] = _lengths(g, M, c["frames"], c["ragged"])
        s["scale"] = math.sqrt(c["qk"])
    else:
        x = 3 * torch.randn(c["rows"], c["n"], generator=g, device="cuda")
        # suppressed tokens
        x.masked_fill_(torch.rand(1, c["n"], generator=g, device="cuda") < 0.05, -math.inf)
        x[:, c["n"] // 2] = 1.0
        s["logits"] = x.to(TYPES[c["type"]])
        tok = torch.randint(0, c["n"], (c["rows"],), generator=g, device="cuda", dtype=torch.int32)
        tok[c["rows"] - c["rows"] // 8:] = -1  # padding behind the last hypothesis
        s["tokens"] = tok
        s["lp"], s["ent"] = zeros(c["rows"]), zeros(c["rows"])
        s["top"] = torch.zeros(c["rows"], c["top"], dtype=torch.int32, device="cuda")
        s["top_lp"] = zeros(c["rows"], c["top"])
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
    if c["kind"] == "append":
        _cache(s).append_dev(s["k_rows"], s["v_rows"], s["pos"], rows=s["n"], cap=c["cap"])
    elif c["kind"] == "attend":
        _cache(s).attend_dev(s["out"], s["q"], s["spans"], c["nk"], s["scale"], acc=s.get("acc"),
                             acc_out=s.get("acc_out"))
    elif c["kind"] == "evict":
        _cache(s).evict_dev(s["dst"], s["acc"], s["acc_out"], s["len"], s["len_out"], s["kept"], c["nk"],
                            sink=c["sink"], recent=c["recent"])
    elif c["kind"] == "cross":
        _needle().cross_attend_dev(s["out"], s["q"], s["k"], s["v"], s["scale"], q_len=s["q_len"], k_len=s["k_len"],
                                   index=s["index"])
    else:
        _needle().logprobs_dev(s["logits"], tokens=s["tokens"], lp=s["lp"], ent=s["ent"], top=s["top"],
                               top_lp=s["top_lp"])


# ---- the plain forms ----------------------------------------------------------------


def _values(s, name):
    """A pool as the values it stands for."""
    return s[name].float() * s[name + "s"].unsqueeze(-1) if name + "s" in s else s[name]


def _plain_append(s):
    c = s["case"]
    R = c["page_rows"]
    i = torch.arange(c["t"], device="cuda")
    b, i = torch.nonzero(i[None, :] < s["n"][:, None], as_tuple=True)
    row = s["pos"].long()[b] + i
    page, at = s["pages"].long()[b, row // R], row % R
    for name in ("k", "v"):
        x = s[name + "_rows"][b, i].float()
        if c["type"] == "i8":
            m = x.abs().amax(-1)
            sc = torch.where(m > 0, m / 127, torch.ones_like(m))
            s[name + "s"][page, at] = sc
            x = torch.round(x / sc.unsqueeze(-1)).clamp(-128, 127)
        s[name][page, at] = x.to(s[name].dtype)


def _softmax_av(logits, mask, v):
    """softmax of the unmasked logits times v, 0 for rows whose mask leaves nothing; the weights beside it."""
    logits = torch.where(mask, logits, torch.full_like(logits, -math.inf))
    m = logits.amax(-1, keepdim=True)
    p = torch.where(mask, torch.exp(logits - torch.where(m == -math.inf, torch.zeros_like(m), m)), torch.zeros_like(logits))
    d = p.sum(-1, keepdim=True)
    p = p / torch.where(d == 0, torch.ones_like(d), d)
    return torch.matmul(p, v), p


def _plain_attend(s):
    c = s["case"]
    B, nk, H, Hk = c["batch"], c["nk"], c["heads"], c["kv_heads"]
    pages = s["pages"].long()
    rows = [s[name][pages].float() * (s[name + "s"][pages].unsqueeze(-1) if name + "s" in s else 1) for name in ("k", "v")]
    k, v = (x.flatten(1, 2)[:, :nk] for x in rows)  # [B, nk, Hk, width]
    q = s["q"].float().view(B, Hk, H // Hk, c["qk"])
    logits = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) / s["scale"]
    j, sp = torch.arange(nk, device="cuda"), s["spans"].unsqueeze(-1)
    mask = ((j >= sp[:, 0]) & (j < sp[:, 1])) | ((j >= sp[:, 2]) & (j < sp[:, 3]))  # [B, nk]
    o, p = _softmax_av(logits, mask[:, None, None, :].expand_as(logits), v.permute(0, 2, 1, 3).contiguous())
    s["out"].copy_(o.reshape(B, H, c["vd"]))
    if c["acc"]:
        s["acc_out"].copy_(torch.where(mask[:, None, :], s["acc"] + p.sum(2), s["acc_out"]))


def _plain_evict(s):
    c = s["case"]
    B, Hk, nk, keep, R = c["batch"], c["kv_heads"], c["nk"], c["keep"], c["page_rows"]
    j = torch.arange(nk, device="cuda")
    n = s["len"].long()[:, None, None]
    held = (j < c["sink"]) | (j >= n - c["recent"])
    score = torch.where(held, torch.full_like(s["acc"], math.inf), s["acc"])
    score = torch.where(j < n, score, torch.full_like(score, -math.inf))
    first = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :keep]
    first = torch.where(first < n, first, torch.full_like(first, nk))  # rows behind the stream's last
    kept = torch.sort(first, dim=-1).values
    live = kept < nk
    src = torch.where(live, kept, torch.zeros_like(kept))
    b, h, i = torch.nonzero(live, as_tuple=True)
    r = src[b, h, i]
    sp, dp = s["pages"].long()[b, r // R], s["dst"].long()[b, i // R]
    for name in ("k", "v", "ks", "vs"):
        if name in s:
            s[name][dp, i % R, h] = s[name][sp, r % R, h]
    s["kept"].copy_(torch.where(live, kept, torch.full_like(kept, -1)))
    s["acc_out"].copy_(torch.where(live, s["acc"].gather(-1, src), s["acc_out"]))
    s["len_out"].copy_(torch.clamp(s["len"], max=keep))


def _plain_cross(s):
    c = s["case"]
    B, t, H, Hk = c["batch"], c["t"], c["heads"], c["kv_heads"]
    idx = s["index"].long()
    k, v = s["k"].float()[idx], s["v"].float()[idx]  # [B, F, Hk, width]
    q = s["q"].float().view(B, t, Hk, H // Hk, c["qk"]).permute(0, 2, 3, 1, 4).reshape(B, Hk, -1, c["qk"])
    logits = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) / s["scale"]
    mask = torch.arange(c["frames"], device="cuda") < s["k_len"][idx][:, None]
    o, _ = _softmax_av(logits, mask[:, None, None, :].expand_as(logits), v.permute(0, 2, 1, 3).contiguous())
    o = o.view(B, Hk, H // Hk, t, c["vd"]).permute(0, 3, 1, 2, 4).reshape(B, t, H, c["vd"])
    rows = (torch.arange(t, device="cuda") < s["q_len"][:, None])[..., None, None]
    s["out"].copy_(torch.where(rows, o.to(s["out"].dtype), s["out"]))


def _plain_logprobs(s):
    c = s["case"]
    x = s["logits"].float()
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    d = e.sum(-1, keepdim=True)
    lse = m + torch.log(d)
    tok = s["tokens"].long()
    given = x.gather(-1, tok.clamp(min=0)[:, None]) - lse
    s["lp"].copy_(torch.where(tok >= 0, given[:, 0], torch.zeros_like(s["lp"])))
    s["ent"].copy_(torch.where(e > 0, e / d * (lse - x), torch.zeros_like(x)).sum(-1))
    if c["top"]:
        top = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :c["top"]]
        s["top"].copy_(top)
        s["top_lp"].copy_(x.gather(-1, top) - lse)


PLAIN = {"append": _plain_append, "attend": _plain_attend, "evict": _plain_evict, "cross": _plain_cross,
         "logprobs": _plain_logprobs}


def _outputs(s):
    kind = s["case"]["kind"]
    if kind == "append":
        return [_values(s, "k"), _values(s, "v")]
    if kind == "attend":
        return [s["out"], s["acc_out"]] if s["case"]["acc"] else [s["out"]]
    if kind == "evict":
        return [_values(s, "k"), _values(s, "v"), s["acc_out"], s["kept"], s["len_out"]]
    if kind == "cross":
        return [s["out"]]
    return [s["lp"], s["ent"], s["top"], s["top_lp"]] if s["case"]["top"] else [s["lp"], s["ent"]]


def run(state):
    if own:
        _run_own(state)
    else:
        PLAIN[state["case"]["kind"]](state)
    return _outputs(state)


# ---- what a pass cannot do without ---------------------------------------------------


def work(case):
    """Bytes read and written once, and operations; unequal lengths count with their mean."""
    c = case
    if c["kind"] == "append":
        rows = c["batch"] * (c["t"] if c["t"] == 1 else (c["t"] + 1) / 2) * c["kv_heads"]
        scales = 8 if c["type"] == "i8" else 0
        return {"bytes": rows * ((c["qk"] + c["vd"]) * (SIZE[c["io"]] + SIZE[c["type"]]) + scales), "flops": 0}
    if c["kind"] == "attend":
        keys = c["batch"] * (c["nk"] if c["spans"] == "full" else (c["nk"] + 1) / 2)
        if c["spans"] == "window":
            keys *= 0.75
        row = (c["qk"] + c["vd"]) * SIZE[c["type"]] + (8 if c["type"] == "i8" else 0) + (8 if c["acc"] else 0)
        ends = c["batch"] * c["heads"] * (c["qk"] + c["vd"]) * SIZE[c["io"]]
        return {"bytes": keys * c["kv_heads"] * row + ends, "flops": 2 * keys * c["heads"] * (c["qk"] + c["vd"])}
    if c["kind"] == "evict":
        heads = c["batch"] * c["kv_heads"]
        kept = min(c["keep"], (c["nk"] + 1) / 2)
        row = (c["qk"] + c["vd"]) * SIZE[c["type"]] + (8 if c["type"] == "i8" else 0)
        return {"bytes": heads * (4 * (c["nk"] + 1) / 2 + kept * (2 * row + 8)), "flops": 0}
    if c["kind"] == "cross":
        part = 0.5 if c["ragged"] else 1
        size = SIZE[c["type"]]
        rows, keys = c["batch"] * c["t"] * part, c["frames"] * part
        return {"bytes": size * (c["qk"] + c["vd"]) * (rows * c["heads"] + c["memories"] * keys * c["kv_heads"]),
                "flops": 2 * rows * keys * c["heads"] * (c["qk"] + c["vd"])}
    return {"bytes": c["rows"] * (c["n"] * SIZE[c["type"]] + 12 + 8 * c["top"]), "flops": 4 * c["rows"] * c["n"]}


# ---- the definitions in float64 --------------------------------------------------------


def _exact_append(s):
    """A row goes to its place; in int8 its scale is float32(max |x| / 127) and its
    codes the nearest whole numbers to float32(x / scale), as the caches hold them."""
    c, R = s["case"], s["case"]["page_rows"]
    outs = []
    for name in ("k", "v"):
        pool = _values(s, name).double()
        n, pos, pages = s["n"].tolist(), s["pos"].tolist(), s["pages"].long()
        for b in range(c["batch"]):
            x = s[name + "_rows"][b, :n[b]].double()
            if c["type"] == "i8":
                sc = (x.abs().amax(-1, keepdim=True) / 127).float().double()
                sc[sc == 0] = 1
                x = torch.round((x / sc).float().double()) * sc
            at = torch.arange(pos[b], pos[b] + n[b], device="cuda")
            pool[pages[b, at // R], at % R] = x
        outs.append(pool)
    return outs


def _exact_attend(s):
    c = s["case"]
    G = c["heads"] // c["kv_heads"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    acc = s["acc_out"].double() if c["acc"] else None
    for b, (lo0, hi0, lo1, hi1) in enumerate(s["spans"].tolist()):
        j = torch.cat([torch.arange(lo0, hi0, device="cuda"), torch.arange(lo1, hi1, device="cuda")])
        if not len(j):
            continue
        page, at = s["pages"].long()[b, j // c["page_rows"]], j % c["page_rows"]
        k, v = (s[x][page, at].double() * (s[x + "s"][page, at].double().unsqueeze(-1) if x + "s" in s else 1)
                for x in ("k", "v"))
        for h in range(c["kv_heads"]):
            w = torch.softmax(s["q"][b, h * G:(h + 1) * G].double() @ k[:, h].t().contiguous() / s["scale"], -1)
            out[b, h * G:(h + 1) * G] = w @ v[:, h].contiguous()
            if c["acc"]:
                acc[b, h, j] = s["acc"][b, h, j].double() + w.sum(0)
    return [out, acc] if c["acc"] else [out]


def _exact_evict(s):
    c, R = s["case"], s["case"]["page_rows"]
    k, v = _values(s, "k").double(), _values(s, "v").double()
    acc = s["acc_out"].double()
    for b, n in enumerate(s["len"].tolist()):
        for h in range(c["kv_heads"]):
            score = s["acc"][b, h, :n].double()
            score[:c["sink"]] = math.inf
            score[max(0, n - c["recent"]):] = math.inf
            # the lowest row first among equals
            rows = torch.argsort(-score, stable=True)[:c["keep"]].sort().values
            i = torch.arange(len(rows), device="cuda")
            src, dst = s["pages"].long()[b, rows // R], s["dst"].long()[b, i // R]
            k[dst, i % R, h] = k[src, rows % R, h]
            v[dst, i % R, h] = v[src, rows % R, h]
            acc[b, h, :len(rows)] = s["acc"][b, h, rows].double()
    return [k, v, acc, None, None]


def _exact_cross(s):
    c = s["case"]
    G = c["heads"] // c["kv_heads"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    for b, (n, m) in enumerate(zip(s["q_len"].tolist(), s["index"].tolist())):
        f = int(s["k_len"][m])
        if not n or not f:
            continue
        for h in range(c["heads"]):
            k, v = s["k"][m, :f, h // G].double(), s["v"][m, :f, h // G].double()
            w = torch.softmax(s["q"][b, :n, h].double() @ k.t().contiguous() / s["scale"], -1)
            out[b, :n, h] = w @ v.contiguous()
    return [out]


def _exact_logprobs(s):
    c = s["case"]
    parts = []
    for lo in range(0, c["rows"], 1024):
        x = s["logits"][lo:lo + 1024].double()
        lp = x - torch.logsumexp(x, -1, keepdim=True)
        tok = s["tokens"][lo:lo + 1024].long()
        given = lp[torch.arange(len(tok), device="cuda"), tok.clamp(min=0)].masked_fill(tok < 0, 0.0)
        parts.append((given, torch.special.entr(lp.exp()).sum(-1), torch.topk(lp, c["top"]).values))
    lp, ent, top_lp = (torch.cat(p) for p in zip(*parts))
    return [lp, ent, None, top_lp] if c["top"] else [lp, ent]


EXACT = {"append": _exact_append, "attend": _exact_attend, "evict": _exact_evict, "cross": _exact_cross,
         "logprobs": _exact_logprobs}


def exact(case, seed):
    return EXACT[case["kind"]](prepare(case, seed))
