"""The operators around steps of several rows as they are used together: prompts
and drafted tokens of a small synthetic model through norms and rotation, paged
caches, attention and verification; captured, from two threads, and refused."""

import math
import threading

import numpy as np
import pytest

from go_whistle_amd import needle
from go_whistle_amd._lib import CQPanic
from page8_ref import CACHES, gen, i32, make_cache, verify64
from serve_ref import host

pytestmark = pytest.mark.gpu

H, HK, W, DIM, N, CAP, R = 4, 2, 64, 128, 300, 128, 16


class Model:
    """One attention layer over tied embeddings, float32."""

    def __init__(self, seed, streams, name):
        import torch

        g = gen(seed)
        mk = lambda *s, z=1.0: torch.randn(*s, generator=g, device="cuda") * z  # noqa: E731
        self.emb, self.wqkv = mk(N, DIM), mk(DIM, (H + 2 * HK) * W, z=DIM ** -0.5)
        self.wo = mk(H * W, DIM, z=0.2)
        self.qg, self.kg = 2 + mk(W, z=0.1), 2 + mk(W, z=0.1)
        a = torch.arange(CAP, device="cuda")[:, None] * 100.0 ** (-torch.arange(W // 2, device="cuda") / (W // 2))
        self.rope = a.cos().contiguous(), a.sin().contiguous()
        self.cache = make_cache(g, name, streams, CAP // R, R, HK, W, W)
        self.streams = streams

    def rows(self, tokens, pos, counts=None):
        """Logits [streams, t, N] of the tokens at positions pos[b] on, appended to the cache."""
        import torch

        B, t = tokens.shape
        x = self.emb[tokens.long().clamp(min=0)]
        qkv = torch.matmul(x.view(-1, DIM), self.wqkv).view(B, t, -1)
        q, k, v = (qkv[..., lo * W:hi * W].unflatten(-1, (hi - lo, W)) for lo, hi in ((0, H), (H, H + HK), (H + HK, H + 2 * HK)))
        needle.qk_norm_rope_dev(q, k, q, k, self.qg, self.kg, self.rope, pos, rows=counts)
        self.cache.append_dev(k, v, pos, rows=counts)
        out = torch.zeros(B, t, H, W, device="cuda")
        self.cache.attend_rows_dev(out, q, pos, math.sqrt(W), rows=counts, window=40, sink=4)
        y = x + torch.matmul(out.view(-1, H * W), self.wo).view(B, t, DIM)
        return torch.matmul(y.view(-1, DIM), self.emb.t().contiguous()).view(B, t, N) / math.sqrt(DIM)


def prompts(seed):
    import torch

    return torch.randint(0, N, (3, 21), generator=gen(seed), device="cuda").int(), i32([21, 9, 15])


def first_tokens(m, p, n):
    import torch

    logits = m.rows(p, i32([0, 0, 0]), n)
    return logits[torch.arange(3, device="cuda"), (n - 1).long()].argmax(-1).int()


def by_tokens(seed, name, steps):
    """Greedy decoding a token at a time."""
    m = Model(seed, 3, name)
    p, n = prompts(seed)
    tok, pos, out = first_tokens(m, p, n), n.clone(), []
    for _ in range(steps):
        out.append(tok)
        tok = m.rows(tok[:, None], pos)[:, 0].argmax(-1).int()
        pos = pos + 1
    return [[int(t[b]) for t in out] for b in range(3)]


@pytest.mark.parametrize("name", ["float32", "float16"])
def test_drafts_give_the_tokens_of_single_steps(name):
    # greedy decoding with drafts, right and wrong ones, is greedy decoding
    import torch

    steps, t = 24, 4
    want = by_tokens(30, name, steps)
    m = Model(30, 3, name)
    p, n = prompts(30)
    tok, pos = first_tokens(m, p, n), n.clone()
    got = [[int(x)] for x in tok]
    rng = np.random.default_rng(1)
    accepted, tokens, lp = i32([0] * 3), torch.zeros(3, t + 1, dtype=torch.int32, device="cuda"), torch.zeros(3, t + 1, device="cuda")
    total = 0
    while min(len(x) for x in got) < steps:
        drafts = []
        for b in range(3):  # what comes, with a wrong token here and there
            d = (want[b] + [0] * 2 * t)[len(got[b]):len(got[b]) + t]
            drafts.append([x if rng.random() < 0.8 else int(rng.integers(0, N)) for x in d])
        drafts = i32(drafts)
        logits = m.rows(torch.cat([tok[:, None], drafts], 1).contiguous(), pos)
        needle.verify_drafts_dev(accepted, tokens, logits, drafts, temperature=0.0, lp=lp)
        a = accepted.tolist()
        for b in range(3):
            got[b] += tokens[b, :a[b] + 1].tolist()
            ref = torch.log_softmax(logits[b, :a[b] + 1].double(), -1)[torch.arange(a[b] + 1, device="cuda"), tokens[b, :a[b] + 1].long()]
            assert torch.allclose(lp[b, :a[b] + 1].double(), ref, rtol=1e-6, atol=1e-6)
        tok = tokens.gather(1, accepted.long()[:, None])[:, 0].contiguous()
        pos = pos + accepted + 1
        total += sum(a)
    assert [x[:steps] for x in got] == want and total > 10


@pytest.mark.parametrize("name", CACHES)
def test_drafts_from_another_model(name):
    # both models' caches of every type, drafts drawn from one and verified against the other
    import torch

    m, d = Model(31, 3, name), Model(32, 3, name)
    d.emb = m.emb + 0.3 * d.emb
    d.wqkv, d.wo = m.wqkv, m.wo
    p, n = prompts(31)
    g, t = gen(33), 3
    tok, pos = first_tokens(m, p, n), n.clone()
    first_tokens(d, p, n)
    accepted, tokens = i32([0] * 3), torch.zeros(3, t + 1, dtype=torch.int32, device="cuda")
    total = 0
    for _ in range(8):
        seq, rows = [tok], []
        for i in range(t):
            rows.append(d.rows(seq[-1][:, None], pos + i)[:, 0])
            seq.append(torch.multinomial(torch.softmax(rows[-1], -1), 1, generator=g)[:, 0].int())
        d.rows(seq[-1][:, None], pos + t)
        drafts, draft = torch.stack(seq[1:], 1).contiguous(), torch.stack(rows, 1)
        target = m.rows(torch.stack(seq, 1).contiguous(), pos)
        u, nxt = torch.rand(3, t, generator=g, device="cuda"), torch.rand(3, generator=g, device="cuda")
        needle.verify_drafts_dev(accepted, tokens, target, drafts, draft=draft, u=u, u_next=nxt)
        for b in range(3):
            a, want, _ = verify64(host(target[b]), host(drafts[b]), host(draft[b]), host(u[b]), float(nxt[b]), t, 1.0)
            assert int(accepted[b]) == a and tokens[b].tolist() == want.tolist()
        total += int(accepted.sum())
        tok = tokens.gather(1, accepted.long()[:, None])[:, 0].contiguous()
        pos = pos + accepted + 1
    assert total > 0 and target.isfinite().all()


def step_calls(seed):
    """A step's calls, parts of long caches and of long logits among them, and their outputs."""
    import torch

    g = gen(seed)
    out, fns = [], []
    for name, io in (("bfloat16", "bfloat16"), ("e4m3", "float16"), ("i8p", "float32")):
        c = make_cache(g, name, 1, 190, 16, 2, 64, 64)
        mk = lambda *s: torch.randn(*s, generator=g, device="cuda").to(getattr(torch, io))  # noqa: E731
        q, k, v = mk(1, 3, 4, 64), mk(1, 3, 2, 64), mk(1, 3, 2, 64)
        gain, pos = torch.rand(64, generator=g, device="cuda") + 0.5, i32([3030])
        a = torch.rand(3040, 32, generator=g, device="cuda")
        qo, ko, o = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(q)
        kb, vb = (torch.zeros(1, 16, 2, 64, device="cuda") for _ in range(2))
        out += [qo, ko, o, kb, vb]

        def call(c=c, q=q, k=k, v=v, gain=gain, pos=pos, rope=(a.cos(), a.sin()), qo=qo, ko=ko, o=o, kb=kb, vb=vb, at=i32([3024])):
            needle.qk_norm_rope_dev(qo, ko, q, k, gain, gain, rope, pos)
            c.append_dev(ko, v, pos)
            c.attend_rows_dev(o, qo, pos, 8.0)
            c.read_dev(kb, vb, at, rows=None)

        fns.append(call)
    x, y = (torch.randn(2, n, 30000, generator=g, device="cuda") * 3 for n in (4, 3))
    d, u, nxt = i32([[5, 29999, 17], [1, 2, 3]]), torch.rand(2, 3, generator=g, device="cuda") * 0.1, torch.rand(2, generator=g, device="cuda")
    acc, tok, lp = i32([0, 0]), torch.zeros(2, 4, dtype=torch.int32, device="cuda"), torch.zeros(2, 4, device="cuda")
    out += [acc, tok, lp]
    fns.append(lambda: needle.verify_drafts_dev(acc, tok, x, d, draft=y, u=u, u_next=nxt, lp=lp))
    return out, lambda: [f() for f in fns]


def expected(out, run):
    import torch

    run()
    torch.cuda.synchronize()
    run()  # the caches' scales have risen
    torch.cuda.synchronize()
    return [o.clone() for o in out]


def test_two_threads():
    import torch

    sets = [step_calls(1), step_calls(2)]
    want = [expected(*s) for s in sets]
    bad = []

    def work(z):
        out, run = sets[z]
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(30):
                for o in out:
                    o.zero_()
                run()
                stream.synchronize()
                bad.extend(i for i, (o, w) in enumerate(zip(out, want[z])) if not torch.equal(o, w))

    threads = [threading.Thread(target=work, args=(z,)) for z in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_two_graphs_and_eager_calls():
    import torch

    sets = [step_calls(s) for s in (3, 4, 5)]
    want = [expected(*s) for s in sets]
    graphs = []
    for _, run in sets[:2]:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            run()
    streams = [torch.cuda.Stream() for _ in sets]
    for r in range(5):
        for out, _ in sets:
            for o in out:
                o.zero_()
        torch.cuda.synchronize()
        for z in range(2):
            with torch.cuda.stream(streams[z]):
                graphs[z].replay()
        with torch.cuda.stream(streams[2]):
            sets[2][1]()
        torch.cuda.synchronize()
        for z, (out, _) in enumerate(sets):
            assert all(torch.equal(o, w) for o, w in zip(out, want[z])), (r, z)


def test_wrappers_refuse():
    import torch

    c = make_cache(gen(1), "e4m3", 2, 4, 16, 2, 64, 64)
    f = lambda *s, t=torch.float32: torch.zeros(*s, device="cuda", dtype=t)  # noqa: E731
    q, pos = f(2, 3, 4, 64), i32([0, 0])
    for kw in (dict(out=f(2, 3, 4, 48)), dict(out=f(2, 3, 4, 64, t=torch.float16)), dict(q=f(3, 3, 4, 64)), dict(pos=i32([0])),
               dict(pos=pos.long()), dict(rows=i32([1])), dict(nk_max=65), dict(nk_max=-1), dict(window=-1), dict(sink=2 ** 40),
               dict(scale=0.0), dict(q=f(2, 3, 4, 64).cpu()), dict(q=f(2, 4, 3, 64).transpose(1, 2)), dict(out=f(2, 1, 4, 64).expand(2, 3, 4, 64))):
        with pytest.raises(CQPanic):
            c.attend_rows_dev(**(dict(out=f(2, 3, 4, 64), q=q, pos=pos, scale=8.0) | kw))
    k = f(2, 3, 2, 64)
    for args in ((k, f(2, 3, 2, 48), pos), (k, k[:, :2], pos), (k, k, pos.long()), (k, k, i32([0])), (k.char(), k.char(), pos),
                 (f(2, 1, 2, 64).expand(2, 3, 2, 64), f(2, 3, 2, 64), pos)):
        with pytest.raises(CQPanic):
            c.read_dev(*args)
    for args, kw in (((f(2, 3, 4, 64), None, q, None), dict(rope=(f(9, 32), f(9, 32)))), ((f(2, 3, 4, 48), None, q, None), {}),
                     ((f(2, 3, 4, 64), None, q, None), dict(q_gain=f(32))), ((f(2, 3, 4, 64), k, q, k.half()), {}),
                     ((f(2, 3, 4, 64), None, q, None), dict(rope=(f(9, 32), f(8, 32)), pos=pos)),
                     ((f(2, 1, 4, 64).expand(2, 3, 4, 64), None, q, None), {})):
        with pytest.raises(CQPanic):
            needle.qk_norm_rope_dev(*args, **kw)
    x, d = f(2, 4, 50), torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    ok = dict(accepted=i32([0, 0]), tokens=torch.zeros(2, 4, dtype=torch.int32, device="cuda"), target=x, drafts=d, u=f(2, 3), u_next=f(2))
    for kw in (dict(target=f(2, 3, 50)), dict(draft=f(2, 4, 50)), dict(u=None), dict(u_next=None), dict(u=f(2, 4)), dict(tokens=d),
               dict(accepted=d[:, 0]), dict(drafts=d.long()), dict(lp=f(2, 3)), dict(temperature=-1.0), dict(target=f(2, 50, 4).transpose(1, 2)),
               dict(drafted=i32([1])), dict(draft=f(2, 3, 50, t=torch.float16))):
        with pytest.raises(CQPanic):
            needle.verify_drafts_dev(**(ok | kw))
