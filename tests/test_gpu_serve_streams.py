"""The serving operators that work in parts, from two threads at once and in
two graphs replayed beside each other: each call's partials are its own."""

import threading

import pytest

from go_whistle_amd import needle

pytestmark = pytest.mark.gpu


def gen(seed):
    import torch

    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def calls(seed):
    """Calls on inputs of their own that all take a workspace, and their outputs."""
    import torch

    g = gen(seed)
    mk = lambda *s, t=torch.float32: torch.randn(*s, generator=g, device="cuda").to(t)  # noqa: E731
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    out, fns = [], []
    for t, typ in ((3, torch.bfloat16), (3, torch.float32), (90, torch.float16)):  # parts of a memory of 3000 frames
        q, k, v = mk(1, t, 2, 64, t=typ), mk(1, 3000, 2, 64, t=typ), mk(1, 3000, 2, 64, t=typ)
        out.append(torch.zeros_like(q))
        fns.append(lambda o=out[-1], q=q, k=k, v=v: needle.cross_attend_dev(o, q, k, v, 8.0))
    x, tok = mk(3, 90000) * 3, i32([5, 89999, -1])  # parts of a row
    lp, ent, tl, top = torch.zeros(3, device="cuda"), torch.zeros(3, device="cuda"), torch.zeros(3, 6, device="cuda"), i32([[0] * 6] * 3)
    out += [lp, ent, tl, top]
    fns.append(lambda: needle.logprobs_dev(x, tok, lp, ent, top, tl))
    c = needle.PagedKV(mk(190, 16, 1, 64), mk(190, 16, 1, 64), torch.randperm(190, generator=g, device="cuda").int().view(1, 190))
    q, o, a, spans = mk(1, 5, 64), torch.zeros(1, 5, 64, device="cuda"), torch.zeros(1, 1, 3040, device="cuda"), i32([[0, 7, 9, 3037]])
    out += [o, a]
    fns.append(lambda: c.attend_dev(o, q, spans, 3040, 8.0, acc_out=a))
    return out, lambda: [f() for f in fns]


def expected(out, run):
    import torch

    run()
    torch.cuda.synchronize()
    want = [o.clone() for o in out]
    assert all(w.count_nonzero() > 0 for w in want)
    return want


def test_two_threads():
    import torch

    sets = [calls(1), calls(2)]
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

    sets = [calls(s) for s in (3, 4, 5)]
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
