"""Layouts of the operands of the operators around steps of several rows:
rows at any stream and row strides are taken wherever written rows share no element
with others, and refused where they do, before any device call (no GPU)."""

import ctypes
import random

import pytest

from go_whistle_amd._lib import CQPanic, HeadsLayout, KvPaged, check, lib

P = 1 << 12  # a pointer that is never dereferenced: the checks come first
BASE = 1 << 24
FAR = 1 << 40


def elements(batch, t, at, width, stream, row):
    return [range(at + b * stream + i * row, at + b * stream + i * row + width) for b in range(batch) for i in range(t)]


def share(batch, t, x, y):
    """Whether rows of two arrays, (address, width, stream, row) in elements, share an element, by counting."""
    seen = set().union(*elements(batch, t, *x))
    return any(not seen.isdisjoint(r) for r in elements(batch, t, *y))


def apart(batch, t, x):
    """Whether an array's rows share no element with each other."""
    spans = elements(batch, t, *x)
    return len(set().union(*spans)) == sum(map(len, spans))


def norm(layout, batch, t, q, k, qo, ko, heads=4, kv_heads=2, width=16, typ=0, rows=None):
    """The call without positions, which are looked at after the layout: None where the layout is taken."""
    size = 2 if typ else 4
    with pytest.raises(CQPanic) as e:
        check(lib().nd_qk_norm_rope_dev(qo * size, ko * size, q * size, k * size, typ, ctypes.byref(layout), batch, t, heads,
                                        kv_heads, width, P, P, P, P, 10, None, rows, None))
    return None if "without positions" in str(e.value) else str(e.value)


ORDERS = {  # (stream stride, row stride) of rows of 128 + 16 elements, 4 streams of 5 rows
    "streams of rows": (5 * 144, 144),
    "rows of streams": (144, 4 * 144),
    "padded streams": (5 * 144 + 16, 144),
    "streams padded by part of a row": (5 * 144 + 100, 144),
    "padded rows of streams": (144, 4 * 144 + 16),
    "backwards": (-5 * 144, -144),
    "rows of streams backwards": (-144, 4 * 144),
}


@pytest.mark.parametrize("order", ORDERS)
@pytest.mark.parametrize("typ", [0, 1])
def test_packed_products_in_place(order, typ):
    # queries of 64 and keys of 32 side by side in rows of 128 (queries, keys, values) and some padding
    s, r = ORDERS[order]
    y = HeadsLayout(s, r, s, r, s, r, s, r)
    assert norm(y, 4, 5, BASE, BASE + 64, BASE, BASE + 64, typ=typ) is None


@pytest.mark.parametrize("order", ORDERS)
def test_two_outputs_of_one_buffer(order):
    s, r = ORDERS[order]
    y = HeadsLayout(640, 128, 640, 128, s, r, s, r)
    for off in (0, 32, 63, 64, 65, 96, 112, 113, 144 - 64, 144):
        x, k = (BASE, 64, s, r), (BASE + off, 32, s, r)
        got = norm(y, 4, 5, FAR, 2 * FAR, BASE, BASE + off)
        assert (got is None) == (not share(4, 5, x, k)), off
        assert got is None or "onto a part" in got


def test_layouts_by_counting():
    """Random strides, the outputs' own and others, small enough to count."""
    rng = random.Random(5)
    taken = refused = 0
    for _ in range(3000):
        batch, t = rng.randint(1, 5), rng.randint(1, 5)
        strides = lambda: rng.choice([(t * 100, 100), (100, batch * 100), (t * 100 + rng.randint(0, 120), 100),  # noqa: E731
                                      (rng.randint(64, 700), rng.randint(64, 700)), (rng.randint(-700, -64), rng.randint(64, 700))])
        ks, kr = strides()
        qs, qr = (ks, kr) if rng.random() < 0.7 else strides()
        q, k = BASE, BASE + rng.randint(-150, 150)
        if not apart(batch, t, (q, 64, qs, qr)) or not apart(batch, t, (k, 32, ks, kr)):
            continue
        y = HeadsLayout(1 << 20, 64, 1 << 20, 32, qs, qr, ks, kr)
        want = share(batch, t, (q, 64, qs, qr), (k, 32, ks, kr))
        got = norm(y, batch, t, FAR, 2 * FAR, q, k)
        assert (got is not None) == want, (batch, t, qs, qr, ks, kr, k - q)
        taken, refused = taken + (not want), refused + want
    assert taken > 200 and refused > 200


def test_counts_may_leave_rows_apart():
    """Of rows[b] rows the host knows only that they are rows: streams closer than t rows are the caller's to keep apart."""
    s, r = 3 * 144 + 8, 144
    y = HeadsLayout(s, r, s, r, s, r, s, r)
    assert norm(y, 4, 5, BASE, BASE + 64, BASE, BASE + 64, rows=P) is None
    # but rows of one stream, and the streams' first rows, meet whatever the counts
    assert "onto a part" in norm(y, 4, 5, FAR, 2 * FAR, BASE, BASE + 63, rows=P)
    assert "onto a part" in norm(y, 4, 5, FAR, 2 * FAR, BASE, BASE + s - 1, rows=P)
    # and streams of t rows that lie apart are taken for whole
    s = 5 * 144
    y = HeadsLayout(s, r, s, r, s, r, s, r)
    assert norm(y, 4, 5, BASE, BASE + 64, BASE, BASE + 64, rows=P) is None
    assert "onto a part" in norm(y, 4, 5, FAR, 2 * FAR, BASE, BASE + s + 2 * r, rows=P)


def test_large_layouts_are_settled():
    """Interleaved rows of many streams and rows: the answer does not take a walk over all of them."""
    batch, t = 4096, 2000
    for s, r in ((6144, batch * 6144), (t * 6144 + 64, 6144), (6144, batch * 6144 + 64)):
        y = HeadsLayout(s, r, s, r, s, r, s, r)
        assert norm(y, batch, t, BASE, BASE + 2048, BASE, BASE + 2048, heads=16, kv_heads=4, width=128) is None


def attend(batch, t, out, q, os, orow, qs, qrow, typ=0, rows=None, heads=4, qk=16, vd=16):
    c = KvPaged(P, P, None, None, P, 1, 2, qk, vd, 4, 16, 8)
    size = 2 if typ else 4
    check(lib().kv_attend_rows_paged_dev(ctypes.byref(c), out * size, os, orow, q * size, qs, qrow, typ, batch, t, heads, rows, P, 64,
                                         0, 0, 4.0, None))


@pytest.mark.parametrize("batch,t", [(1, 1), (3, 1), (1, 5), (3, 5)])
@pytest.mark.parametrize("typ", [0, 1])
def test_attention_onto_its_queries(batch, t, typ):
    # outputs of 64 in rows of 144, the queries at every place that shares an element with them
    for rows in (None, P):
        for qrow, qs in ((144, t * 144), (144, t * 144 + 8), (batch * 144, 144), (64, t * 64), (0, 0), (200, 77)):
            for off in (0, 1, 63, -63, 64, 100, t * 64 - 1):
                if share(batch, t, (BASE, 64, t * 144, 144), (BASE + off, 64, qs, qrow)):
                    with pytest.raises(CQPanic, match="onto its queries"):
                        attend(batch, t, BASE, BASE + off, t * 144, 144, qs, qrow, typ=typ, rows=rows)


@pytest.mark.parametrize("batch,t", [(1, 1), (3, 1), (1, 5), (3, 5)])
@pytest.mark.parametrize("typ", [0, 1])
def test_keys_and_values_read_to_one_place(batch, t, typ):
    # key rows of 2 x 16 and value rows of 2 x 32 values, each apart from its own
    c, size = KvPaged(P, P, None, None, P, 1, 2, 16, 32, 4, 16, 8), 2 if typ else 4
    for rows in (None, P):
        for vrow, vs in ((144, t * 144), (144, t * 144 + 8), (batch * 144, 144), (64, t * 64), (200, 77 + t * 200)):
            for off in (0, 1, 31, -63, 32, 100, t * 64 - 1):
                if share(batch, t, (BASE, 32, t * 144, 144), (BASE + off, 64, vs, vrow)):
                    with pytest.raises(CQPanic, match="to one place"):
                        check(lib().kv_read_paged_dev(ctypes.byref(c), BASE * size, t * 144, 144, (BASE + off) * size, vs, vrow, typ,
                                                      batch, t, rows, P, None))
